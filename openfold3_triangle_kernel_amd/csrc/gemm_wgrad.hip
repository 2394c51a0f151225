// Split-K weight-gradient products (MN-contiguous operands, f32 partials
// folded in fixed order): the TriMul dW5 and the pair-stack
// projection weight gradients.  Own translation unit for its stage shape:
// 64-deep k-steps, two stages (measured best for these long-K, few-tile
// products; the contraction shape in gemm.hip is 32 deep, three stages).  The
// linear layer's products (tpf_row_gemm_bf16) run on this shape too.
#define TPF_GEMM_IMPL gk64
#include "gemm_impl.hpp"

namespace tpf {

using namespace gk64;

int gemm_launch_wgrad(const GemmArgs& g0, hipStream_t stream, const char* fn) {
  GemmArgs g = g0;
  int rc = gemm_prepare(g, 0, 0, 1, g0.batch > 0 ? g0.batch : 1, fn);
  if (rc) return rc;
  dim3 grid((unsigned)((gemm_tiles(g) + 7) / 8 * 8));
  hipLaunchKernelGGL((gemm_bf16_kernel<false, false, true>), grid, dim3(256), 0, stream, g);
  return check_launch(fn);
}

}  // namespace tpf

// Weight gradient of a linear layer over many rows: dW[m][n] = sum_r dy[r][m] x[r][n]
// (dy [R][M] and x [R][N] row-major bf16, both read MN-contiguous), split over
// R with f32 partials and the fixed-order fold (deterministic).  The shape
// of every projection weight gradient of the pair stack (K = B*N^2 rows).
// The split count fills one round of 512 workgroups (two per CU on 256 CUs)
// without spilling into a second: a launch of 515 for 5 output tiles ran
// its last 3 workgroups as a round of their own, doubling the time.  At
// most 256 splits: a one-tile product gains nothing from 512 (its fold of
// twice the partials cost more, 9 -> 25 us at 128 x 128).  The count depends
// on the shape only (fixed fold order on every device).
static int wgrad_splits(int64_t R, int64_t M, int64_t N) {
  const int64_t tiles = ((M + tpf::kGM - 1) / tpf::kGM) * ((N + tpf::kGN - 1) / tpf::kGN);
  int64_t s = 512 / tiles;
  if (s > R / 256) s = R / 256;
  if (s > 256) s = 256;
  if (s < 1) s = 1;
  return (int)s;
}

extern "C" int64_t tpf_wgrad_bf16_workspace_bytes(int64_t R, int64_t M, int64_t N) {
  return (int64_t)wgrad_splits(R, M, N) * M * N * 4;
}

extern "C" int tpf_wgrad_bf16(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x,
                              int64_t R, int64_t M, int64_t N, float* dw, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* fn = "tpf_wgrad_bf16";
  if (!dy || !x || !dw || !workspace) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (R < 1 || M < 1 || N < 1 || R > INT32_MAX || M > INT32_MAX || N > INT32_MAX)
    return tpf::set_error(TPF_ERR_SHAPE, "%s: bad shape", fn);
  if (workspace_bytes < tpf_wgrad_bf16_workspace_bytes(R, M, N))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  const int splits = wgrad_splits(R, M, N);
  tpf::GemmArgs g{};
  g.A = (const __bf16*)dy; g.a_ld = ld_dy; g.a_bs = 0;
  g.B = (const __bf16*)x; g.b_ld = ld_x; g.b_bs = 0;
  g.C = workspace; g.c_ld = N; g.c_bs = 0; g.c_split = M * N;
  g.M = (int)M; g.N = (int)N; g.K = (int)R; g.ksplit = splits;
  g.k_chunk = (int)((R + splits - 1) / splits); g.alpha = 1.f;
  hipStream_t s = (hipStream_t)stream;
  int rc = tpf::gemm_launch_wgrad(g, s, fn);
  if (rc) return rc;
  return tpf::fold_launch((const float*)workspace, dw, M * N, M * N, splits, s, fn);
}

// y [M, N] = a [M, K] b^T (b [N, K], b_kc = 1) or a b (b [K, N]) of contiguous BF16
// rows, f32 sums rounded once.  More than one tile of columns runs on 64-deep k-steps:
// 84 us against the 32-deep 101 at 8192 x 1024 -> 4096, 76 against 83 the other way
// (818 and 900 TFLOP/s).  One tile of columns is a stream of a, which the 32-deep
// shape keeps more stages of in flight: 49 us against 55 at 147456 x 512 -> 128.  The
// weight-stationary row kernel takes the shapes that it has, as in tpf_gemm_bf16.
// No choice depends on M, and all sum in the same order.
extern "C" int tpf_row_gemm_bf16(const void* a, int64_t a_ld, const void* b, int b_kc, void* y,
                                 int64_t M, int64_t N, int64_t K, void* stream) {
  const char* fn = "tpf_row_gemm_bf16";
  if (!a || !b || !y) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (M < 1 || N < 1 || K < 1 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
    return tpf::set_error(TPF_ERR_SHAPE, "%s: bad shape", fn);
  const int64_t b_ld = b_kc ? K : N;
  hipStream_t s = (hipStream_t)stream;
  int rc = TPF_OK;
  if (tpf::rowgemm_try((const __bf16*)a, a_ld, (const __bf16*)b, b_kc, b_ld, (__bf16*)y, N, M, N, K, s,
                       &rc, fn))
    return rc;
  tpf::GemmArgs g{};
  g.A = (const __bf16*)a; g.a_ld = a_ld;
  g.B = (const __bf16*)b; g.b_ld = b_ld;
  g.C = y; g.c_ld = N;
  g.M = (int)M; g.N = (int)N; g.K = (int)K; g.ksplit = 1; g.k_chunk = (int)K; g.alpha = 1.f;
  if (N <= tpf::kGN) return tpf::gemm_launch(g, 1, b_kc ? 1 : 0, 0, 1, s, fn);
  if ((rc = tpf::gemm_prepare(g, 1, b_kc ? 1 : 0, 0, 1, fn))) return rc;
  const dim3 grid((unsigned)((tpf::gemm_tiles(g) + 7) / 8 * 8));
  if (b_kc) hipLaunchKernelGGL((tpf::gemm_bf16_kernel<true, true, false>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((tpf::gemm_bf16_kernel<true, false, false>), grid, dim3(256), 0, s, g);
  return tpf::check_launch(fn);
}
