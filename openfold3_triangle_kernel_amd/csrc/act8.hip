// Activations in 8 bits (act8.hpp): packing and unpacking of rows, and the
// weight gradient of a linear layer whose input is kept that way.
#define TPF_GEMM_GK 64
#define TPF_GEMM_NS 2
#include "act8.hpp"
#include "gemm_core.hpp"
#include "tpf_gemm.hpp"
#include "tpf_status.hpp"

namespace tpf {

// Chunks of eight channels, numbered through the padded rows; a thread handles
// U of them, 256 apart.  The workgroup's first chunk is split into row and
// chunk on the scalar side, the threads' offsets by 32-bit arithmetic.
struct ActArgs {
  const void* src;
  void* dst;
  int64_t ld;  // elements between the rows of the unpacked side
  int64_t R;
  int C, pitch;
  FastDiv chunks;  // pitch / 8
  uint8_t *codes, *scales;
};

template <int DT, bool PACK>
__global__ __launch_bounds__(256) void act8_kernel(ActArgs a) {
  constexpr int U = 2, EB = act_bytes<DT>();
  const int64_t first = (int64_t)blockIdx.x * (256 * U);
  const int64_t row0 = first / a.chunks.d;
  const uint32_t rem = (uint32_t)(first - row0 * a.chunks.d);
  Raw8<DT> raw[U];
  u32x2 code[U];
  uint32_t scale[U];
  int64_t row[U];
  int c[U], n[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = rem + 256 * u + threadIdx.x, q = fdiv(i, a.chunks);
    row[u] = row0 + q;
    c[u] = 8 * (int)(i - q * a.chunks.d);
    n[u] = row[u] < a.R ? min(8, max(0, a.C - c[u])) : 0;
    if (PACK) {
      if (n[u] > 0) raw[u] = load8<DT>((const char*)a.src + (row[u] * a.ld + c[u]) * EB, n[u]);
    } else if (n[u] > 0) {
      code[u] = *reinterpret_cast<const u32x2*>(a.codes + row[u] * a.pitch + c[u]);
      scale[u] = a.scales[row[u] * (a.pitch / kActBlock) + c[u] / kActBlock];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[8] = {};
    if (PACK) {
      if (n[u] > 0) {
        to_f32<DT>(raw[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= n[u]) f[i] = 0.f;
      }
      const u32x2 b = encode8<DT == 1 ? kActTopF16 : kActTop>(f, scale[u]);
      if (row[u] < a.R) {
        *reinterpret_cast<u32x2*>(a.codes + row[u] * a.pitch + c[u]) = b;
        if ((threadIdx.x & 3) == 0)
          a.scales[row[u] * (a.pitch / kActBlock) + c[u] / kActBlock] = (uint8_t)scale[u];
      }
    } else if (n[u] > 0) {
      decode8(code[u], scale[u], f);
      store8<DT>((char*)a.dst + (row[u] * a.ld + c[u]) * EB, f, n[u]);
    }
  }
}

template <bool PACK>
static int act8_launch(ActArgs a, int64_t dt, hipStream_t s, const char* fn) {
  const int64_t n = (a.R * a.chunks.d + 511) / 512;
  if (n >= (int64_t)1 << 24)  // 2^32 threads
    return set_error(TPF_ERR_SHAPE, "%s: too many values", fn);
  const dim3 grid((unsigned)n), block(256);
  if (dt == TPF_BF16) hipLaunchKernelGGL((act8_kernel<0, PACK>), grid, block, 0, s, a);
  else if (dt == TPF_F16) hipLaunchKernelGGL((act8_kernel<1, PACK>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((act8_kernel<2, PACK>), grid, block, 0, s, a);
  return check_launch(fn);
}

static int act8_check(ActArgs& a, const void* plain, int64_t ld, int64_t R, int64_t C, int64_t dt,
                      const void* codes, const void* scales, const char* fn) {
  if (!plain || !codes || !scales) return set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (R < 1 || C < 1 || C > (1 << 24) || R > ((int64_t)1 << 40) || ld < 0)
    return set_error(TPF_ERR_SHAPE, "%s: bad shape R=%lld C=%lld", fn, (long long)R, (long long)C);
  if (dt < 0 || dt > 2) return set_error(TPF_ERR_ARG, "%s: unknown type", fn);
  if ((uintptr_t)codes % 8) return set_error(TPF_ERR_ARG, "%s: codes must start on 8 bytes", fn);
  a.ld = ld; a.R = R; a.C = (int)C; a.pitch = (int)((C + 31) / 32 * 32);
  a.chunks = make_fastdiv((uint32_t)a.pitch / 8);
  a.codes = (uint8_t*)const_cast<void*>(codes);
  a.scales = (uint8_t*)const_cast<void*>(scales);
  return TPF_OK;
}

// dW[n][k] = sum_r dy[r][n] x~[r][k]: 128 x 128 tiles over 64 rows a step (the
// layouts of gemm_core.hpp, both operands read transposed from LDS).  dy goes
// into LDS directly; the codes come through registers, one step ahead, and are
// decoded once per tile on their way: a thread decodes one block of 32 (one
// scale), and every decoded value is exact in BF16.  8192 x 1024 -> 4096: 103 us (670
// TFLOP/s), as long as torch's product of the same BF16 operands takes; 256-wide
// tiles of eight waves, 128 x 64 a wave, and decoding between the products measured
// 102 to 114 us and were not kept.
struct Wgrad8Args {
  const __bf16* dy;
  int64_t ld;
  const uint8_t *codes, *scales;
  int64_t R;
  int N, K, pitch, splits, chunk;  // rows of a split, a multiple of 64
  float* part;                     // [splits][N][K] f32, null when unsplit
  void* dw;
  int out_f32;
};

__global__ __launch_bounds__(256, 2) void wgrad8_kernel(Wgrad8Args a) {
  constexpr int TM = 128, NB = 2;
  __shared__ __attribute__((aligned(1024))) char smem[2][2][kGTileBytes];
  const int tn = (a.N + TM - 1) / TM, tk = (a.K + TM - 1) / TM;
  const int64_t T = xcd_order((int64_t)tn * tk * a.splits);
  if (T < 0) return;
  const int nt = (int)(T % tn);
  const int64_t u = T / tn;
  const int kt_ = (int)(u % tk), split = (int)(u / tk);
  const int n0 = nt * TM, k0 = kt_ * TM;
  const int64_t rbeg = (int64_t)split * a.chunk;
  const int rows = (int)min((int64_t)a.chunk, a.R - rbeg);
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = w >> 1, wn = w & 1;

  f32x16 acc[NB][NB];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = zero16();

  TileLoader<false> la;
  la.init(GemmOperand{a.dy + rbeg * a.ld, a.ld, a.N}, n0);
  // This thread's block of the codes' tile: row tid / 4, columns 32 (tid % 4).
  const int br = threadIdx.x >> 2, bc = 32 * (threadIdx.x & 3);
  const bool bin = k0 + bc < a.pitch;
  const uint8_t* cp = a.codes + (rbeg + br) * a.pitch + k0 + bc;
  const uint8_t* sp = a.scales + (rbeg + br) * (a.pitch / kActBlock) + (k0 + bc) / kActBlock;
  u32x4 code[2];
  uint32_t scale;
  auto fetch = [&](int r) {  // rows r .. r + 63 of the split
    const bool in = bin && r + br < rows;
    code[0] = code[1] = (u32x4)0x80808080u;
    scale = 127u;
    if (in) {
      code[0] = *reinterpret_cast<const u32x4*>(cp + (int64_t)r * a.pitch);
      code[1] = *reinterpret_cast<const u32x4*>(cp + (int64_t)r * a.pitch + 16);
      scale = sp[(int64_t)r * (a.pitch / kActBlock)];
    }
  };
  auto decode = [&](char* tile) {
    __bf16* B = reinterpret_cast<__bf16*>(tile);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[8];
      u32x2 b;
      b[0] = code[j >> 1][2 * (j & 1)];
      b[1] = code[j >> 1][2 * (j & 1) + 1];
      decode8(b, scale, f);
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = f2bf(f[e]);
      const int slot = ((bc >> 3) + j) ^ ((br & 3) << 1);
      *reinterpret_cast<bf16x8*>(B + br * TM + slot * 8) = v;
    }
  };

  fetch(0);
  la.issue(0, rows, smem[0][0]);
  decode(smem[0][1]);
  fetch(kGK);
  int st = 0;
  for (int r = 0; r < rows; r += kGK, st ^= 1) {
    wait_vmcnt<0>();
    lds_barrier();
    if (r + kGK < rows) {
      la.issue(r + kGK, rows, smem[st ^ 1][0]);
      decode(smem[st ^ 1][1]);
      fetch(r + 2 * kGK);
    }
    const __bf16* As = reinterpret_cast<const __bf16*>(smem[st][0]);
    const __bf16* Bs = reinterpret_cast<const __bf16*>(smem[st][1]);
#pragma unroll
    for (int s = 0; s < kGK / 16; ++s) {
      bf16x8 af[NB], bf[NB];
#pragma unroll
      for (int t = 0; t < NB; ++t) {
        af[t] = tile_frag<false>(As, 64 * wm + 32 * t, s);
        bf[t] = tile_frag<false>(Bs, 64 * wn + 32 * t, s);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma32(af[i], bf[j], acc[i][j]);
    }
  }
  const int rl = lane & 31, hl = lane >> 5;
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int col = k0 + 64 * wn + 32 * j + rl;
      if (col >= a.K) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int row = n0 + 64 * wm + 32 * i + 8 * (e >> 2) + 4 * hl + (e & 3);
        if (row >= a.N) continue;
        const int64_t at = (int64_t)row * a.K + col;
        if (a.part) a.part[(int64_t)split * a.N * a.K + at] = acc[i][j][e];
        else if (a.out_f32) reinterpret_cast<float*>(a.dw)[at] = acc[i][j][e];
        else reinterpret_cast<__bf16*>(a.dw)[at] = f2bf(acc[i][j][e]);
      }
    }
}

// Sums the splits, four values a thread: RANGES threads share them, each a range in
// ascending order, and the ranges join in order.  Eight ranges where there are many
// splits, which have few values (128 of 512 x 128: 7.8 us with one range).
template <int RANGES>
__global__ __launch_bounds__(256) void wgrad8_fold_kernel(const float* part, int64_t n, int splits,
                                                          void* dw, int out_f32) {
  constexpr int G = 256 / RANGES;
  __shared__ f32x4 red[RANGES][G];
  const int g = threadIdx.x % G, q = threadIdx.x / G;
  const int64_t i = 4 * ((int64_t)blockIdx.x * G + g);
  const bool in = i < n;  // n is a multiple of 64
  const int per = (splits + RANGES - 1) / RANGES, p1 = min(splits, (q + 1) * per);
  f32x4 s = (f32x4)0.f;
  int p = q * per;
  if (in) {
    for (; p + 8 <= p1; p += 8) {
      f32x4 v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ld4f_nt(part + (int64_t)(p + e) * n + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; p < p1; ++p) s += ld4f_nt(part + (int64_t)p * n + i);
  }
  if constexpr (RANGES > 1) {
    red[q][g] = s;
    __syncthreads();
    if (q) return;
#pragma unroll
    for (int e = 1; e < RANGES; ++e) s += red[e][g];
  }
  if (!in) return;
  if (out_f32) {
    *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(dw) + i) = s;
  } else {
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f2bf(s[e]);
    *reinterpret_cast<bf16x4*>(reinterpret_cast<__bf16*>(dw) + i) = o;
  }
}

// Row splits: one round of 512 workgroups (two a CU), 256 rows a split at
// least, and few enough rows that a split's dy lies within 32-bit offsets.
static int wgrad8_plan(Wgrad8Args& a) {
  const int64_t tiles = (int64_t)((a.N + 127) / 128) * ((a.K + 127) / 128);
  int64_t s = 512 / tiles;
  if (s > a.R / 256) s = a.R / 256;
  if (s > 256) s = 256;
  if (s < 1) s = 1;
  const int64_t span = ((int64_t)kBufOOB - 1) / (2 * a.ld) / 64 * 64;  // rows below 2 GiB
  if (span < 64) return 0;
  int64_t chunk = ((a.R + s - 1) / s + 63) / 64 * 64;
  if (chunk > span) chunk = span;
  if ((a.R + chunk - 1) / chunk > 65536) return 0;
  a.chunk = (int)chunk;
  a.splits = (int)((a.R + chunk - 1) / chunk);
  return 1;
}

}  // namespace tpf

extern "C" int tpf_act8_pack(const void* x, int64_t ld, int64_t R, int64_t C, int64_t dtype,
                             void* codes, void* scales, void* stream) {
  const char* fn = "tpf_act8_pack";
  tpf::ActArgs a{};
  if (int rc = tpf::act8_check(a, x, ld, R, C, dtype, codes, scales, fn)) return rc;
  a.src = x;
  return tpf::act8_launch<true>(a, dtype, (hipStream_t)stream, fn);
}

extern "C" int tpf_act8_unpack(const void* codes, const void* scales, int64_t R, int64_t C, void* x,
                               int64_t ld, int64_t dtype, void* stream) {
  const char* fn = "tpf_act8_unpack";
  tpf::ActArgs a{};
  if (int rc = tpf::act8_check(a, x, ld, R, C, dtype, codes, scales, fn)) return rc;
  a.dst = x;
  return tpf::act8_launch<false>(a, dtype, (hipStream_t)stream, fn);
}

static int wgrad8_args(tpf::Wgrad8Args& a, int64_t R, int64_t N, int64_t K, int64_t ld,
                       const char* fn) {
  if (R < 1 || N < 8 || K < 8 || N % 8 || K % 8 || N > (1 << 24) || K > (1 << 24) || ld < N || ld % 8)
    return tpf::set_error(TPF_ERR_SHAPE, "%s: bad shape R=%lld N=%lld K=%lld", fn, (long long)R,
                          (long long)N, (long long)K);
  a.R = R; a.N = (int)N; a.K = (int)K; a.ld = ld; a.pitch = (int)((K + 31) / 32 * 32);
  if (!tpf::wgrad8_plan(a)) return tpf::set_error(TPF_ERR_SHAPE, "%s: too many rows", fn);
  return TPF_OK;
}

extern "C" int64_t tpf_wgrad_act8_workspace_bytes(int64_t R, int64_t N, int64_t K, int64_t ld_dy) {
  tpf::Wgrad8Args a{};
  if (wgrad8_args(a, R, N, K, ld_dy, "tpf_wgrad_act8_workspace_bytes")) return -1;
  return a.splits > 1 ? (int64_t)a.splits * N * K * 4 : 0;
}

extern "C" int tpf_wgrad_act8(const void* dy, int64_t ld_dy, const void* codes, const void* scales,
                              int64_t R, int64_t N, int64_t K, void* dw, int64_t dw_dtype,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "tpf_wgrad_act8";
  if (!dy || !codes || !scales || !dw) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  tpf::Wgrad8Args a{};
  if (int rc = wgrad8_args(a, R, N, K, ld_dy, fn)) return rc;
  if (dw_dtype != TPF_BF16 && dw_dtype != TPF_F32)
    return tpf::set_error(TPF_ERR_ARG, "%s: the gradient is BF16 or FP32", fn);
  if (((uintptr_t)dy | (uintptr_t)codes | (uintptr_t)dw | (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  if (a.splits > 1 && (!workspace || workspace_bytes < (int64_t)a.splits * N * K * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.dy = (const __bf16*)dy; a.codes = (const uint8_t*)codes; a.scales = (const uint8_t*)scales;
  a.part = a.splits > 1 ? (float*)workspace : nullptr;
  a.dw = dw; a.out_f32 = dw_dtype == TPF_F32;
  hipStream_t s = (hipStream_t)stream;
  const int64_t tiles = ((N + 127) / 128) * ((K + 127) / 128) * a.splits;
  if ((tiles + 7) / 8 * 8 > INT32_MAX) return tpf::set_error(TPF_ERR_SHAPE, "%s: too large", fn);
  hipLaunchKernelGGL(tpf::wgrad8_kernel, dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(256), 0, s, a);
  if (a.part) {
    const int64_t n = N * K;
    if (a.splits >= 32)
      hipLaunchKernelGGL(tpf::wgrad8_fold_kernel<8>, dim3((unsigned)((n / 4 + 31) / 32)), dim3(256), 0,
                         s, a.part, n, a.splits, dw, a.out_f32);
    else
      hipLaunchKernelGGL(tpf::wgrad8_fold_kernel<1>, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256),
                         0, s, a.part, n, a.splits, dw, a.out_f32);
  }
  return tpf::check_launch(fn);
}
