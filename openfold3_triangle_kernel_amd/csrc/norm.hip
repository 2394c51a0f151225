// Layer norm over rows of any channel count, in BF16, FP16 or FP32, with
// statistics and parameters in 32 bits; forward, and the backward with the
// parameters' gradients.
//
//   xh = (x - mean) rstd,  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum dy xh,  db = sum dy
//
// The bound is the rows' bytes, each read and written once: 2 passes forward, 3
// backward.  TPR threads share a row and hold it in registers, K chunks of
// eight channels each (chunk k TPR + t), so the variance is formed from the
// differences to the mean without a second read.  Rows wider than 1024 threads
// hold are read again from the caches (the wide kernels).  A workgroup walks
// over rows, the next row's loads in flight, with the parameters and the
// backward's column sums in registers; column sums of the workgroups are folded
// in a fixed order.  16384 x 4096 BF16: forward 60 us, backward 84 and 7 for the fold
// (4.5 and 4.8 TB/s; a large copy reaches 4.9); 147456 x 128 forward and backward 42.
//
// 8-bit form: the forward can write xh as act8.hpp holds it, 33/32 byte a
// channel, and the backward reads that in place of the rows.
#include "act8.hpp"
#include "tpf_status.hpp"

namespace tpf {

struct NormArgs {
  const void* x;
  int64_t x_ld;  // elements between rows of x
  int64_t R;
  int C;
  const void *w, *b;  // parameters, null for 1 and 0
  int pdt;            // their type
  float eps;
  void* y;
  float *mean, *rstd;      // null when no backward follows (mean also with codes)
  uint8_t *codes, *scales;  // the 8-bit form of xh [R][pitch], [R][pitch / 32]
  int pitch;
  // backward
  const void* dy;
  void* dx;      // rows at dx_ld
  int64_t dx_ld;
  float* part;   // [workgroups][2][C]
};

// A parameter's eight channels (`fill` past the end or where there is none).
__device__ __forceinline__ void param8(const void* p, int pdt, int c, int C, float fill,
                                       float (&f)[8]) {
  const int n = min(8, C - c);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fill;
  if (!p || n <= 0) return;
  if (pdt == 2) to_f32<2>(load8<2>((const char*)p + (int64_t)c * 4, n), f);
  else if (pdt == 0) to_f32<0>(load8<0>((const char*)p + (int64_t)c * 2, n), f);
  else to_f32<1>(load8<1>((const char*)p + (int64_t)c * 2, n), f);
}

// Sums of N values over the threads of a row; every thread gets the same bits.
// `turn` alternates between calls, so one barrier a call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int turn) {
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[n]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    __shared__ float red[2][N][W];
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) red[turn][n][w] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float s = red[turn][n][0];
#pragma unroll
      for (int i = 1; i < W; ++i) s += red[turn][n][i];
      v[n] = s;
    }
  }
}

template <int DT, int TPR, int K, bool CODES>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(NormArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, EB = act_bytes<DT>();
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  float w[K][8], b[K][8];
  int n[K];  // channels of the chunk inside the row
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 8 * (k * TPR + t);
    n[k] = min(8, max(0, a.C - c));
    param8(a.w, a.pdt, c, a.C, 1.f, w[k]);
    param8(a.b, a.pdt, c, a.C, 0.f, b[k]);
  }
  const float inv_c = 1.f / (float)a.C;
  const int64_t step = (int64_t)gridDim.x * RPB;
  Raw8<DT> raw[K];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (r < a.R && n[k] > 0)
        raw[k] = load8<DT>((const char*)a.x + (r * a.x_ld + 8 * (k * TPR + t)) * EB, n[k]);
  };
  int64_t r = (int64_t)blockIdx.x * RPB + slot;
  load(r);
  // Threads of one workgroup run the same number of turns: rows past the end
  // are computed on what their registers hold and not written.
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.R; base += step, r += step) {
    float x[K][8], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (n[k] > 0 && r < a.R) to_f32<DT>(raw[k], x[k]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += x[k][i];
    }
    load(r + step);
    row_sum<TPR, 1>(s, 0);
    const float mean = s[0] / (float)a.C;  // divided: exact where the sum is
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] = i < n[k] ? x[k][i] - mean : 0.f;
        s[0] = fmaf(x[k][i], x[k][i], s[0]);
      }
    row_sum<TPR, 1>(s, 1);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv_c, a.eps));
    if (r >= a.R) continue;
    if (t == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = 8 * (k * TPR + t);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] *= rstd;
        y[i] = fmaf(x[k][i], w[k][i], b[k][i]);
      }
      if (n[k] > 0) store8<DT>((char*)a.y + (r * a.C + c) * EB, y, n[k]);
      if constexpr (CODES) {
        uint32_t scale;
        const u32x2 code = encode8(x[k], scale);
        if (c < a.pitch) {
          *reinterpret_cast<u32x2*>(a.codes + r * a.pitch + c) = code;
          if ((t & 3) == 0) a.scales[r * (a.pitch / kActBlock) + c / kActBlock] = (uint8_t)scale;
        }
      }
    }
  }
}

// The row's dx, and the column sums over the workgroup's rows.
template <int DT, int TPR, int K, bool CODES>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_bwd_kernel(NormArgs a) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR, EB = act_bytes<DT>();
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  float w[K][8], dw[K][8], db[K][8];
  int n[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 8 * (k * TPR + t);
    n[k] = min(8, max(0, a.C - c));
    param8(a.w, a.pdt, c, a.C, 1.f, w[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[k][i] = db[k][i] = 0.f;
  }
  const float inv_c = 1.f / (float)a.C;
  const int64_t step = (int64_t)gridDim.x * RPB;
  Raw8<DT> rx[K], rg[K];
  u32x2 rc[K];
  uint32_t rs[K];
  float mean_n = 0.f, rstd_n = 0.f;
  auto load = [&](int64_t r) {
    if (r >= a.R) return;
    if constexpr (!CODES) mean_n = a.mean[r];
    rstd_n = a.rstd[r];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (n[k] > 0) {
        const int c = 8 * (k * TPR + t);
        rg[k] = load8<DT>((const char*)a.dy + (r * a.C + c) * EB, n[k]);
        if constexpr (CODES) {
          rc[k] = *reinterpret_cast<const u32x2*>(a.codes + r * a.pitch + c);
          rs[k] = a.scales[r * (a.pitch / kActBlock) + c / kActBlock];
        } else {
          rx[k] = load8<DT>((const char*)a.x + (r * a.x_ld + c) * EB, n[k]);
        }
      }
  };
  int64_t r = (int64_t)blockIdx.x * RPB + slot;
  load(r);
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < a.R; base += step, r += step, turn ^= 1) {
    float x[K][8], g[K][8], s[2] = {0.f, 0.f};
    const float mean = mean_n, rstd = rstd_n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (n[k] > 0 && r < a.R) {
        to_f32<DT>(rg[k], g[k]);
        if constexpr (CODES) decode8(rc[k], rs[k], x[k]);
        else to_f32<DT>(rx[k], x[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (!CODES) x[k][i] = (x[k][i] - mean) * rstd;
          if (i >= n[k]) x[k][i] = g[k][i] = 0.f;
          dw[k][i] = fmaf(g[k][i], x[k][i], dw[k][i]);
          db[k][i] += g[k][i];
          g[k][i] *= w[k][i];
          s[0] += g[k][i];
          s[1] = fmaf(g[k][i], x[k][i], s[1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = g[k][i] = 0.f;
      }
    }
    load(r + step);
    row_sum<TPR, 2>(s, turn);
    if (r >= a.R) continue;
    const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (n[k] <= 0) continue;
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = rstd * (g[k][i] - m0 - x[k][i] * m1);
      store8<DT>((char*)a.dx + (r * a.dx_ld + 8 * (k * TPR + t)) * EB, d, n[k]);
    }
  }
  if (!a.part) return;
  // Column sums of the RPB rows that a workgroup works on at a time, in slot
  // order.
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n[k]) {
          part[8 * (k * TPR + t) + i] = dw[k][i];
          part[a.C + 8 * (k * TPR + t) + i] = db[k][i];
        }
  } else {
    constexpr int W = 8 * K * TPR;
    __shared__ float cols[RPB][W];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          cols[slot][8 * (k * TPR + t) + i] = which ? db[k][i] : dw[k][i];
      __syncthreads();
      for (int c = threadIdx.x; c < W && c < a.C; c += NT) {
        float s = cols[0][c];
#pragma unroll
        for (int q = 1; q < RPB; ++q) s += cols[q][c];
        part[which * a.C + c] = s;
      }
    }
  }
}

// Rows wider than the kernels above hold: one workgroup of 1024 threads a row,
// the row read again from the caches for each pass.
template <int DT, bool CODES>
__global__ __launch_bounds__(1024) void norm_fwd_wide_kernel(NormArgs a) {
  constexpr int EB = act_bytes<DT>();
  const int chunks = (a.C + 31) / 32 * 4;  // whole blocks
  const float inv_c = 1.f / (float)a.C;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const char* x = (const char*)a.x + r * a.x_ld * EB;
    float s[1] = {0.f}, f[8];
    for (int j = threadIdx.x; 8 * j < a.C; j += 1024) {
      to_f32<DT>(load8<DT>(x + 8 * j * EB, min(8, a.C - 8 * j)), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += f[i];
    }
    row_sum<1024, 1>(s, 0);
    const float mean = s[0] / (float)a.C;  // divided: exact where the sum is
    s[0] = 0.f;
    for (int j = threadIdx.x; 8 * j < a.C; j += 1024) {
      to_f32<DT>(load8<DT>(x + 8 * j * EB, min(8, a.C - 8 * j)), f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8 * j + i < a.C) s[0] = fmaf(f[i] - mean, f[i] - mean, s[0]);
    }
    row_sum<1024, 1>(s, 1);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv_c, a.eps));
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
    for (int j = threadIdx.x; j < chunks; j += 1024) {  // whole groups of four lanes
      const int c = 8 * j, n = min(8, max(0, a.C - c));
      float w[8], b[8], y[8];
      if (n > 0) to_f32<DT>(load8<DT>(x + c * EB, n), f);
      param8(a.w, a.pdt, c, a.C, 1.f, w);
      param8(a.b, a.pdt, c, a.C, 0.f, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = i < n ? (f[i] - mean) * rstd : 0.f;
        y[i] = fmaf(f[i], w[i], b[i]);
      }
      if (n > 0) store8<DT>((char*)a.y + (r * a.C + c) * EB, y, n);
      if constexpr (CODES) {
        uint32_t scale;
        const u32x2 code = encode8(f, scale);
        *reinterpret_cast<u32x2*>(a.codes + r * a.pitch + c) = code;
        if ((j & 3) == 0) a.scales[r * (a.pitch / kActBlock) + c / kActBlock] = (uint8_t)scale;
      }
    }
  }
}

// dx of wide rows; the column sums are norm_cols_kernel's.
template <int DT, bool CODES>
__global__ __launch_bounds__(1024) void norm_bwd_wide_kernel(NormArgs a) {
  constexpr int EB = act_bytes<DT>();
  const float inv_c = 1.f / (float)a.C;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x, turn ^= 1) {
    const float mean = CODES ? 0.f : a.mean[r], rstd = a.rstd[r];
    auto load = [&](int c, int n, float (&x)[8], float (&g)[8]) {
      float w[8];
      to_f32<DT>(load8<DT>((const char*)a.dy + (r * a.C + c) * EB, n), g);
      if constexpr (CODES) {
        decode8(*reinterpret_cast<const u32x2*>(a.codes + r * a.pitch + c),
                a.scales[r * (a.pitch / kActBlock) + c / kActBlock], x);
      } else {
        to_f32<DT>(load8<DT>((const char*)a.x + (r * a.x_ld + c) * EB, n), x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (x[i] - mean) * rstd;
      }
      param8(a.w, a.pdt, c, a.C, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        g[i] = i < n ? g[i] * w[i] : 0.f;
        x[i] = i < n ? x[i] : 0.f;
      }
    };
    float s[2] = {0.f, 0.f}, x[8], g[8];
    for (int c = 8 * threadIdx.x; c < a.C; c += 8192) {
      load(c, min(8, a.C - c), x, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[0] += g[i];
        s[1] = fmaf(g[i], x[i], s[1]);
      }
    }
    row_sum<1024, 2>(s, turn);
    const float m0 = s[0] * inv_c, m1 = s[1] * inv_c;
    for (int c = 8 * threadIdx.x; c < a.C; c += 8192) {
      const int n = min(8, a.C - c);
      load(c, n, x, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = rstd * (g[i] - m0 - x[i] * m1);
      store8<DT>((char*)a.dx + (r * a.dx_ld + c) * EB, g, n);
    }
  }
}

// Column sums of wide rows: a thread owns eight channels, a workgroup 2048 of
// them and every gridDim.y-th row.
template <int DT, bool CODES>
__global__ __launch_bounds__(256) void norm_cols_kernel(NormArgs a) {
  constexpr int EB = act_bytes<DT>();
  const int c = 8 * (blockIdx.x * 256 + threadIdx.x), n = min(8, a.C - c);
  if (n <= 0) return;
  float dw[8] = {}, db[8] = {};
  for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
    float x[8], g[8];
    to_f32<DT>(load8<DT>((const char*)a.dy + (r * a.C + c) * EB, n), g);
    if constexpr (CODES) {
      decode8(*reinterpret_cast<const u32x2*>(a.codes + r * a.pitch + c),
              a.scales[r * (a.pitch / kActBlock) + c / kActBlock], x);
    } else {
      const float mean = a.mean[r], rstd = a.rstd[r];
      to_f32<DT>(load8<DT>((const char*)a.x + (r * a.x_ld + c) * EB, n), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (x[i] - mean) * rstd;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[i] = fmaf(g[i], x[i], dw[i]);
      db[i] += g[i];
    }
  }
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.C + c;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      part[i] = dw[i];
      part[a.C + i] = db[i];
    }
}

// Folds the workgroups' column sums in ascending order within 16 ranges, then
// the ranges; a workgroup forms 16 of the 2 C columns.
__global__ __launch_bounds__(256) void norm_fold_kernel(const float* part, int groups, int C, void* dw,
                                                        void* db, int pdt) {
  __shared__ float red[16][17];
  const int col = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t i = (int64_t)blockIdx.x * 16 + col;
  const int per = (groups + 15) / 16, g0 = q * per, g1 = min(groups, g0 + per);
  float s = 0.f;
  if (i < 2 * (int64_t)C) {
    int g = g0;
    for (; g + 8 <= g1; g += 8) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = part[(int64_t)(g + e) * 2 * C + i];
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; g < g1; ++g) s += part[(int64_t)g * 2 * C + i];
  }
  red[q][col] = s;
  __syncthreads();
  if (q || i >= 2 * (int64_t)C) return;
#pragma unroll
  for (int e = 1; e < 16; ++e) s += red[e][col];
  void* dst = i < C ? dw : db;
  const int64_t c = i < C ? i : i - C;
  if (!dst) return;
  if (pdt == 2) reinterpret_cast<float*>(dst)[c] = s;
  else if (pdt == 0) reinterpret_cast<__bf16*>(dst)[c] = f2bf(s);
  else reinterpret_cast<_Float16*>(dst)[c] = (_Float16)s;
}

// Threads a row and chunks a thread of a width.  One chunk a thread up to 128
// channels (147456 x 128 training 42 us, 44 with two), two in a wave up to 1024, where
// more rows of a workgroup are worth as much as more threads a row; a workgroup a row
// beyond; k = 0 above 8192 channels, the wide kernels.
struct NormShape {
  int tpr, k;
};
static NormShape norm_shape(int C) {
  const int chunks = (C + 31) / 32 * 4;  // whole blocks of the 8-bit form
  for (int tpr : {8, 16})
    if (chunks <= tpr) return {tpr, 1};
  for (int tpr : {16, 32, 64})
    if (chunks <= 2 * tpr) return {tpr, 2};
  for (int k : {1, 2})
    if (chunks <= 256 * k) return {256, k};
  if (chunks <= 1024) return {1024, 1};
  return {1024, 0};
}

// Workgroups of the backward, and partials to fold: as many as keep a CU's loads in
// flight with the registers that they hold, four a CU with one chunk a thread, two
// with two (10007 x 1531 FP32 training: 82 us at 1024, 93 at 512; 16384 x 4096 BF16,
// two chunks: 150 at 512, 167 at 1024).
static int norm_groups(int64_t R, int C) {
  const NormShape s = norm_shape(C);
  const int rpb = s.tpr >= 256 || !s.k ? 1 : 256 / s.tpr;
  const int64_t most = !s.k ? 64 : s.tpr > 256 ? 256 : s.tpr > 64 ? 1024 / s.k : 1024;
  const int64_t need = (R + rpb - 1) / rpb;
  return (int)(need < most ? need : most);
}

template <int DT, bool CODES, bool BWD>
static void norm_launch(const NormArgs& a, int groups, hipStream_t s) {
  const NormShape sh = norm_shape(a.C);
#define TPF_NORM(TPR, K)                                                                         \
  if (sh.tpr == TPR && sh.k == K) {                                                              \
    constexpr int RPB = TPR >= 256 ? 1 : 256 / TPR;                                              \
    if constexpr (BWD) {                                                                         \
      hipLaunchKernelGGL((norm_bwd_kernel<DT, TPR, K, CODES>), dim3((unsigned)groups),           \
                         dim3(TPR > 256 ? TPR : 256), 0, s, a);                                  \
    } else {                                                                                     \
      int64_t g = (a.R + RPB - 1) / RPB;                                                         \
      if (g > 2048) g = 2048;                                                                    \
      hipLaunchKernelGGL((norm_fwd_kernel<DT, TPR, K, CODES>), dim3((unsigned)g),                \
                         dim3(TPR > 256 ? TPR : 256), 0, s, a);                                  \
    }                                                                                            \
    return;                                                                                      \
  }
  TPF_NORM(8, 1) TPF_NORM(16, 1) TPF_NORM(16, 2) TPF_NORM(32, 2) TPF_NORM(64, 2)
  TPF_NORM(256, 1) TPF_NORM(256, 2)
  TPF_NORM(1024, 1)
#undef TPF_NORM
  const unsigned rows = (unsigned)(a.R < 1024 ? a.R : 1024);
  if constexpr (BWD) {
    hipLaunchKernelGGL((norm_bwd_wide_kernel<DT, CODES>), dim3(rows), dim3(1024), 0, s, a);
    if (a.part)
      hipLaunchKernelGGL((norm_cols_kernel<DT, CODES>),
                         dim3((unsigned)((a.C + 2047) / 2048), (unsigned)groups), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((norm_fwd_wide_kernel<DT, CODES>), dim3(rows), dim3(1024), 0, s, a);
  }
}

template <bool BWD>
static void norm_dispatch(const NormArgs& a, int dt, int groups, hipStream_t s) {
  if (a.codes) {
    if (dt == TPF_BF16) norm_launch<0, true, BWD>(a, groups, s);
    else if (dt == TPF_F16) norm_launch<1, true, BWD>(a, groups, s);
    else norm_launch<2, true, BWD>(a, groups, s);
  } else {
    if (dt == TPF_BF16) norm_launch<0, false, BWD>(a, groups, s);
    else if (dt == TPF_F16) norm_launch<1, false, BWD>(a, groups, s);
    else norm_launch<2, false, BWD>(a, groups, s);
  }
}

static int norm_check(int64_t R, int64_t C, int64_t ld, int64_t dt, int64_t pdt, const char* fn) {
  if (R < 1 || C < 1 || C > (1 << 24) || R > ((int64_t)1 << 40) || ld < 0)
    return set_error(TPF_ERR_SHAPE, "%s: bad shape R=%lld C=%lld", fn, (long long)R, (long long)C);
  if (dt < 0 || dt > 2 || pdt < 0 || pdt > 2)
    return set_error(TPF_ERR_ARG, "%s: unknown type", fn);
  return TPF_OK;
}

}  // namespace tpf

extern "C" int tpf_norm_forward(const void* x, int64_t x_ld, int64_t R, int64_t C, int64_t dtype,
                                const void* weight, const void* bias, int64_t param_dtype, double eps,
                                void* y, float* mean, float* rstd, void* codes, void* scales,
                                void* stream) {
  const char* fn = "tpf_norm_forward";
  if (!x || !y) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (int rc = tpf::norm_check(R, C, x_ld, dtype, param_dtype, fn)) return rc;
  if ((codes != nullptr) != (scales != nullptr) || (uintptr_t)codes % 8)
    return tpf::set_error(TPF_ERR_ARG, "%s: codes and scales are both given or both null", fn);
  tpf::NormArgs a{};
  a.x = x; a.x_ld = x_ld; a.R = R; a.C = (int)C; a.w = weight; a.b = bias; a.pdt = (int)param_dtype;
  a.eps = (float)eps; a.y = y; a.mean = mean; a.rstd = rstd;
  a.codes = (uint8_t*)codes; a.scales = (uint8_t*)scales; a.pitch = (int)((C + 31) / 32 * 32);
  tpf::norm_dispatch<false>(a, (int)dtype, 0, (hipStream_t)stream);
  return tpf::check_launch(fn);
}

extern "C" int64_t tpf_norm_backward_workspace_bytes(int64_t R, int64_t C) {
  if (tpf::norm_check(R, C, 0, 0, 0, "tpf_norm_backward_workspace_bytes")) return -1;
  return (int64_t)tpf::norm_groups(R, (int)C) * 2 * C * 4;
}

extern "C" int tpf_norm_backward(const void* dy, const void* x, int64_t x_ld, const void* codes,
                                 const void* scales, const float* mean, const float* rstd, int64_t R,
                                 int64_t C, int64_t dtype, const void* weight, int64_t param_dtype,
                                 void* dx, int64_t dx_ld, void* dweight, void* dbias, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* fn = "tpf_norm_backward";
  if (!dy || !rstd || !dx) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (int rc = tpf::norm_check(R, C, x_ld, dtype, param_dtype, fn)) return rc;
  if ((codes != nullptr) != (scales != nullptr) || (uintptr_t)codes % 8)
    return tpf::set_error(TPF_ERR_ARG, "%s: codes and scales are both given or both null", fn);
  if (!codes && (!x || !mean))
    return tpf::set_error(TPF_ERR_ARG, "%s: either the rows with their means or the codes", fn);
  const bool params = dweight || dbias;
  const int groups = tpf::norm_groups(R, (int)C);
  if (params && (!workspace || workspace_bytes < (int64_t)groups * 2 * C * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  tpf::NormArgs a{};
  a.x = x; a.x_ld = x_ld; a.R = R; a.C = (int)C; a.w = weight; a.pdt = (int)param_dtype;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.codes = (uint8_t*)const_cast<void*>(codes); a.scales = (uint8_t*)const_cast<void*>(scales);
  a.pitch = (int)((C + 31) / 32 * 32);
  a.dy = dy; a.dx = dx; a.dx_ld = dx_ld; a.part = params ? (float*)workspace : nullptr;
  hipStream_t s = (hipStream_t)stream;
  tpf::norm_dispatch<true>(a, (int)dtype, groups, s);
  if (params)
    hipLaunchKernelGGL(tpf::norm_fold_kernel, dim3((unsigned)((2 * C + 15) / 16)), dim3(256), 0, s,
                       a.part, groups, (int)C, dweight, dbias, (int)param_dtype);
  return tpf::check_launch(fn);
}
