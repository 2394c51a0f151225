// Norms of queries and keys for each head with the rotation by position, in one pass;
// its backward; and the same on the way into a paged cache.
//
//   x^ = x / sqrt(mean(x^2) + eps)  (or x),  z = x^ w,  t = position f_c,
//   y_a = z_a cos t - z_b sin t,  y_b = z_b cos t + z_a sin t
//
// over the pairs (a, b) of the first 2 half channels, (c, c + half) or (2 c, 2 c + 1);
// the other channels are y = z.  Backward: dz = R^T dy, dw = sum of dz x^ over the
// rows, g = dz w, dx = (g - x^ mean(g x^)) / sqrt(mean(x^2) + eps).
//
// Bound by memory: a row (a token's head) is read and written once.  A lane owns eight
// pairs (or sixteen channels that only pass), L lanes a row, and a wave takes the heads
// of one token 64 / L at a time, so the angles of a token are formed once, a pair a
// lane, and shared through LDS.  A turn's fraction is formed in 64 bits, position
// times f / 2 pi less the nearest whole number: the angle is within 2^-25 of a turn while position
// times f is below 2^28 radians, where 32 bits would have lost it past a few thousand.  2 x 4096 tokens,
// 32 + 8 heads of 128, BF16: 40 us forward (4.2 TB/s, what a copy reaches is 4.9), 69 backward
// (3.6 TB/s: the weights' sums leave three waves a SIMD).
#include "paged.hpp"
#include "tpf_status.hpp"

namespace tpf {

constexpr int kRotMaxHalf = 128;  // pairs of the widest row

struct RotArgs {
  // Sides: 0 queries, 1 keys, 2 values (of the cache, moved as they are).
  const void* x[3];
  const void* dy[2];
  void* y[3];  // forward: outputs; backward: dx
  int64_t x_s[3][3], dy_s[2][3], y_s[3][3];  // element strides: batch, head, position
  const void* w[2];
  int w_type;        // element type of the weights
  int heads[3];
  const int64_t* pos64;
  const int32_t* pos32;
  int64_t pos_sb, pos_sn;  // strides of the positions
  const double* freq;
  int64_t tokens;  // batch times positions
  int64_t N;
  int D, half, units;  // lanes of a row that hold channels
  int slices;      // waves that share a token's heads
  FastDiv div_slices, div_n;
  float eps;
  int norm, inter;
  float* part;     // [groups, 2, D] partial gradients of the weights
  PagedTables t;   // append
};

template <int TY> struct RotType;
template <> struct RotType<TPF_BF16> { typedef __bf16 E; };
template <> struct RotType<TPF_F16> { typedef _Float16 E; };
template <> struct RotType<TPF_F32> { typedef float E; };

// Where a lane's sixteen channels are: entries 0 .. 7 are the pairs' first channels, 8 .. 15
// the second ones.  With halves lane u < nr has the pairs 8 u .. 8 u + 7 and the others
// sixteen channels that pass; interleaved, lane u has the channels 16 u .. 16 u + 15, and pairs
// from `half` on pass as they are (turned by 0, an infinity would make its neighbour NaN).
struct RotUnit {
  int a0, b0, na, nb, pairs;  // (pairs that turn)
  bool turns, inter;
  __device__ __forceinline__ RotUnit(const RotArgs& r, int u) {
    inter = r.inter;
    pairs = r.half - 8 * u;
    if (inter) {
      a0 = 16 * u;
      b0 = 16 * u + 1;
      na = max(0, min(8, (r.D - 16 * u + 1) / 2));
      nb = max(0, min(8, (r.D - 16 * u) / 2));
      turns = pairs > 0;
      return;
    }
    const int nr = (r.half + 7) / 8;
    turns = u < nr;
    if (turns) {
      na = nb = min(8, r.half - 8 * u);
      a0 = 8 * u;
      b0 = r.half + 8 * u;
    } else {
      a0 = 2 * r.half + 16 * (u - nr);
      b0 = a0 + 8;
      na = max(0, min(8, r.D - a0));
      nb = max(0, min(8, r.D - b0));
    }
  }
  __device__ __forceinline__ bool has(int e) const { return e < 8 ? e < na : e - 8 < nb; }
  __device__ __forceinline__ int channel(int e) const {
    return inter ? a0 + 2 * (e & 7) + (e >> 3) : e < 8 ? a0 + e : b0 + e - 8;
  }
};

// A lane's channels of a row in memory's order: its sixteen channels, or eight and eight; in
// vectors of W, which all strides, D and half are multiples of (interleaved: half may be any).
template <int TY, int W>
struct RotRow {
  typedef typename RotType<TY>::E E;
  typedef E V __attribute__((ext_vector_type(W > 1 ? W : 2)));
  E x[16];
  static __device__ __forceinline__ bool has(const RotUnit& u, int j) {
    return u.inter ? j < u.na + u.nb : u.has(j);
  }
  static __device__ __forceinline__ int channel(const RotUnit& u, int j) {
    return u.inter || j < 8 ? u.a0 + j : u.b0 + j - 8;
  }
  __device__ __forceinline__ void load(const E* p, const RotUnit& u, bool in) {
#pragma unroll
    for (int j = 0; j < 16; j += W) {
#pragma unroll
      for (int e = 0; e < W; ++e) x[j + e] = (E)0.f;
      if (in && has(u, j)) {
        if constexpr (W == 1) {
          x[j] = p[channel(u, j)];
        } else {
          const V v = *reinterpret_cast<const V*>(p + channel(u, j));
#pragma unroll
          for (int e = 0; e < W; ++e) x[j + e] = v[e];
        }
      }
    }
  }
  __device__ __forceinline__ void get(const RotUnit& u, float (&a)[8], float (&b)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = (float)(u.inter ? x[2 * i] : x[i]);
      b[i] = (float)(u.inter ? x[2 * i + 1] : x[8 + i]);
    }
  }
  static __device__ __forceinline__ void store(E* p, const RotUnit& u, const float (&a)[8],
                                               const float (&b)[8]) {
    E y[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const E va = (E)a[i], vb = (E)b[i];
      y[i] = va;
      y[8 + i] = vb;
    }
    if (u.inter) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[2 * i] = (E)a[i];
        y[2 * i + 1] = (E)b[i];
      }
    }
#pragma unroll
    for (int j = 0; j < 16; j += W)
      if (has(u, j)) {
        if constexpr (W == 1) {
          p[channel(u, j)] = y[j];
        } else {
          V v;
#pragma unroll
          for (int e = 0; e < W; ++e) v[e] = y[j + e];
          *reinterpret_cast<V*>(p + channel(u, j)) = v;
        }
      }
  }
};

__device__ __forceinline__ float rot_param(const void* p, int type, int c) {
  if (type == TPF_F32) return ((const float*)p)[c];
  if (type == TPF_F16) return (float)((const _Float16*)p)[c];
  return bf2f(((const u16*)p)[c]);
}
// Both sides' weights into LDS in the lanes' order (1 without one, 0 past the row); a barrier
// has to follow.
template <int L>
__device__ __forceinline__ void rot_weights(const RotArgs& r, float (*w)[16 * L]) {
  for (int i = threadIdx.x; i < 32 * L; i += 256) {
    const int s = i / (16 * L), e = i % (16 * L);
    const RotUnit u(r, e / 16);
    const int x = e % 16;
    w[s][e] = !u.has(x) ? 0.f : r.w[s] ? rot_param(r.w[s], r.w_type, u.channel(x)) : 1.f;
  }
}
__device__ __forceinline__ void rot_eight(const float* p, float (&x)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p + 4 * q);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * q + e] = v[e];
  }
}

// The cosines and sines of position p: lane l forms those of the pairs l, l + 64, into
// the wave's part of LDS.
__device__ __forceinline__ void rot_angles(const RotArgs& r, int64_t p, float* cs) {
  const int lane = threadIdx.x & 63;
  for (int c = lane; c < (r.half + 7) / 8 * 8; c += 64) {
    float s = 0.f, co = 1.f;  // past the last pair
    if (c < r.half) {
      double t = (double)p * (r.freq[c] * 0.15915494309189533577);  // turns
      t -= __builtin_rint(t);
      sincospif(2.f * (float)t, &s, &co);
    }
    cs[c] = co;
    cs[kRotMaxHalf + c] = s;
  }
  __builtin_amdgcn_wave_barrier();
}

template <int L>
__device__ __forceinline__ float rot_squares(const float (&a)[8], const float (&b)[8]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(a[i], a[i], fmaf(b[i], b[i], s));
  return lanes_sum<L>(s);
}

// Side of head hh of a token's queries, keys and values, and its number there.
__device__ __forceinline__ int rot_side(const RotArgs& r, int hh, int& head) {
  const int h0 = r.heads[0], h1 = h0 + r.heads[1];
  const int s = hh < h0 ? 0 : hh < h1 ? 1 : 2;
  head = hh - (s == 0 ? 0 : s == 1 ? h0 : h1);
  return s;
}

// Forward, and (PAGED) the way into the cache: a wave has a share of a token's heads.
template <int TY, int L, int W, bool PAGED>
__global__ __launch_bounds__(256) void rot_fwd_kernel(RotArgs r) {
  typedef RotRow<TY, W> Row;
  typedef typename Row::E E;
  __shared__ __attribute__((aligned(16))) float lds[4][2 * kRotMaxHalf];
  __shared__ __attribute__((aligned(16))) float weights[2][16 * L];
  constexpr int RPW = 64 / L;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r.norm) {
    rot_weights<L>(r, weights);
    __syncthreads();
  }
  const uint32_t item = blockIdx.x * 4 + w;  // (below 2^26)
  const uint32_t token = fdiv(item, r.div_slices);
  const int slice = (int)(item - token * r.slices);
  if (token >= r.tokens) return;  // (no barrier follows)
  const int64_t b = fdiv(token, r.div_n), n = token - b * r.N;
  const RotUnit u(r, lane % L);
  const int total = r.heads[0] + r.heads[1] + r.heads[2];

  const int step = RPW * r.slices;
  auto address = [&](int hh) {
    int head;
    const int s = rot_side(r, hh, head);
    return (const E*)r.x[s] + b * r.x_s[s][0] + head * r.x_s[s][1] + n * r.x_s[s][2];
  };
  Row next;
  int hh = slice * RPW + lane / L;
  next.load(hh < total ? address(hh) : nullptr, u, hh < total);

  int64_t p = n, page = 0, place = 0;
  bool mine = true, placed = false;  // in a sequence; with a place in the cache
  if constexpr (PAGED) {
    const int s = paged_search<PagedWave>(r.t.S, [&](int x) { return paged_start(r.t, x) <= token; });
    mine = s < r.t.S;
    if (mine) {
      p = paged_length(r.t, s) - paged_start(r.t, s + 1) + token;
      placed = paged_place(r.t, s, p, &page, &place);
    }
  } else {
    if (r.pos64) p = r.pos64[b * r.pos_sb + n * r.pos_sn];
    else if (r.pos32) p = r.pos32[b * r.pos_sb + n * r.pos_sn];
  }
  float co[8], si[8];
  if (r.half) {
    rot_angles(r, p, lds[w]);
    if (u.turns) {
      rot_eight(lds[w] + 8 * (lane % L), co);
      rot_eight(lds[w] + kRotMaxHalf + 8 * (lane % L), si);
    }
  }
  const float inv_d = 1.f / (float)r.D;

  for (; hh - lane / L < total; hh += step) {
    const Row row = next;
    const int hn = hh + step;
    next.load(hn < total ? address(hn) : nullptr, u, hn < total);
    float a[8], c[8];
    row.get(u, a, c);
    int head;
    const int s = rot_side(r, min(hh, total - 1), head);
    if (!PAGED || s < 2) {
      if (r.norm) {
        const float rstd = 1.f / sqrtf(fmaf(rot_squares<L>(a, c), inv_d, r.eps));
        float wa[8], wb[8];
        rot_eight(weights[s == 1] + 16 * (lane % L), wa);
        rot_eight(weights[s == 1] + 16 * (lane % L) + 8, wb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] = a[i] * rstd * wa[i];
          c[i] = c[i] * rstd * wb[i];
        }
      }
      if (u.turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = a[i], y = c[i];
          a[i] = i < u.pairs ? x * co[i] - y * si[i] : x;
          c[i] = i < u.pairs ? y * co[i] + x * si[i] : y;
        }
      }
    }
    if (hh >= total) continue;
    E* dst = (E*)r.y[s];
    if (PAGED && s) {
      if (!placed) continue;
      dst += page * r.y_s[s][0] + head * r.y_s[s][1] + place * r.y_s[s][2];
    } else {
      dst += b * r.y_s[s][0] + head * r.y_s[s][1] + n * r.y_s[s][2];
      if (PAGED && !mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = c[i] = 0.f;
      }
    }
    Row::store(dst, u, a, c);
  }
}

// Backward: a workgroup's waves take tokens in turn and keep the weights' gradients of
// their channels in registers; what the rows, waves and workgroups have is added in a
// fixed order (and by rot_fold_kernel: 4 us).
template <int TY, int L, int W>
__global__ __launch_bounds__(256) void rot_bwd_kernel(RotArgs r) {
  typedef RotRow<TY, W> Row;
  typedef typename Row::E E;
  __shared__ __attribute__((aligned(16))) float lds[4][2 * kRotMaxHalf];
  __shared__ __attribute__((aligned(16))) float weights[2][16 * L];
  constexpr int RPW = 64 / L;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r.norm) {
    rot_weights<L>(r, weights);
    __syncthreads();
  }
  const RotUnit u(r, lane % L);
  const int total = r.heads[0] + r.heads[1], step = RPW * r.slices;
  const float inv_d = 1.f / (float)r.D;
  float ga[2][8], gb[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ga[0][i] = ga[1][i] = gb[0][i] = gb[1][i] = 0.f;

  const uint32_t items = (uint32_t)(r.tokens * r.slices);  // (below 2^26)
  for (uint32_t item = blockIdx.x * 4 + w; item < items; item += gridDim.x * 4) {
    const uint32_t token = fdiv(item, r.div_slices);
    const int slice = (int)(item - token * r.slices);
    const int64_t b = fdiv(token, r.div_n), n = token - b * r.N;
    Row nx, nd;
    int hh = slice * RPW + lane / L;
    auto load = [&](int h) {
      int head;
      const int s = rot_side(r, min(h, total - 1), head);
      nd.load((const E*)r.dy[s] + b * r.dy_s[s][0] + head * r.dy_s[s][1] + n * r.dy_s[s][2], u, h < total);
      if (r.norm)
        nx.load((const E*)r.x[s] + b * r.x_s[s][0] + head * r.x_s[s][1] + n * r.x_s[s][2], u, h < total);
    };
    load(hh);
    int64_t p = n;
    if (r.pos64) p = r.pos64[b * r.pos_sb + n * r.pos_sn];
    else if (r.pos32) p = r.pos32[b * r.pos_sb + n * r.pos_sn];
    float co[8], si[8];
    if (r.half) {
      __builtin_amdgcn_wave_barrier();
      rot_angles(r, p, lds[w]);
      if (u.turns) {
        rot_eight(lds[w] + 8 * (lane % L), co);
        rot_eight(lds[w] + kRotMaxHalf + 8 * (lane % L), si);
      }
    }
    for (; hh - lane / L < total; hh += step) {
      const Row rx = nx, rd = nd;
      load(hh + step);
      float a[8], c[8];
      rd.get(u, a, c);
      if (u.turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = a[i], y = c[i];
          a[i] = i < u.pairs ? x * co[i] + y * si[i] : x;
          c[i] = i < u.pairs ? y * co[i] - x * si[i] : y;
        }
      }
      int head;
      const int s = rot_side(r, min(hh, total - 1), head);
      if (r.norm) {
        float xa[8], xb[8];
        rx.get(u, xa, xb);
        const float rstd = 1.f / sqrtf(fmaf(rot_squares<L>(xa, xb), inv_d, r.eps));
        float dot = 0.f, wa[8], wb[8];
        rot_eight(weights[s] + 16 * (lane % L), wa);
        rot_eight(weights[s] + 16 * (lane % L) + 8, wb);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          xa[i] *= rstd;
          xb[i] *= rstd;
          const float va = a[i] * xa[i], vb = c[i] * xb[i];
          if (hh < total) {
            if (s) {
              ga[1][i] += va;
              gb[1][i] += vb;
            } else {
              ga[0][i] += va;
              gb[0][i] += vb;
            }
          }
          a[i] *= wa[i];
          c[i] *= wb[i];
          dot = fmaf(a[i], xa[i], fmaf(c[i], xb[i], dot));
        }
        dot = lanes_sum<L>(dot) * inv_d;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] = rstd * fmaf(-xa[i], dot, a[i]);
          c[i] = rstd * fmaf(-xb[i], dot, c[i]);
        }
      }
      if (hh < total)
        Row::store((E*)r.y[s] + b * r.y_s[s][0] + head * r.y_s[s][1] + n * r.y_s[s][2], u, a, c);
    }
  }
  if (!r.part) return;
  __shared__ float sums[4][2][16 * L];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a = ga[s][i], c = gb[s][i];
#pragma unroll
      for (int o = L; o < 64; o <<= 1) {
        a += __shfl_xor(a, o);
        c += __shfl_xor(c, o);
      }
      if (lane < L) {
        sums[w][s][16 * lane + i] = a;
        sums[w][s][16 * lane + 8 + i] = c;
      }
    }
  __syncthreads();
  for (int t = threadIdx.x; t < 32 * L; t += 256) {
    const int s = t / (16 * L), e = t - s * 16 * L;
    const RotUnit v(r, e / 16);
    if (v.has(e % 16))
      r.part[((int64_t)blockIdx.x * 2 + s) * r.D + v.channel(e % 16)] =
          ((sums[0][s][e] + sums[1][s][e]) + sums[2][s][e]) + sums[3][s][e];
  }
}

// The weights' gradients from the workgroups' sums: sixteen channels of a side a workgroup,
// sixteen ranges of the sums, whose partial sums meet in LDS in order.
__global__ __launch_bounds__(256) void rot_fold_kernel(const float* part, int groups, int D, void* dq,
                                                       void* dk, int type) {
  __shared__ float sums[16][16];
  const int s = blockIdx.y, c = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
  void* out = s ? dk : dq;
  if (!out) return;
  const int per = (groups + 15) / 16, end = min(groups, (q + 1) * per);
  float v = 0.f;
  if (c < D) {
#pragma unroll 16
    for (int g = q * per; g < end; ++g) v += part[((int64_t)g * 2 + s) * D + c];
  }
  sums[q][threadIdx.x & 15] = v;
  __syncthreads();
  if (q || c >= D) return;
#pragma unroll
  for (int x = 1; x < 16; ++x) v += sums[x][threadIdx.x & 15];
  if (type == TPF_F32) ((float*)out)[c] = v;
  else if (type == TPF_F16) ((_Float16*)out)[c] = (_Float16)v;
  else ((u16*)out)[c] = f2bf_bits(v);
}

// A token's heads are shared by waves as long as there are fewer than 16384 (8192 backward,
// whose workgroups take several tokens): 2 x 4096 tokens, 32 + 8 heads of 128 in 40 us forward
// against 45 with 8192 and 43 with 40960; backward 71 against 79 with 16384.  An append's waves
// first find their token's place: 4096 (8 chunks of up to 1024 tokens, 16 heads of 80 and as many
// keys and values: 22 us against 23 with 8192 and 24 with 16384; 8 of 256, 32 heads on 8 of 128: 14, 14, 16).
static void rot_plan(RotArgs& r, int rows_per_wave, bool backward) {
  const int total = r.heads[0] + r.heads[1] + r.heads[2];
  const int most = (total + rows_per_wave - 1) / rows_per_wave;
  int64_t s = ((backward ? 8192 : r.heads[2] ? 4096 : 16384) + r.tokens - 1) / r.tokens;
  s = s < 1 ? 1 : s > most ? most : s;
  const int64_t turns = (most + s - 1) / s;  // (as few waves as take no more of them)
  r.slices = (int)((most + turns - 1) / turns);
  r.div_slices = make_fastdiv((uint32_t)r.slices);
  r.div_n = make_fastdiv((uint32_t)r.N);
}

static int rot_lanes(const RotArgs& r) {
  int l = 4;
  while (l < r.units) l *= 2;
  return l;
}

// Workgroups of a backward: three a CU, as many as its registers let run (the same tokens: 71 us
// against 87 with 1024, a third of which had to wait).
constexpr int64_t kRotGroups = 768;

static int64_t rot_groups(const RotArgs& r) {
  const int64_t n = (r.tokens * r.slices + 3) / 4;
  return n < kRotGroups ? n : kRotGroups;
}

template <int TY, int L, int W>
static void rot_launch(const RotArgs& r, int mode, hipStream_t s) {
  const dim3 all((unsigned)((r.tokens * r.slices + 3) / 4));
  if (mode == 0) hipLaunchKernelGGL((rot_fwd_kernel<TY, L, W, false>), all, dim3(256), 0, s, r);
  if constexpr (TY != TPF_F32)
    if (mode == 1) hipLaunchKernelGGL((rot_fwd_kernel<TY, L, W, true>), all, dim3(256), 0, s, r);
  if (mode == 2)
    hipLaunchKernelGGL((rot_bwd_kernel<TY, L, W>), dim3((unsigned)rot_groups(r)), dim3(256), 0, s, r);
}
template <int TY, int L>
static void rot_wide(const RotArgs& r, int mode, int w, hipStream_t s) {
  if (w == 8 && TY != TPF_F32) rot_launch<TY, L, TY == TPF_F32 ? 4 : 8>(r, mode, s);
  else if (w >= 4) rot_launch<TY, L, 4>(r, mode, s);
  else if (w == 2) rot_launch<TY, L, 2>(r, mode, s);
  else rot_launch<TY, L, 1>(r, mode, s);
}
template <int TY>
static void rot_pick(const RotArgs& r, int mode, int w, hipStream_t s) {
  switch (rot_lanes(r)) {
    case 4: rot_wide<TY, 4>(r, mode, w, s); break;
    case 8: rot_wide<TY, 8>(r, mode, w, s); break;
    case 16: rot_wide<TY, 16>(r, mode, w, s); break;
    default: rot_wide<TY, 32>(r, mode, w, s);
  }
}
static void rot_run(const RotArgs& r, int64_t type, int mode, int w, hipStream_t s) {
  if (type == TPF_BF16) rot_pick<TPF_BF16>(r, mode, w, s);
  else if (type == TPF_F16) rot_pick<TPF_F16>(r, mode, w, s);
  else rot_pick<TPF_F32>(r, mode, w, s);
}

// Sizes of a call into r; 0 or an error code.
static int rot_check(RotArgs& r, int64_t B, int64_t N, int64_t H, int64_t Hk, int64_t Hv, int64_t D,
                     int64_t half, int64_t type, int64_t w_type, double eps, int norm,
                     int inter, bool backward, const char* fn) {
  const int64_t lim = (int64_t)1 << 30;
  if (B < 1 || N < 1 || B > lim || N > lim || H < 0 || Hk < 0 || H + Hk < 1 || H > 65535 || Hk > 65535 ||
      D < 1 || D > 256 || half < 0 || 2 * half > D)
    return set_error(TPF_ERR_SHAPE, "%s: bad shape B=%lld N=%lld H=%lld Hk=%lld D=%lld half=%lld", fn,
                     (long long)B, (long long)N, (long long)H, (long long)Hk, (long long)D,
                     (long long)half);
  if (type < 0 || type > 2 || w_type < 0 || w_type > 2)
    return set_error(TPF_ERR_ARG, "%s: unknown type", fn);
  if (norm && !(eps >= 0.0 && eps < 1e30))
    return set_error(TPF_ERR_ARG, "%s: eps must be between 0 and 1e30", fn);
  r.tokens = B * N;
  r.N = N;
  r.heads[0] = (int)H; r.heads[1] = (int)Hk; r.heads[2] = (int)Hv;
  r.D = (int)D; r.half = (int)half;
  r.inter = inter;
  r.units = (int)(inter ? (D + 15) / 16 : (half + 7) / 8 + (D - 2 * half + 15) / 16);
  r.norm = norm;
  r.eps = (float)eps;
  r.w_type = (int)w_type;
  rot_plan(r, 64 / rot_lanes(r), backward);
  if ((double)B * (double)N * r.slices > 4.0 * (double)kMaxGroups)  // (four waves a workgroup)
    return set_error(TPF_ERR_SHAPE, "%s: too many tokens", fn);
  return TPF_OK;
}

// Elements of the widest vectors (up to `w`) that the rows at p with these strides allow.
static int rot_width(const RotArgs& r, int64_t type, int w, const void* p, const int64_t* strides) {
  const int size = type == TPF_F32 ? 4 : 2;
  const int64_t all = (r.inter ? 0 : r.half) | r.D | strides[0] | strides[1] | strides[2];
  while (w > 1 && (all % w || (uintptr_t)p % (w * size))) w /= 2;
  return w;
}

}  // namespace tpf

static int rot_entry(tpf::RotArgs& r, const tpf_rotary_shape* s, const void* positions,
                     const double* frequencies, const void* qw, const void* kw, double eps,
                     bool backward, const char* fn) {
  if (!s) return tpf::set_error(TPF_ERR_ARG, "%s: null shape", fn);
  if (int rc = tpf::rot_check(r, s->B, s->N, s->H, s->Hk, 0, s->D, s->half, s->dtype, s->weight_dtype, eps,
                              s->norm != 0, s->interleaved != 0, backward, fn))
    return rc;
  if (s->half && !frequencies) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (s->position_bits != 32 && s->position_bits != 64)
    return tpf::set_error(TPF_ERR_ARG, "%s: positions have 32 or 64 bits", fn);
  if (s->position_bits == 64) r.pos64 = (const int64_t*)positions;
  else r.pos32 = (const int32_t*)positions;
  r.pos_sb = s->position_stride[0];
  r.pos_sn = s->position_stride[1];
  r.freq = frequencies;
  r.w[0] = qw;
  r.w[1] = kw;
  for (int i = 0; i < 3; ++i) {
    r.x_s[0][i] = s->q_stride[i];
    r.x_s[1][i] = s->k_stride[i];
    r.y_s[0][i] = s->out_q_stride[i];
    r.y_s[1][i] = s->out_k_stride[i];
  }
  return TPF_OK;
}

extern "C" int tpf_rotary_forward(const void* q, const void* k, const void* positions,
                                  const double* frequencies, const void* q_weight,
                                  const void* k_weight, double eps, void* q_out, void* k_out,
                                  const tpf_rotary_shape* shape, void* stream) {
  const char* fn = "tpf_rotary_forward";
  tpf::RotArgs r{};
  if (int rc = rot_entry(r, shape, positions, frequencies, q_weight, k_weight, eps, false, fn)) return rc;
  if ((shape->H && (!q || !q_out)) || (shape->Hk && (!k || !k_out)))
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  r.x[0] = q; r.x[1] = k; r.y[0] = q_out; r.y[1] = k_out;
  int w = 8;
  for (int i = 0; i < 2; ++i)
    if (r.heads[i]) {
      w = tpf::rot_width(r, shape->dtype, w, r.x[i], r.x_s[i]);
      w = tpf::rot_width(r, shape->dtype, w, r.y[i], r.y_s[i]);
    }
  tpf::rot_run(r, shape->dtype, 0, w, (hipStream_t)stream);
  return tpf::check_launch(fn);
}

extern "C" int64_t tpf_rotary_backward_workspace_bytes(const tpf_rotary_shape* shape) {
  tpf::RotArgs r{};
  if (rot_entry(r, shape, nullptr, (const double*)16, nullptr, nullptr, 0.0, true,
                "tpf_rotary_backward_workspace_bytes"))
    return -1;
  return tpf::rot_groups(r) * 2 * r.D * 4;
}

extern "C" int tpf_rotary_backward(const void* q, const void* k, const void* dq_out, const void* dk_out,
                                   const void* positions, const double* frequencies,
                                   const void* q_weight, const void* k_weight, double eps, void* dq,
                                   void* dk, void* dq_weight, void* dk_weight, void* workspace,
                                   int64_t workspace_bytes, const tpf_rotary_shape* shape,
                                   const int64_t* grad_strides, void* stream) {
  const char* fn = "tpf_rotary_backward";
  tpf::RotArgs r{};
  if (int rc = rot_entry(r, shape, positions, frequencies, q_weight, k_weight, eps, true, fn)) return rc;
  if (!grad_strides || (shape->H && (!dq_out || !dq || (r.norm && !q))) ||
      (shape->Hk && (!dk_out || !dk || (r.norm && !k))))
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  const bool want = dq_weight || dk_weight;
  if (want && !r.norm) return tpf::set_error(TPF_ERR_ARG, "%s: weights belong to a norm", fn);
  if (want && (!workspace || workspace_bytes < tpf::rot_groups(r) * 2 * r.D * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  r.x[0] = q; r.x[1] = k; r.dy[0] = dq_out; r.dy[1] = dk_out; r.y[0] = dq; r.y[1] = dk;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) r.dy_s[i][j] = grad_strides[3 * i + j];
  r.part = want ? (float*)workspace : nullptr;
  int w = 8;
  for (int i = 0; i < 2; ++i)
    if (r.heads[i]) {
      if (r.norm) w = tpf::rot_width(r, shape->dtype, w, r.x[i], r.x_s[i]);
      w = tpf::rot_width(r, shape->dtype, w, r.dy[i], r.dy_s[i]);
      w = tpf::rot_width(r, shape->dtype, w, r.y[i], r.y_s[i]);
    }
  hipStream_t st = (hipStream_t)stream;
  tpf::rot_run(r, shape->dtype, 2, w, st);
  if (want)
    hipLaunchKernelGGL(tpf::rot_fold_kernel, dim3((r.D + 15) / 16, 2), dim3(256), 0, st, r.part,
                       (int)tpf::rot_groups(r), r.D, dq_weight, dk_weight, r.w_type);
  return tpf::check_launch(fn);
}

namespace tpf {

int paged_check(PagedTables& t, const tpf_paged_batch* b, const char* fn) {
  if (!b) return set_error(TPF_ERR_ARG, "%s: null batch", fn);
  const int64_t lim = (int64_t)1 << 30;
  if (b->S < 0 || b->S > lim || b->T < 1 || b->T > lim || b->width < 0 || b->width > lim || b->page < 1 ||
      b->page > lim || b->pages < 0 || b->pages > lim || b->table_stride < 0 ||
      (double)b->width * (double)b->page > (double)lim)
    return set_error(TPF_ERR_SHAPE, "%s: bad batch S=%lld T=%lld width=%lld page=%lld pages=%lld", fn,
                     (long long)b->S, (long long)b->T, (long long)b->width, (long long)b->page,
                     (long long)b->pages);
  if ((b->S && b->width && !b->tables) || !b->starts || (b->S && !b->lengths))
    return set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  t.tables = b->tables;
  t.starts = b->starts;
  t.lengths = b->lengths;
  t.table_ld = b->table_stride;
  t.T = b->T;
  t.S = (int)b->S;
  t.width = (int)b->width;
  t.page = (int)b->page;
  t.pages = (int)b->pages;
  t.div_page = make_fastdiv((uint32_t)b->page);
  return TPF_OK;
}

}  // namespace tpf

extern "C" int64_t tpf_paged_row(const tpf_paged_batch* batch, int64_t s, int64_t state) {
  tpf::PagedTables t{};
  if (tpf::paged_check(t, batch, "tpf_paged_row") || s < 0 || s >= t.S) return -1;
  int64_t page, place;
  return tpf::paged_place(t, (int)s, state, &page, &place) ? page * t.page + place : -1;
}

extern "C" int64_t tpf_paged_rows(const tpf_paged_batch* batch, int64_t group, int64_t tile_rows, int64_t at,
                                  int64_t* rows) {
  tpf::PagedTables t{};
  const int64_t lim = (int64_t)1 << 30;
  if (tpf::paged_check(t, batch, "tpf_paged_rows") || !rows || group < 1 || group > lim / t.T ||
      t.S > lim / 256 || at < 0)
    return -1;
  tpf::PagedRows r;
  if (tile_rows == 0) {
    if (at >= t.T * group || !r.row<tpf::PagedHost>(t, (int)group, at)) return -1;
  } else if ((tile_rows != 32 && tile_rows != 128) || at > t.T * group / tile_rows + t.S ||
             !r.tile<tpf::PagedHost>(t, (int)group, (int)tile_rows, (int)at)) {
    return -1;
  }
  rows[0] = r.r0;
  rows[1] = r.R;
  rows[2] = r.token;
  return r.s;
}

extern "C" int tpf_paged_append(const void* q, const void* k, const void* v, const double* frequencies,
                                const void* q_weight, const void* k_weight, double eps, void* q_out,
                                void* k_cache, void* v_cache, const tpf_append_shape* s,
                                const tpf_paged_batch* batch, void* stream) {
  const char* fn = "tpf_paged_append";
  tpf::RotArgs r{};
  if (!s) return tpf::set_error(TPF_ERR_ARG, "%s: null shape", fn);
  if (int rc = tpf::paged_check(r.t, batch, fn)) return rc;
  if (s->dtype != TPF_BF16 && s->dtype != TPF_F16)
    return tpf::set_error(TPF_ERR_ARG, "%s: dtype must be TPF_BF16 or TPF_F16", fn);
  if (s->Hk < 1) return tpf::set_error(TPF_ERR_SHAPE, "%s: no kv heads", fn);
  if (int rc = tpf::rot_check(r, 1, batch->T, s->H, s->Hk, s->Hk, s->D, s->half, s->dtype, s->weight_dtype,
                              eps, s->norm != 0, s->interleaved != 0, false, fn))
    return rc;
  if (!k || !v || (batch->pages && (!k_cache || !v_cache)) || (s->H && (!q || !q_out)) || (s->half && !frequencies))
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  r.x[0] = q; r.x[1] = k; r.x[2] = v;
  r.y[0] = q_out; r.y[1] = k_cache; r.y[2] = v_cache;
  r.w[0] = q_weight; r.w[1] = k_weight;
  r.freq = frequencies;
  const int64_t* in[3] = {s->q_stride, s->k_stride, s->v_stride};
  int w = 8;
  for (int i = 0; i < 3; ++i) {
    r.x_s[i][1] = in[i][1];
    r.x_s[i][2] = in[i][0];
  }
  r.y_s[0][1] = s->D;
  r.y_s[0][2] = s->H * s->D;
  for (int i = 1; i < 3; ++i) {
    r.y_s[i][0] = s->Hk * batch->page * s->D;
    r.y_s[i][1] = batch->page * s->D;
    r.y_s[i][2] = s->D;
  }
  for (int i = 0; i < 3; ++i)
    if (r.heads[i]) {
      w = tpf::rot_width(r, s->dtype, w, r.x[i], r.x_s[i]);
      w = tpf::rot_width(r, s->dtype, w, r.y[i], r.y_s[i]);
    }
  tpf::rot_run(r, s->dtype, 1, w, (hipStream_t)stream);
  return tpf::check_launch(fn);
}
