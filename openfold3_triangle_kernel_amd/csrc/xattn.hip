// Cross attention to states of another length: forward.
//
//   s_ij = scale q_i . k_j + mask_j,  p = softmax_j(s),  o_i = sum_j p_ij v_j
//
// over R = G * Nq rows of a kv head and its Nk states (xattn.hpp), in one pass
// over the states with a running maximum and sum.  A wave owns 32 QB rows and
// forms S^T = K Q^T, so a lane holds one row's scores: maxima and sums are
// lane-local up to one exchange with lane ^ 32, and the S^T tile goes back into
// the matrix cores as it stands for O^T += V^T P^T.  A row without a live state
// gives 0.
#include "gemm_core.hpp"  // xcd_order
#include "tpf_status.hpp"
#include "xattn.hpp"

namespace tpf {

// The maximum of a row before its first live state, and the least one after it: a row
// whose scores are all -inf (infinite operands) is told from a row without a state.
constexpr float kXaLow = -3.402823466e38f, kXaSeen = -3.3e38f;
constexpr int kXaMaxSplits = 256;  // threads of the workgroup that joins a row's splits

// Running softmax state of a wave's rows; scores and maxima m are in raw units
// (before the scale).  The maximum is raised only once a row's scores pass it by
// 8 powers of two: p then stays below 256, which 32-bit sums and either operand
// type hold, and the outputs are rescaled a few times per call instead of every
// tile.  p is one fused multiply-add and an exponential, 2^(c s - c m); where a
// tile has additive values, which may be of any size, the maximum is taken off
// first, 2^(c (s - m)).
//
// p enters the second product rounded to the operands' type, and the outputs are
// divided by n, the sum of the rounded p: they are means of V with weights that sum
// to 1, so what the states' values have in common passes exactly (divided by the
// unrounded sum, the roundings of p would scale it).  The backward's p come from
// scores again and are divided by l, the sum of the unrounded ones, which only a
// forward with statistics forms (32 heads, 4096 x 4096 x 128: 305 us with it and the
// residual's stores against 284 without).  n is summed among the second product's steps,
// whose time hides it (before them, 4096 x 4096 x 128 took 289 us instead of 272).
template <int DP, int QB, bool F16, bool STATS>
struct XRows {
  static constexpr int DS = DP / 16, DB = DP / 32;
  bf16x8 q[QB][DS];
  f32x16 o[QB][DB];
  float m[QB], l[QB], n[QB];

  __device__ __forceinline__ void init(const XAttnArgs& a, int b, int hk, int r0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = r0 + 32 * qb + (lane & 31);
      int g, i;
      xa_row(a, r < a.R ? r : a.R - 1, g, i);
      const u16* p = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn;
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        q[qb][s] = d < a.D ? *reinterpret_cast<const bf16x8*>(p + d) : zero8();
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) o[qb][db] = zero16();
      m[qb] = kXaLow;
      l[qb] = n[qb] = 0.f;
    }
  }

  // KB blocks of 32 states from k0 on, in the tiles K and V.
  template <int KB>
  __device__ __forceinline__ void step(const XAttnArgs& a, const u16* K, const u16* V, uint64_t live,
                                       const float* fmask, int k0) {
    f32x16 s[QB][KB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[qb][kb] = zero16();
    if constexpr (DP > 96) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int d = 0; d < DS; ++d) {
        const bf16x8 kf = xa_frag<DP>(K, 32 * kb, d);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) s[qb][kb] = xa_mfma<F16>(kf, q[qb][d], s[qb][kb]);
      }
    if constexpr (DP > 96) __builtin_amdgcn_s_setprio(0);
    const uint64_t whole = KB == 2 ? ~0ull : 0xffffffffull;
    if (live != whole || fmask) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          xa_mask32(s[qb][kb], (uint32_t)(live >> (32 * kb)), fmask, k0 + 32 * kb, a.Nk, a.inv_scale,
                    a.mask_floor);
    }
    bf16x8 p[QB][2 * KB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float t = kXaSeen;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = xa_max(t, s[qb][kb][r]);
      t = xa_max32(t);
      if (__ballot((t - m[qb]) * a.c > 8.f)) {
        const float mn = xa_max(m[qb], t), al = fast_exp2((m[qb] - mn) * a.c);
        m[qb] = mn;
        if constexpr (STATS) l[qb] *= al;
        n[qb] *= al;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[qb][db][r] *= al;
      }
      float off = xa_min(-m[qb] * a.c, -kXaLow), sum = 0.f;  // (finite beside a score of -inf)
      if (fmask) {
        off = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[qb][kb][r] -= m[qb];
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[qb][kb][r] = fast_exp2(fmaf(s[qb][kb][r], a.c, off));
          if constexpr (STATS) sum += s[qb][kb][r];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          p[qb][2 * kb + t] = xa_pack8<F16>(s[qb][kb], 8 * t);
        }
      }
      if constexpr (STATS) l[qb] += sum;
    }
    if constexpr (DP > 96) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const bf16x8 vf = xa_frag_t<DP>(V, 32 * kb, t, db);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) o[qb][db] = xa_mfma<F16>(vf, p[qb][2 * kb + t], o[qb][db]);
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const u32x4 w = __builtin_bit_cast(u32x4, p[qb][2 * kb + t]);
#pragma unroll
          for (int e = 0; e < 4; ++e) n[qb] = xa_add_pair<F16>(w[e], n[qb]);
        }
      }
    if constexpr (DP > 96) __builtin_amdgcn_s_setprio(0);
  }
};

// 1 / sum of a row with the maximum m; 0 for a row without a live state, NaN for one
// whose scores are all -inf.
__device__ __forceinline__ float xa_inverse(float n, float m) {
  return n == 0.f ? (m == kXaLow ? 0.f : __builtin_nanf("")) : 1.f / n;
}

// A row's statistics for the backward: log2 of the sum and the raw maximum, or
// without additive masks the two as one log-sum-exp.
__device__ __forceinline__ void xa_store_stats(const XAttnArgs& a, int64_t row, float m, float l) {
  const float ll = __log2f(l);
  if (a.mask_kind == kMaskF32) {
    a.lse[row] = ll;
    a.lse[(int64_t)a.B * a.Hk * a.R + row] = m;
  } else {
    a.lse[row] = fmaf(m, a.c, ll);
  }
}

// Writes four channels of a row's output at `at`, and what their rounding drops where
// the backward wants it: its delta = dO . O takes O from both.
template <bool F16>
__device__ __forceinline__ void xa_store4(const XAttnArgs& a, int64_t at, float x0, float x1, float x2,
                                          float x3) {
  uint2 v;
  v.x = xa_pair<F16>(x0, x1);
  v.y = xa_pair<F16>(x2, x3);
  *reinterpret_cast<uint2*>(a.out + at) = v;
  if constexpr (!F16) {
    if (a.res) {
      uint2 r;
      r.x = xa_pair<false>(x0 - __uint_as_float(v.x << 16), x1 - __uint_as_float(v.x & 0xffff0000u));
      r.y = xa_pair<false>(x2 - __uint_as_float(v.y << 16), x3 - __uint_as_float(v.y & 0xffff0000u));
      *reinterpret_cast<uint2*>(a.res + at) = r;
    }
  }
}

// Writes a row's outputs that this lane holds (channels 32 db + 8 g4 + 4 h + e).
template <int DB, bool F16>
__device__ __forceinline__ void xa_store_row(const XAttnArgs& a, int b, int hk, int r,
                                             const f32x16 (&o)[DB], float inv) {
  const int h = (threadIdx.x >> 5) & 1;
  int g, i;
  xa_row(a, r, g, i);
  const int64_t at = (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int d = 32 * db + 8 * g4 + 4 * h;
      if (d < a.D)
        xa_store4<F16>(a, at + d, o[db][4 * g4] * inv, o[db][4 * g4 + 1] * inv,
                       o[db][4 * g4 + 2] * inv, o[db][4 * g4 + 3] * inv);
    }
}

// Four waves of 32 QB rows share K and V tiles of 64 states, two stages deep.
// Tiles without a live state are passed over.  KW = 2: two groups of four waves
// take a row tile's states in turn (64 each of every 128) and join their results in
// LDS, for grids that give a CU one workgroup: the SIMDs then have two waves (16
// heads on 4, 4 x 509 x 1021 x 80: 24.5 us against 28.6 with two splits in memory).
// 32 heads, 4096 x 4096 x 128 in 268 to 289 us from card to card (950 to 1025 TFLOP/s, the
// matrix and the vector units busy about half the time each), 64 channels in 154 to 173.
template <int DP, int QB, bool F16, int KW, bool STATS>
__global__ __launch_bounds__(256 * KW, 2) void xattn_fwd_kernel(XAttnArgs a) {
  constexpr int KT = 64, TILE = KT * DP, DB = DP / 32;
  static_assert(KW == 1 || QB == 1, "a group's results fit its tiles");
  __shared__ __attribute__((aligned(1024))) u16 smem[KW][2][2][TILE];
  __shared__ float ml[KW == 2 ? 768 : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = KW == 2 ? wave >> 2 : 0, w = wave & 3, lane = threadIdx.x & 63;
  const int64_t total = (int64_t)a.B * a.Hk * a.splits * a.tiles;
  const int64_t T = xcd_order(total);
  if (T < 0) return;
  const int tile = (int)(T % a.tiles);
  const int64_t u = T / a.tiles;
  const int split = (int)(u % a.splits);
  const int64_t bh = u / a.splits;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  const int r0 = tile * 128 * QB + w * 32 * QB;
  const int kbeg = split * a.chunk, kend = min(a.Nk, kbeg + a.chunk);
  const u16* kp = a.k + b * a.k_sb + hk * a.k_sh;
  const u16* vp = a.v + b * a.v_sb + hk * a.v_sh;

  XTiles<KW> t;
  t.init(a, b, kbeg, kend);
  XTileLoader<DP, KT, 4> lk, lv;
  lk.init(w, a.k_sn, a.D);
  lv.init(w, a.v_sn, a.D);
  XRows<DP, QB, F16, STATS> rows;
  rows.init(a, b, hk, r0);

  // With one group a round always has a live state (no branch then: with it, 4096 x
  // 4096 x 128 took 6 % longer).
  auto issue = [&](int st) {
    const uint64_t live = KW == 2 && group ? t.live[KW - 1] : t.live[0];
    const int64_t k = t.k0 + KT * group;
    if (KW == 1 || live) {
      lk.issue(kp + k * a.k_sn, live, w, smem[group][st][0]);
      lv.issue(vp + k * a.v_sn, live, w, smem[group][st][1]);
    }
  };
  bool more = t.advance();
  if (more) issue(0);
  int st = 0;
  while (more) {
    const int kc = t.k0 + KT * group;
    const uint64_t lc = KW == 2 && group ? t.live[KW - 1] : t.live[0];
    const bool vc = KW == 2 && group ? t.values[KW - 1] : t.values[0];
    wait_vmcnt<0>();
    lds_barrier();
    more = t.advance();
    if (more) issue(st ^ 1);
    if (KW == 1 || lc)
      rows.template step<2>(a, smem[group][st][0], smem[group][st][1], lc,
                            vc ? t.mask.f : nullptr, kc);
    st ^= 1;
  }
  if constexpr (KW == 2) {
    static_assert(sizeof(smem) >= 4 * DB * 4096, "the join fits");
    char* lds = reinterpret_cast<char*>(&smem[0][0][0][0]);
    __syncthreads();
    if (group) {
      xa_give<DB>(lds, w, rows.o[0]);
      ml[3 * (64 * w + lane)] = rows.m[0];
      ml[3 * (64 * w + lane) + 1] = rows.l[0];
      ml[3 * (64 * w + lane) + 2] = rows.n[0];
    }
    __syncthreads();
    if (group) return;
    const float m1 = ml[3 * (64 * w + lane)], l1 = ml[3 * (64 * w + lane) + 1];
    const float n1 = ml[3 * (64 * w + lane) + 2];
    const float m = xa_max(rows.m[0], m1);
    const float f0 = fast_exp2((rows.m[0] - m) * a.c), f1 = fast_exp2((m1 - m) * a.c);
    xa_take<DB>(lds, w, rows.o[0], f0, f1);
    rows.l[0] = f0 * rows.l[0] + f1 * l1;
    rows.n[0] = f0 * rows.n[0] + f1 * n1;
    rows.m[0] = m;
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = r0 + 32 * qb + (lane & 31);
    const float l = xor32_sum(rows.l[qb]), n = xor32_sum(rows.n[qb]);
    if (r >= a.R) continue;
    if (a.splits == 1) {
      xa_store_row<DP / 32, F16>(a, b, hk, r, rows.o[qb], xa_inverse(n, rows.m[qb]));
      if (a.lse && lane < 32) xa_store_stats(a, bh * a.R + r, rows.m[qb], l);
    } else {
      const int64_t pr = (bh * a.splits + split) * a.R + r;
      if (lane < 32) {
        a.part_ml[3 * pr] = rows.m[qb];
        a.part_ml[3 * pr + 1] = l;
        a.part_ml[3 * pr + 2] = n;
      }
      float* p = a.part_o + pr * a.D;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int d = 32 * db + 8 * g4 + 4 * (lane >> 5);
          if (d < a.D) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = rows.o[qb][db][4 * g4 + e];
            *reinterpret_cast<f32x4*>(p + d) = v;
          }
        }
    }
  }
}

// Few rows (at most 32 QB, one decoded token above all): the states' bytes are
// the bound.  Every wave streams tiles of 32 states of its own, two stages deep
// without a barrier, and the four waves' results meet in LDS at the end.  8 sequences of
// 32 kv heads with 4096 states, one row each (537 MB, unsplit): 96 us, 5.6 TB/s.  16 tokens of 32 heads on 8
// with 8191 ragged states (403 MB live) in two splits: 79 us with the join.
template <int DP, int QB, bool F16, bool STATS>
__global__ __launch_bounds__(256, 1) void xattn_few_kernel(XAttnArgs a) {
  constexpr int KT = 32, TILE = KT * DP, NI = KT * DP / 512;
  constexpr int OP = DP + 4;  // pitch of the joined rows (f32)
  __shared__ __attribute__((aligned(1024))) u16 smem[4][2][2][TILE];
  static_assert(sizeof(smem) >= 4 * 32 * (OP + 3) * 4, "the join fits");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t T = xcd_order((int64_t)a.B * a.Hk * a.splits);
  if (T < 0) return;
  const int64_t bh = T / a.splits;
  const int split = (int)(T - bh * a.splits);
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  const int kbeg = split * a.chunk, kend = min(a.Nk, kbeg + a.chunk);
  const u16* kp = a.k + b * a.k_sb + hk * a.k_sh;
  const u16* vp = a.v + b * a.v_sb + hk * a.v_sh;

  XMask mask;
  mask.init(a, b);
  XTileLoader<DP, KT, 1> lk, lv;
  lk.init(0, a.k_sn, a.D);
  lv.init(0, a.v_sn, a.D);
  XRows<DP, QB, F16, STATS> rows;
  rows.init(a, b, hk, 0);

  int k0 = kbeg + KT * (w - 4);
  uint64_t live = 0;
  bool values = false;
  auto load = [&](int k) { return mask.load(k, min(kend, k + KT)); };
  uint32_t raw = load(k0 + 4 * KT);
  auto advance = [&]() {
    for (;;) {
      k0 += 4 * KT;
      if (k0 >= kend) return false;
      live = mask.live(raw);
      values = mask.values(raw);
      raw = load(k0 + 4 * KT);
      if (live) return true;
    }
  };
  auto issue = [&](int st) {
    lk.issue(kp + (int64_t)k0 * a.k_sn, live, 0, smem[w][st][0]);
    lv.issue(vp + (int64_t)k0 * a.v_sn, live, 0, smem[w][st][1]);
  };
  bool more = advance();
  if (more) issue(0);
  int st = 0;
  while (more) {
    const int kc = k0;
    const uint64_t lc = live;
    const bool vc = values;
    more = advance();
    if (more) {
      issue(st ^ 1);
      wait_vmcnt<2 * NI>();  // this tile's loads are older than the next one's
    } else {
      wait_vmcnt<0>();
    }
    rows.template step<1>(a, smem[w][st][0], smem[w][st][1], lc, vc ? mask.f : nullptr, kc);
    st ^= 1;
  }

  float* O = reinterpret_cast<float*>(&smem[0][0][0][0]);
  float* ML = O + 4 * 32 * OP;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    __syncthreads();
    const float lw = xor32_sum(rows.l[qb]), nw = xor32_sum(rows.n[qb]);
    float* ow = O + (w * 32 + (lane & 31)) * OP;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = rows.o[qb][db][4 * g4 + e];
        *reinterpret_cast<f32x4*>(ow + 32 * db + 8 * g4 + 4 * (lane >> 5)) = v;
      }
    if (lane < 32) {
      ML[3 * (w * 32 + lane)] = rows.m[qb];
      ML[3 * (w * 32 + lane) + 1] = lw;
      ML[3 * (w * 32 + lane) + 2] = nw;
    }
    __syncthreads();
    const int rl = threadIdx.x >> 3, r = 32 * qb + rl;
    if (r >= a.R) continue;
    float m = kXaLow, l = 0.f, n = 0.f, f[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) m = xa_max(m, ML[3 * (x * 32 + rl)]);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f[x] = fast_exp2((ML[3 * (x * 32 + rl)] - m) * a.c);
      l += f[x] * ML[3 * (x * 32 + rl) + 1];
      n += f[x] * ML[3 * (x * 32 + rl) + 2];
    }
    const int64_t pr = (bh * a.splits + split) * a.R + r;
    const float inv = xa_inverse(n, m);
    int g, i;
    xa_row(a, r, g, i);
    for (int d = 4 * (threadIdx.x & 7); d < a.D; d += 32) {
      f32x4 o = (f32x4)0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(O + (x * 32 + rl) * OP + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += f[x] * v[e];
      }
      if (a.splits == 1) {
        xa_store4<F16>(a, (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + d, o[0] * inv,
                       o[1] * inv, o[2] * inv, o[3] * inv);
      } else {
        *reinterpret_cast<f32x4*>(a.part_o + pr * a.D + d) = o;
      }
    }
    if ((threadIdx.x & 7) == 0) {
      if (a.splits == 1) {
        if (a.lse) xa_store_stats(a, bh * a.R + r, m, l);
      } else {
        a.part_ml[3 * pr] = m;
        a.part_ml[3 * pr + 1] = l;
        a.part_ml[3 * pr + 2] = n;
      }
    }
  }
}

// Joins the key splits: o = sum_s 2^(c (m_s - m)) o_s / sum_s 2^(c (m_s - m)) n_s
// in ascending order.  A thread forms four channels of one row.
template <bool F16>
__global__ __launch_bounds__(256) void xattn_join_kernel(XAttnArgs a) {
  const int dv = a.D / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = t / dv;
  if (row >= (int64_t)a.B * a.Hk * a.R) return;
  const int d = 4 * (int)(t - row * dv);
  const int64_t bh = row / a.R;
  const int r = (int)(row - bh * a.R);
  const float* ml = a.part_ml + 3 * (bh * a.splits * a.R + r);
  const float* po = a.part_o + (bh * a.splits * a.R + r) * a.D + d;
  float m = kXaLow;
  for (int s = 0; s < a.splits; ++s) m = xa_max(m, ml[3 * (int64_t)s * a.R]);
  float l = 0.f, n = 0.f;
  f32x4 o = (f32x4)0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float w = fast_exp2((ml[3 * (int64_t)s * a.R] - m) * a.c);
    l += w * ml[3 * (int64_t)s * a.R + 1];
    n += w * ml[3 * (int64_t)s * a.R + 2];
    const f32x4 v = *reinterpret_cast<const f32x4*>(po + (int64_t)s * a.R * a.D);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += w * v[e];
  }
  const float inv = xa_inverse(n, m);
  int g, i;
  xa_row(a, r, g, i);
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  xa_store4<F16>(a, (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + d, o[0] * inv, o[1] * inv,
                 o[2] * inv, o[3] * inv);
  if (a.lse && d == 0) xa_store_stats(a, row, m, l);
}

// The same for many splits (eight or more; fewer do better with a thread a row and
// four channels): a workgroup joins one row, its 256 threads 32 groups of four
// channels by eight ranges of splits (s mod 8), the ranges meeting in LDS in order.
// One token of 32 heads, 16384 states in 32 splits: 19.5 us in all against 30.
template <bool F16>
__global__ __launch_bounds__(256) void xattn_join_few_kernel(XAttnArgs a) {
  __shared__ float wt[kXaMaxSplits], part[8][32][4], red[4][3];
  const int64_t row = blockIdx.x, bh = row / a.R;
  const int r = (int)(row - bh * a.R), tid = threadIdx.x, w = tid >> 6;
  const float* ml = a.part_ml + 3 * (bh * a.splits * a.R + r);
  float m0 = kXaLow, l0 = 0.f, n0 = 0.f;  // this thread's split (at most 256)
  if (tid < a.splits) {
    m0 = ml[3 * (int64_t)tid * a.R];
    l0 = ml[3 * (int64_t)tid * a.R + 1];
    n0 = ml[3 * (int64_t)tid * a.R + 2];
  }
  float m = m0;
#pragma unroll
  for (int o = 32; o; o >>= 1) m = xa_max(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) red[w][0] = m;
  __syncthreads();
  m = xa_max(xa_max(red[0][0], red[1][0]), xa_max(red[2][0], red[3][0]));
  const float f = tid < a.splits ? fast_exp2((m0 - m) * a.c) : 0.f;
  wt[tid] = f;
  const float ls = lanes_sum<64>(f * l0), ns = lanes_sum<64>(f * n0);
  if ((tid & 63) == 0) {
    red[w][1] = ls;
    red[w][2] = ns;
  }
  __syncthreads();
  const float l = red[0][1] + red[1][1] + red[2][1] + red[3][1];
  const float n = red[0][2] + red[1][2] + red[2][2] + red[3][2];
  const int dg = tid & 31, q = tid >> 5, d = 4 * dg;
  f32x4 o = (f32x4)0.f;
  if (d < a.D) {
    const float* po = a.part_o + (bh * a.splits * a.R + r) * a.D + d;
#pragma unroll 4
    for (int s = q; s < a.splits; s += 8) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(po + (int64_t)s * a.R * a.D);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += wt[s] * v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[q][dg][e] = o[e];
  __syncthreads();
  if (q || d >= a.D) return;
#pragma unroll
  for (int x = 1; x < 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += part[x][dg][e];
  const float inv = xa_inverse(n, m);
  int g, i;
  xa_row(a, r, g, i);
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  xa_store4<F16>(a, (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + d, o[0] * inv, o[1] * inv,
                 o[2] * inv, o[3] * inv);
  if (a.lse && tid == 0) xa_store_stats(a, row, m, l);
}

// Up to 64 rows run on the streaming kernel, 32 or 64 at once; more on the tile
// kernel, 128 rows a workgroup, or 256 up to 64 channels where those fill the
// chip twice (512): each K and V fragment then feeds two products (64 channels,
// 4096 x 4096, 32 heads: 172 us against 186), while smaller grids do better with
// twice the workgroups (512 x 1500, 128 heads: 40 us against 45).  Either kernel
// splits the states only while it has less than one workgroup a CU: further
// splits cost more in prologues and partials than they level (16 tokens of 32
// heads, 8191 ragged states: 86 us at 256 workgroups, 90 at 512, 117 at 2048, before the
// wave number moved to the scalar side: 79 now).  A
// split has 256 states (four tiles for every two waves) or 128 (two tiles) at least
// and there are four or none (one token, 8 heads: 512 states in 7.4 us unsplit, 10.2
// split; one kv head of 65536 states in 13.5 us, with at most 64 splits 16; 128 rows
// of 8192 states in 12.4 us, from 512 states a split 18.4).
static void xattn_plan(XAttnArgs& a) {
  const bool few = a.R <= 64;
  const int64_t BH = (int64_t)a.B * a.Hk;
  a.qb = few ? (a.R > 32 ? 2 : 1) : a.D <= 64 && BH * ((a.R + 255) / 256) >= 512 ? 2 : 1;
  a.tiles = few ? 1 : (int)((a.R + 128 * a.qb - 1) / (128 * a.qb));
  int64_t s = 256 / (BH * a.tiles);
  const int64_t step = few ? 256 : 128;
  const int64_t most = a.Nk < 4 * step ? 1 : a.Nk / step;
  if (s > most) s = most;
  if (s > kXaMaxSplits) s = kXaMaxSplits;
  if (s < 1) s = 1;
  const int64_t tiles = (a.Nk + 63) / 64;
  a.chunk = (int)((tiles + s - 1) / s) * 64;
  a.splits = (int)((a.Nk + a.chunk - 1) / a.chunk);
  a.kw = !few && a.qb == 1 && BH * a.tiles * a.splits <= 256 && a.chunk >= 128 ? 2 : 1;
}

static int64_t xattn_part_floats(const XAttnArgs& a) {
  return a.splits > 1 ? (int64_t)a.B * a.Hk * a.splits * a.R * (a.D + 3) : 0;
}

// Sizes and strides as the kernels need them; 0 or an error code.
int xattn_check(XAttnArgs& a, const tpf_xattn_shape* s, double scale, const char* fn) {
  if (!s) return set_error(TPF_ERR_ARG, "%s: null shape", fn);
  if (s->B < 1 || s->H < 1 || s->Hk < 1 || s->Nq < 1 || s->Nk < 1 || s->D < 8 || s->D > 128 ||
      s->D % 8 || s->H % s->Hk)
    return set_error(TPF_ERR_SHAPE, "%s: bad shape B=%lld H=%lld Hk=%lld Nq=%lld Nk=%lld D=%lld", fn,
                     (long long)s->B, (long long)s->H, (long long)s->Hk, (long long)s->Nq,
                     (long long)s->Nk, (long long)s->D);
  const int64_t G = s->H / s->Hk, lim = (int64_t)1 << 30;
  if (s->Nk > lim || s->Nq > lim || s->B > lim || s->H > lim || G * s->Nq > lim ||
      (double)s->B * s->Hk * ((double)(G * s->Nq) / 64 + 1) * 64 > 2e9 ||
      s->B * s->Hk * ((G * s->Nq + 127) / 128) > kXaMaxGroups ||
      (double)s->B * s->Hk * ((double)s->Nk / 64 + 1) > 2e9)
    return set_error(TPF_ERR_SHAPE, "%s: too many rows or states", fn);
  for (int i = 0; i < 3; ++i) {
    const int64_t* st = i == 0 ? s->q_stride : i == 1 ? s->k_stride : s->v_stride;
    for (int j = 0; j < 3; ++j)
      if (st[j] < 0 || st[j] % 8)
        return set_error(TPF_ERR_SHAPE, "%s: strides must be multiples of 8 elements", fn);
    if (i && st[2] >= ((int64_t)1 << 23))
      return set_error(TPF_ERR_SHAPE, "%s: state stride too large", fn);
  }
  if (s->dtype != TPF_BF16 && s->dtype != TPF_F16)
    return set_error(TPF_ERR_ARG, "%s: dtype must be TPF_BF16 or TPF_F16", fn);
  if (s->mask_kind < 0 || s->mask_kind > 2 || s->mask_stride < 0)
    return set_error(TPF_ERR_ARG, "%s: bad mask", fn);
  if (!(scale > 1e-30) || !(scale < 1e30))  // it and its reciprocal in FP32
    return set_error(TPF_ERR_ARG, "%s: the scale must be between 1e-30 and 1e30", fn);
  a.q_sb = s->q_stride[0]; a.q_sh = s->q_stride[1]; a.q_sn = s->q_stride[2];
  a.k_sb = s->k_stride[0]; a.k_sh = s->k_stride[1]; a.k_sn = s->k_stride[2];
  a.v_sb = s->v_stride[0]; a.v_sh = s->v_stride[1]; a.v_sn = s->v_stride[2];
  a.mask_sb = s->mask_stride;
  a.mask_kind = s->mask_kind;
  a.B = (int)s->B; a.H = (int)s->H; a.Hk = (int)s->Hk; a.G = (int)G; a.Nq = (int)s->Nq;
  a.Nk = (int)s->Nk; a.D = (int)s->D; a.R = (int)(G * s->Nq);
  a.div_nq = make_fastdiv((uint32_t)s->Nq);
  a.c = (float)(scale * 1.4426950408889634);
  a.inv_scale = (float)(1.0 / scale);
  a.mask_floor = -1.5e38f;  // finite masks stay finite in raw units
  return TPF_OK;
}

template <int DP, bool F16, bool STATS>
static void xattn_launch(const XAttnArgs& a, hipStream_t s) {
  const int64_t groups = (int64_t)a.B * a.Hk * a.splits;
  const dim3 grid((unsigned)((groups * a.tiles + 7) / 8 * 8));
  if (a.R <= 64) {
    if (a.qb == 1) hipLaunchKernelGGL((xattn_few_kernel<DP, 1, F16, STATS>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((xattn_few_kernel<DP, 2, F16, STATS>), grid, dim3(256), 0, s, a);
    return;
  }
  if constexpr (DP <= 64) {
    if (a.qb == 2) {
      hipLaunchKernelGGL((xattn_fwd_kernel<DP, 2, F16, 1, STATS>), grid, dim3(256), 0, s, a);
      return;
    }
  }
  if (a.kw == 2) hipLaunchKernelGGL((xattn_fwd_kernel<DP, 1, F16, 2, STATS>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((xattn_fwd_kernel<DP, 1, F16, 1, STATS>), grid, dim3(256), 0, s, a);
}

template <bool F16, bool STATS>
static void xattn_pick(const XAttnArgs& a, hipStream_t s) {
  if (a.D <= 32) xattn_launch<32, F16, STATS>(a, s);
  else if (a.D <= 64) xattn_launch<64, F16, STATS>(a, s);
  else if (a.D <= 96) xattn_launch<96, F16, STATS>(a, s);
  else xattn_launch<128, F16, STATS>(a, s);
}

template <bool F16>
static void xattn_forward(const XAttnArgs& a, hipStream_t s) {
  if (a.lse) xattn_pick<F16, true>(a, s);
  else xattn_pick<F16, false>(a, s);
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.R, n = rows * (a.D / 4);
    if (a.splits >= 8)
      hipLaunchKernelGGL(xattn_join_few_kernel<F16>, dim3((unsigned)rows), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL(xattn_join_kernel<F16>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
  }
}

}  // namespace tpf

extern "C" int64_t tpf_xattn_forward_workspace_bytes(const tpf_xattn_shape* shape) {
  tpf::XAttnArgs a{};
  if (tpf::xattn_check(a, shape, 1.0, "tpf_xattn_forward_workspace_bytes")) return -1;
  tpf::xattn_plan(a);
  return tpf::xattn_part_floats(a) * 4;
}

static int xattn_forward_entry(const void* q, const void* k, const void* v, const void* mask, void* out,
                               float* lse, void* residual, void* workspace, int64_t workspace_bytes,
                               const tpf_xattn_shape* shape, double scale, void* stream,
                               const char* fn) {
  if (!q || !k || !v || !out) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  tpf::XAttnArgs a{};
  if (int rc = tpf::xattn_check(a, shape, scale, fn)) return rc;
  if ((a.mask_kind != 0) != (mask != nullptr))
    return tpf::set_error(TPF_ERR_ARG, "%s: mask pointer and mask kind disagree", fn);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)residual |
       (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  tpf::xattn_plan(a);
  const int64_t floats = tpf::xattn_part_floats(a);
  if (floats && (!workspace || workspace_bytes < floats * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.q = (const tpf::u16*)q; a.k = (const tpf::u16*)k; a.v = (const tpf::u16*)v;
  a.mask = mask; a.out = (tpf::u16*)out; a.res = (tpf::u16*)residual; a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_ml = floats ? a.part_o + (int64_t)a.B * a.Hk * a.splits * a.R * a.D : nullptr;
  if (shape->dtype == TPF_F16) tpf::xattn_forward<true>(a, (hipStream_t)stream);
  else tpf::xattn_forward<false>(a, (hipStream_t)stream);
  return tpf::check_launch(fn);
}

extern "C" int tpf_xattn_forward(const void* q, const void* k, const void* v, const void* mask,
                                 void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                 const tpf_xattn_shape* shape, double scale, void* stream) {
  return xattn_forward_entry(q, k, v, mask, out, lse, nullptr, workspace, workspace_bytes, shape, scale,
                             stream, "tpf_xattn_forward");
}

extern "C" int tpf_xattn_forward_shadow_bf16(const void* q, const void* k, const void* v,
                                             const void* mask, void* out, float* lse, void* residual,
                                             void* workspace, int64_t workspace_bytes,
                                             const tpf_xattn_shape* shape, double scale, void* stream) {
  const char* fn = "tpf_xattn_forward_shadow_bf16";
  if (!lse || !residual) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (shape && shape->dtype != TPF_BF16) return tpf::set_error(TPF_ERR_ARG, "%s: BF16 only", fn);
  return xattn_forward_entry(q, k, v, mask, out, lse, residual, workspace, workspace_bytes, shape, scale,
                             stream, fn);
}
