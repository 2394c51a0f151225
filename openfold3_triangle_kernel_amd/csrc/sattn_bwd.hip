// Causal self-attention: backward.
//
//   p_ij = 2^(c s_ij - lse_i) for the states j that row i sees, 0 for others
//   delta_i = dO_i . O_i (O with what its rounding dropped, where the forward kept that)
//   dS = p (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q,  dV = p^T dO
//
// over the rows and states of sattn.hpp in two launches, each of which rebuilds p, as cross
// attention's (xattn_bwd.hip): the first forms dQ and delta, a wave's lanes holding rows;
// the second dK and dV, a wave's lanes holding states.  A state is seen by a run of rows:
// from its own token's on, to the end of its window, or of the tokens for the sinks.  The
// sinks' tiles of states therefore have far more rows than the others; their rows are split
// over workgroups whose 32-bit sums are added in ascending order, so results do not change
// from call to call.  7 products of 2 D operations a visible pair; bound by the matrix cores.
#include "sattn.hpp"

namespace tpf {

struct SAttnGrad {
  SAttnArgs f;
  const u16 *o, *res, *dout;  // [B, N, H, D]; res null when not kept
  const float* lse;
  float* delta;  // [B, Hk, R]
  u16 *dq, *dk, *dv;
  int64_t dq_s[3], dk_s[3], dv_s[3];
  float scale;
  int ktiles;          // tiles of 128 states
  int sunk, splits, rchunk;  // tiles with sinks, parts of their rows, rows of a part
  float *part_k, *part_v;    // [splits, B*Hk, 128 sunk, D], null when there are no parts
};

// Four consecutive channels of a lane's row or state, as f32 partial or rounded with
// the scale.
template <int DB>
__device__ __forceinline__ void sg_store(const f32x16 (&o)[DB], int D, u16* dst, float* part, float scale,
                                         bool zero) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const int d = 32 * db + 8 * g4 + 4 * h;
      if (d < D) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = zero ? 0.f : o[db][4 * g4 + e];
        if (part) {
          *reinterpret_cast<f32x4*>(part + d) = v;
        } else {
          uint2 x;
          x.x = xa_pair<false>(v[0] * scale, v[1] * scale);
          x.y = xa_pair<false>(v[2] * scale, v[3] * scale);
          *reinterpret_cast<uint2*>(dst + d) = x;
        }
      }
    }
}

// dQ and delta: four waves of 32 rows share K and V tiles of 64 states.
template <int DP>
__global__ __launch_bounds__(256, 2) void sattn_dq_kernel(SAttnGrad ga) {
  constexpr int KT = 64, TILE = KT * DP, DS = DP / 16, DB = DP / 32, RT = 128;
  __shared__ __attribute__((aligned(1024))) u16 smem[2][2][TILE];
  const SAttnArgs& a = ga.f;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t T = xcd_order((int64_t)a.B * a.Hk * a.tiles);
  if (T < 0) return;
  const int64_t bh = T / a.tiles;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  const int t0 = sa_tile((int)(T - bh * a.tiles), a.tiles, a.order) * RT, r0 = t0 + w * 32;
  auto position = [&](int r) { return (int)fdiv((uint32_t)min(r, a.R - 1), a.div_g); };
  const int pmax = position(t0 + RT - 1), p0 = position(r0), p1 = position(r0 + 31);
  const SSpan span(position(t0), pmax, a.window, a.sinks);
  const int r = r0 + (lane & 31), rc = min(r, a.R - 1);
  const int i = position(r), g = rc - i * a.G;

  STiles<false, KT, 1> t;
  t.mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  t.init(span, 0, span.n, pmax + 1);
  const u16* kp = a.k + b * a.k_sb + hk * a.k_sh;
  const u16* vp = a.v + b * a.v_sb + hk * a.v_sh;
  XTileLoader<DP, KT, 4> lk, lv;
  lk.init(w, a.k_sn, a.D);
  lv.init(w, a.v_sn, a.D);

  bf16x8 q[DS], dO[DS];
  float delta = 0.f;
  {
    const u16* qp = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn;
    const int64_t oo = (((int64_t)b * a.N + i) * a.H + hk * a.G + g) * a.D;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = 16 * s + 8 * h;
      const bool in = d < a.D;
      q[s] = in ? *reinterpret_cast<const bf16x8*>(qp + d) : zero8();
      dO[s] = in ? *reinterpret_cast<const bf16x8*>(ga.dout + oo + d) : zero8();
      const bf16x8 o = in ? *reinterpret_cast<const bf16x8*>(ga.o + oo + d) : zero8();
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(bf2f(dO[s][e]), bf2f(o[e]), delta);
    }
    if (ga.res) {  // (a loop of its own: its loads go out together)
      bf16x8 x[DS];
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const int d = 16 * s + 8 * h;
        x[s] = d < a.D ? *reinterpret_cast<const bf16x8*>(ga.res + oo + d) : zero8();
      }
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(bf2f(dO[s][e]), bf2f(x[s][e]), delta);
    }
  }
  delta = xor32_sum(delta);
  const float lse = ga.lse[bh * a.R + rc];
  if (lane < 32 && r < a.R) ga.delta[bh * a.R + r] = delta;

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();

  auto issue = [&](int st) {
    lk.issue(kp + (int64_t)t.k0 * a.k_sn, t.live, w, smem[st][0]);
    lv.issue(vp + (int64_t)t.k0 * a.v_sn, t.live, w, smem[st][1]);
  };
  bool more = t.advance(a, span);
  if (more) issue(0);
  int st = 0;
  while (more) {
    const int kc = t.k0;
    const uint64_t lc = t.live;
    wait_vmcnt<0>();
    lds_barrier();
    more = t.advance(a, span);
    if (more) issue(st ^ 1);
    u16 *K = smem[st][0], *V = smem[st][1];
    st ^= 1;
    if (!sa_whole(a, position(t0), pmax, kc, KT)) {
      // A state whose K is not finite: its V makes dO V^T, and so dS, NaN.
      sa_clean<DP, XTileLoader<DP, KT, 4>::NI>(K, w, [&](int row) { V[row * DP + xa_swz<DP>(row) * 8] = 0x7fc0; });
      lds_barrier();
    }
    if (r0 >= a.R) continue;
    const bool whole = lc == ~0ull && sa_whole(a, p0, p1, kc, KT);
    uint64_t sees = ~0ull;
    if (!whole) {
      sees = sa_sees(a, i, kc, lc);
      if (__ballot(sees != 0) == 0) continue;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint32_t bits = (uint32_t)(sees >> (32 * kb));
      if (!whole && __ballot(bits != 0) == 0) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int d = 0; d < DS; ++d) s = mfma32(xa_frag<DP>(K, 32 * kb, d), q[d], s);
#pragma unroll
      for (int d = 0; d < DS; ++d) dp = mfma32(xa_frag<DP>(V, 32 * kb, d), dO[d], dp);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = fast_exp2(fmaf(s[e], a.c, -lse)) * (dp[e] - delta);
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((bits >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1)) s[e] = 0.f;
      }
      const bf16x8 x0 = xa_pack8<false>(s, 0), x1 = xa_pack8<false>(s, 8);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dq[db] = mfma32(xa_frag_t<DP>(K, 32 * kb, 0, db), x0, dq[db]);
        dq[db] = mfma32(xa_frag_t<DP>(K, 32 * kb, 1, db), x1, dq[db]);
      }
    }
  }
  if (r >= a.R) return;
  sg_store<DB>(dq, a.D,
               ga.dq + b * ga.dq_s[0] + (int64_t)(hk * a.G + g) * ga.dq_s[1] + (int64_t)i * ga.dq_s[2],
               nullptr, ga.scale, false);
}

// Direct 4-byte global -> LDS load: lane i writes dst_base + 4 i.
__device__ __forceinline__ void sg_lds4(const void* src, void* dst_base) {
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_offset(dst_base));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :: "v"(src), "s"(lds) : "memory", "m0");
}

// 16 zero bytes, then the log-sum-exp of an absent row: its p is 0.
__device__ const float kSaNone[8] = {0.f, 0.f, 0.f, 0.f, __builtin_inff(), 0.f, 0.f, 0.f};

// dK and dV: four waves of 32 states each pass over tiles of RT of the rows that see them.
// A state's column of the tiles depends on that state alone, so dead states are left to run
// and their gradients written as 0.  Above 64 channels V stays in LDS (and at 128 the tiles
// have 32 rows), so that a wave fits 256 registers and two run on a SIMD.
template <int DP>
__global__ __launch_bounds__(256, 2) void sattn_dkdv_kernel(SAttnGrad ga) {
  constexpr bool VLDS = DP > 64;
  constexpr int RT = DP == 128 ? 32 : 64, TILE = RT * DP, DS = DP / 16, DB = DP / 32, CPR = DP / 8;
  constexpr int NI = RT * CPR / 256;
  static_assert(RT * CPR % 256 == 0, "whole instructions");
  __shared__ __attribute__((aligned(1024))) u16 smem[2][2][TILE];
  __shared__ __attribute__((aligned(1024))) float stats[2][2][64];
  __shared__ __attribute__((aligned(1024))) u16 vs[VLDS ? 128 * DP : 8];
  const SAttnArgs& a = ga.f;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t BH = (int64_t)a.B * a.Hk;
  const int units = ga.sunk * ga.splits + ga.ktiles - ga.sunk;
  const int64_t T = xcd_order(BH * units);
  if (T < 0) return;
  const int64_t bh = T / units;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  // The sinks' parts first, then the tiles, the earlier ones (which have more rows) first.
  int unit = (int)(T - bh * units), tile, split = 0;
  if (unit < ga.sunk * ga.splits) {
    tile = unit / ga.splits;
    split = unit - tile * ga.splits;
  } else {
    tile = ga.ktiles - 1 - sa_tile(unit - ga.sunk * ga.splits, ga.ktiles - ga.sunk, a.order);
  }
  const int k0 = tile * 128, kw = k0 + w * 32, k = kw + (lane & 31), kc = min(k, a.N - 1);
  // Rows that see the tile's states, from a whole tile of rows on, and those of this part.
  const bool all = tile < ga.sunk || a.window >= a.N;
  int rbeg = (int)((int64_t)k0 * a.G / RT * RT);
  int rend = all ? a.R : (int)min((int64_t)a.R, ((int64_t)min(k0 + 127, a.N - 1) + a.window) * a.G);
  if (tile < ga.sunk) {
    const int64_t from = rbeg + (int64_t)split * ga.rchunk;
    rend = (int)min((int64_t)rend, from + ga.rchunk);
    rbeg = (int)min(from, (int64_t)rend);
  }
  // Rows that see this lane's state, and those that see all of the wave's.
  const int from = kc * a.G;
  const int to = a.window >= a.N || kc < a.sinks ? a.R : (int)min((int64_t)a.R, ((int64_t)kc + a.window) * a.G);
  const int wfrom = min(kw + 31, a.N - 1) * a.G;
  const int wto = a.window >= a.N || kw + 31 < a.sinks
                      ? a.R : (int)min((int64_t)a.R, ((int64_t)min(kw, a.N - 1) + a.window) * a.G);

  const int tfrom = min(k0 + 127, a.N - 1) * a.G;  // and of the tile's
  const int tto = a.window >= a.N || k0 + 127 < a.sinks ? a.R : (int)min((int64_t)a.R, ((int64_t)k0 + a.window) * a.G);

  bool live = k < a.N;
  if (a.mask) live = live && a.mask[b * a.mask_sb + kc] != 0;
  bf16x8 kf[DS], vf[VLDS ? 1 : DS];
  {
    const u16* kp = a.k + b * a.k_sb + hk * a.k_sh + (int64_t)kc * a.k_sn;
    const u16* vp = a.v + b * a.v_sb + hk * a.v_sh + (int64_t)kc * a.v_sn;
    const int row = w * 32 + (lane & 31);
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = 16 * s + 8 * h;
      const bool in = live && d < a.D;
      kf[s] = in ? *reinterpret_cast<const bf16x8*>(kp + d) : zero8();
      const bf16x8 x = in ? *reinterpret_cast<const bf16x8*>(vp + d) : zero8();
      if constexpr (VLDS)
        *reinterpret_cast<bf16x8*>(vs + row * DP + ((2 * s + h) ^ xa_swz<DP>(row)) * 8) = x;
      else
        vf[s] = x;
    }
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    dk[db] = zero16();
    dv[db] = zero16();
  }

  // Fixed offsets of this lane's rows and chunks in a tile that begins with a token.
  const int64_t o_sn = (int64_t)a.H * a.D;
  uint32_t qo[NI], oo[NI];
  bool near = RT % a.G == 0 && a.q_sn < (1 << 23) && a.q_sh < (1 << 23) && o_sn < (1 << 23);
#pragma unroll
  for (int t = 0; t < NI; ++t) {
    const int p = 64 * (NI * w + t) + lane, row = p / CPR;
    const int chunk = (p - row * CPR) ^ xa_swz<DP>(row);
    const int i = (int)fdiv((uint32_t)row, a.div_g), g = row - i * a.G;
    const bool in = near && 8 * chunk < a.D;
    qo[t] = in ? (uint32_t)(i * a.q_sn + g * a.q_sh + 8 * chunk) * 2u : kBufOOB;
    oo[t] = in ? (uint32_t)(i * o_sn + g * a.D + 8 * chunk) * 2u : kBufOOB;
  }
  auto issue = [&](int r0, int st) {
    char* dst = reinterpret_cast<char*>(smem[st][0]) + NI * w * 1024;
    if (near && r0 + RT <= rend) {
      const int i0 = (int)fdiv((uint32_t)r0, a.div_g);
      const i32x4 qr = buffer_rsrc(a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh + (int64_t)i0 * a.q_sn);
      const i32x4 dr = buffer_rsrc(ga.dout + (((int64_t)b * a.N + i0) * a.H + hk * a.G) * a.D);
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        buf2lds16(qr, qo[t], dst + t * 1024);
        buf2lds16(dr, oo[t], dst + t * 1024 + TILE * 2);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        const int p = 64 * (NI * w + t) + lane, row = p / CPR;
        const int chunk = (p - row * CPR) ^ xa_swz<DP>(row);
        const int r = r0 + row;
        const u16 *qs = (const u16*)kSaNone, *os = (const u16*)kSaNone;
        if (r < rend && 8 * chunk < a.D) {
          const int i = (int)fdiv((uint32_t)r, a.div_g), g = r - i * a.G;
          qs = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn + 8 * chunk;
          os = ga.dout + (((int64_t)b * a.N + i) * a.H + hk * a.G + g) * a.D + 8 * chunk;
        }
        g2lds16(qs, dst + t * 1024);
        g2lds16(os, dst + t * 1024 + TILE * 2);
      }
    }
    if (w < 2) {  // wave 0: lse, 1: delta of the tile's rows
      const float* src = w == 0 ? ga.lse : ga.delta;
      sg_lds4(lane < RT && r0 + lane < rend ? src + bh * a.R + r0 + lane : kSaNone + (w ? 0 : 4), stats[st][w]);
    }
  };

  const bool some = __syncthreads_or(live ? 1 : 0);
  if (some && rbeg < rend) {
    issue(rbeg, 0);
    int st = 0;
    for (int r0 = rbeg; r0 < rend; r0 += RT, st ^= 1) {
      wait_vmcnt<0>();
      lds_barrier();
      if (r0 + RT < rend) issue(r0 + RT, st ^ 1);
      u16 *Q = smem[st][0], *dO = smem[st][1];
      if (r0 < tfrom || r0 + RT > tto) {
        // A row whose Q or dO is not finite: its statistic makes p and dS NaN.
        auto mark = [&](int row) { stats[st][0][row] = __builtin_nanf(""); };
        sa_clean<DP, NI>(Q, w, mark);
        sa_clean<DP, NI>(dO, w, mark);
        lds_barrier();
      }
#pragma unroll
      for (int rb = 0; rb < RT / 32; ++rb) {
        const int rr = r0 + 32 * rb;
        const bool whole = rr >= wfrom && rr + 32 <= wto;
        uint32_t bits = ~0u;
        if (!whole) {
          bits = sa_ones32(to - 1 - rr) & ~sa_ones32(from - 1 - rr);
          if (__ballot(bits != 0) == 0) continue;
        }
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int d = 0; d < DS; ++d) s = mfma32(xa_frag<DP>(Q, 32 * rb, d), kf[d], s);
#pragma unroll
        for (int d = 0; d < DS; ++d)
          dp = mfma32(xa_frag<DP>(dO, 32 * rb, d),
                      VLDS ? xa_frag<DP>(vs, 32 * w, d) : vf[VLDS ? 0 : d], dp);
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(&stats[st][0][32 * rb + 8 * g4 + 4 * h]);
          const f32x4 de = *reinterpret_cast<const f32x4*>(&stats[st][1][32 * rb + 8 * g4 + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = fast_exp2(fmaf(s[4 * g4 + e], a.c, -ls[e]));
            s[4 * g4 + e] = p;
            dp[4 * g4 + e] = p * (dp[4 * g4 + e] - de[e]);
          }
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!((bits >> (8 * (e >> 2) + 4 * h + (e & 3))) & 1)) s[e] = dp[e] = 0.f;
        }
        bf16x8 pb[2], sb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          pb[t] = xa_pack8<false>(s, 8 * t);
          sb[t] = xa_pack8<false>(dp, 8 * t);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            dv[db] = mfma32(xa_frag_t<DP>(dO, 32 * rb, t, db), pb[t], dv[db]);
            dk[db] = mfma32(xa_frag_t<DP>(Q, 32 * rb, t, db), sb[t], dk[db]);
          }
      }
    }
  }
  if (k >= a.N) return;
  const bool part = ga.part_k && tile < ga.sunk;
  const int64_t po = (((int64_t)split * BH + bh) * (128 * ga.sunk) + k) * a.D;
  sg_store<DB>(dk, a.D, ga.dk + b * ga.dk_s[0] + hk * ga.dk_s[1] + (int64_t)k * ga.dk_s[2],
               part ? ga.part_k + po : nullptr, ga.scale, !live);
  sg_store<DB>(dv, a.D, ga.dv + b * ga.dv_s[0] + hk * ga.dv_s[1] + (int64_t)k * ga.dv_s[2],
               part ? ga.part_v + po : nullptr, 1.f, !live);
}

// Sums the parts [splits, BH, n, D] of the sinks' states in ascending order, four channels
// a thread; blockIdx.y 0: dK, 1: dV.
__global__ __launch_bounds__(256) void sattn_fold_kernel(SAttnGrad ga) {
  const SAttnArgs& a = ga.f;
  const float* part = blockIdx.y ? ga.part_v : ga.part_k;
  u16* dst = blockIdx.y ? ga.dv : ga.dk;
  const int64_t* st = blockIdx.y ? ga.dv_s : ga.dk_s;
  const float scale = blockIdx.y ? 1.f : ga.scale;
  const int n = 128 * ga.sunk, dv = a.D / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, row = t / dv, BH = (int64_t)a.B * a.Hk;
  if (row >= BH * n) return;
  const int d = 4 * (int)(t - row * dv);
  const int64_t bh = row / n;
  const int k = (int)(row - bh * n), b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  if (k >= a.N) return;
  f32x4 o = (f32x4)0.f;
  for (int s = 0; s < ga.splits; ++s) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + ((int64_t)s * BH * n + row) * a.D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += v[e];
  }
  uint2 x;
  x.x = xa_pair<false>(o[0] * scale, o[1] * scale);
  x.y = xa_pair<false>(o[2] * scale, o[3] * scale);
  *reinterpret_cast<uint2*>(dst + b * st[0] + hk * st[1] + (int64_t)k * st[2] + d) = x;
}

// The sinks' tiles are split into parts of about as many rows as the other tiles have.
static int window_grad_plan(SAttnGrad& g, const char* fn) {
  SAttnArgs& a = g.f;
  const int64_t BH = (int64_t)a.B * a.Hk;
  a.tiles = (a.R + 127) / 128;
  a.splits = 1;
  g.ktiles = (a.N + 127) / 128;
  g.sunk = a.window < a.N ? (int)((((int64_t)a.sinks < a.N ? a.sinks : a.N) + 127) / 128) : 0;
  g.splits = 1;
  g.rchunk = a.R;
  if (g.sunk) {
    int64_t rows = ((int64_t)a.window + 128) * a.G;
    if (rows < 1024) rows = 1024;
    rows = (rows + 63) / 64 * 64;
    if (rows < a.R) {
      g.rchunk = (int)rows;
      g.splits = (int)((a.R + rows - 1) / rows);
    }
  }
  if (BH * ((int64_t)g.sunk * g.splits + g.ktiles) > kXaMaxGroups ||
      BH * g.sunk * 128 * (a.D / 4) / 256 + 1 > kXaMaxGroups / 2)
    return set_error(TPF_ERR_SHAPE, "%s: too many states", fn);
  return TPF_OK;
}

// Workspace in floats: delta, then the parts.
struct WindowSpace {
  int64_t delta, part, total;
  explicit WindowSpace(const SAttnGrad& g) {
    const int64_t BH = (int64_t)g.f.B * g.f.Hk;
    delta = (BH * g.f.R + 3) / 4 * 4;
    part = g.splits > 1 ? g.splits * BH * g.sunk * 128 * g.f.D : 0;
    total = delta + 2 * part;
  }
};

template <int DP>
static void window_grad_launch(const SAttnGrad& g, hipStream_t s) {
  const SAttnArgs& a = g.f;
  const int64_t BH = (int64_t)a.B * a.Hk;
  const int64_t n1 = BH * a.tiles, n2 = BH * ((int64_t)g.sunk * g.splits + g.ktiles - g.sunk);
  hipLaunchKernelGGL((sattn_dq_kernel<DP>), dim3((unsigned)((n1 + 7) / 8 * 8)), dim3(256), 0, s, g);
  hipLaunchKernelGGL((sattn_dkdv_kernel<DP>), dim3((unsigned)((n2 + 7) / 8 * 8)), dim3(256), 0, s, g);
}

}  // namespace tpf

extern "C" int64_t tpf_window_backward_workspace_bytes(const tpf_window_shape* shape) {
  tpf::SAttnGrad g{};
  const char* fn = "tpf_window_backward_workspace_bytes";
  if (tpf::window_check(g.f, shape, 1.0, fn) || tpf::window_grad_plan(g, fn)) return -1;
  return tpf::WindowSpace(g).total * 4;
}

extern "C" int tpf_window_backward_bf16(const void* q, const void* k, const void* v, const void* mask,
                                        const void* out, const void* residual, const void* dout,
                                        const float* lse, void* dq, void* dk, void* dv, void* workspace,
                                        int64_t workspace_bytes, const tpf_window_shape* shape,
                                        const int64_t* grad_strides, double scale, void* stream) {
  const char* fn = "tpf_window_backward_bf16";
  if (!q || !k || !v || !out || !dout || !lse || !dq || !dk || !dv || !workspace || !grad_strides)
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  tpf::SAttnGrad g{};
  tpf::SAttnArgs& a = g.f;
  if (int rc = tpf::window_check(a, shape, scale, fn)) return rc;
  if (shape->dtype != TPF_BF16) return tpf::set_error(TPF_ERR_ARG, "%s: BF16 only", fn);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)residual | (uintptr_t)dout |
       (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  for (int i = 0; i < 9; ++i)
    if (grad_strides[i] < 0 || grad_strides[i] % 8)
      return tpf::set_error(TPF_ERR_SHAPE, "%s: gradient strides must be multiples of 8 elements", fn);
  if (int rc = tpf::window_grad_plan(g, fn)) return rc;
  const tpf::WindowSpace ws(g);
  if (workspace_bytes < ws.total * 4)
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.q = (const tpf::u16*)q; a.k = (const tpf::u16*)k; a.v = (const tpf::u16*)v;
  a.mask = (const uint8_t*)mask;
  g.o = (const tpf::u16*)out; g.res = (const tpf::u16*)residual; g.dout = (const tpf::u16*)dout; g.lse = lse;
  g.dq = (tpf::u16*)dq; g.dk = (tpf::u16*)dk; g.dv = (tpf::u16*)dv;
  for (int i = 0; i < 3; ++i) {
    g.dq_s[i] = grad_strides[i];
    g.dk_s[i] = grad_strides[3 + i];
    g.dv_s[i] = grad_strides[6 + i];
  }
  g.scale = (float)scale;
  float* w = (float*)workspace;
  g.delta = w;
  g.part_k = ws.part ? w + ws.delta : nullptr;
  g.part_v = ws.part ? w + ws.delta + ws.part : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (a.D <= 32) tpf::window_grad_launch<32>(g, s);
  else if (a.D <= 64) tpf::window_grad_launch<64>(g, s);
  else if (a.D <= 96) tpf::window_grad_launch<96>(g, s);
  else tpf::window_grad_launch<128>(g, s);
  if (ws.part) {
    const int64_t n = ((int64_t)a.B * a.Hk * g.sunk * 128 * (a.D / 4) + 255) / 256;
    hipLaunchKernelGGL(tpf::sattn_fold_kernel, dim3((unsigned)n, 2), dim3(256), 0, s, g);
  }
  return tpf::check_launch(fn);
}
