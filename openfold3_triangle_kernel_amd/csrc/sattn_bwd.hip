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
// sinks' tiles of states therefore have far more rows than the others, and without a window the
// first tiles twice the mean's; rows are split over workgroups whose 32-bit sums are added in
// ascending order, so results do not change from call to call.  7 products of 2 D operations a
// visible pair; bound by the matrix cores.  2 x 4096 tokens, 32 heads on 8 of 128: dQ 472 us (870
// TFLOP/s), dK and dV 606 (900), the fold 20.
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
  // The dK / dV launch: tiles of 128 states, the first `sunk` of them with sinks, whose rows
  // are in `splits` parts of schunk, those of the others in `parts` of rchunk; without a window
  // parts are the same runs of chunk_tiles tiles' rows for every tile (grad_unit).
  int ktiles, sunk, splits, schunk, rchunk, parts, chunk_tiles;
  SOrder order;
  float *part_k, *part_v;  // [parts, B*Hk, N, D], null without parts
  float *sunk_k, *sunk_v;  // [splits, B*Hk, 128 sunk, D]
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
  int64_t bh;
  int unit;
  if (!sa_unit(a.order, &bh, &unit)) return;
  const int b = (int)sa_div((uint32_t)bh, a.Hk), hk = (int)bh - b * a.Hk;
  const int t0 = (a.tiles - 1 - unit) * RT, r0 = t0 + w * 32;  // (later rows see more states)
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
  {
    // A row whose Q or dO is not finite has no delta: the other launch tells it by that.
    SExponents<false> x;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      x.add(q[s]);
      x.add(dO[s]);
    }
    if (xor32_sum(x.bad() ? 1.f : 0.f) != 0.f) delta = __builtin_nanf("");
  }
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
      sa_look<DP, XTileLoader<DP, KT, 4>::NI, false, true>(K, w, [&](int row) { V[row * DP + xa_swz<DP>(row) * 8] = 0x7fc0; });
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
        const uint32_t mine = bits >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((mine >> (8 * (e >> 2) + (e & 3))) & 1)) s[e] = 0.f;
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

// Direct 4-byte buffer -> LDS load: lane i writes dst_base + 4 i with element i of the n at src,
// zero past them.  (The lane's number is formed on the spot: with 128 channels one kept from
// before is a spilled one, whose return from memory would wait for every load under way.)
__device__ __forceinline__ void sg_lds4(const float* src, int n, void* dst_base) {
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_offset(dst_base));
  i32x4 rsrc = buffer_rsrc(src);
  rsrc[2] = __builtin_amdgcn_readfirstlane(4 * n);
  uint32_t at;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0\n\t"
               "v_lshlrev_b32 %0, 2, %0" : "=&v"(at));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(lds), "v"(at), "s"(rsrc) : "memory", "m0");
}

// 16 zero bytes.
__device__ const uint32_t kSaNone[4] = {0, 0, 0, 0};

// Unit `unit` of a head: its tile of states, which part of the rows that see it, and those
// rows (from a whole tile of rows on).  Without a window tile t is seen by all rows from
// 128 t G on; these run in the chunks that all tiles share: first the tiles' whole chunks, then
// each chunk's own tiles, the longest first.
__device__ __forceinline__ bool grad_unit(const SAttnGrad& ga, int unit, int* tile, int* part, int* rbeg,
                                          int* rend) {
  const SAttnArgs& a = ga.f;
  if (a.window >= a.N) {
    const int per = ga.chunk_tiles, whole = ga.parts * (ga.parts - 1) / 2 * per;
    int c, t;
    if (unit < whole) {
      c = 1;
      t = unit;
      while (t >= c * per) t -= c++ * per;
    } else {
      const int i = (int)sa_div(unit - whole, ga.parts);
      c = unit - whole - i * ga.parts;
      t = c * per + i;
      if (t >= ga.ktiles) return false;
    }
    *tile = t;
    *part = c;
    *rbeg = max(t, c * per) * 128 * a.G;
    *rend = (int)min((int64_t)a.R, ((int64_t)c + 1) * per * 128 * a.G);
    return true;
  }
  const int sinks = ga.sunk * ga.splits;
  int t, p, n, chunk = ga.rchunk;
  if (unit < sinks) {
    chunk = ga.schunk;
    t = (int)sa_div(unit, ga.splits);
    p = unit - t * ga.splits;
    n = a.R;
  } else {
    // (All tiles' first parts, then their second ones, ...: the last ones are the short ones.)
    p = (int)sa_div(unit - sinks, ga.ktiles - ga.sunk);
    t = unit - sinks - p * (ga.ktiles - ga.sunk) + ga.sunk;
    n = (int)min((int64_t)a.R, ((int64_t)min(t * 128 + 127, a.N - 1) + a.window) * a.G);
  }
  const int64_t from = (int64_t)t * 128 * a.G + (int64_t)p * chunk;
  *tile = t;
  *part = p;
  *rbeg = (int)min(from, (int64_t)n);
  *rend = (int)min(from + chunk, (int64_t)n);
  return true;
}

// dK and dV: four waves of 32 states each pass over tiles of RT of the rows that see them.
// A state's column of the tiles depends on that state alone, so dead states are left to run
// and their gradients written as 0.  Above 64 channels V stays in LDS (and at 128 the tiles
// have 32 rows), so that a wave fits 256 registers and two run on a SIMD; with 64 channels three
// do (16 heads on 4, 16384 tokens, window 1024: 10 % less time than with two).
template <int DP>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void sattn_dkdv_kernel(SAttnGrad ga) {
  constexpr bool VLDS = DP > 64;
  constexpr int RT = DP == 128 ? 32 : 64, TILE = RT * DP, DS = DP / 16, DB = DP / 32, CPR = DP / 8;
  constexpr int NI = RT * CPR / 256;
  static_assert(RT * CPR % 256 == 0, "whole instructions");
  __shared__ __attribute__((aligned(1024))) u16 smem[2][2][TILE];
  __shared__ __attribute__((aligned(1024))) float stats[2][2][64];
  __shared__ __attribute__((aligned(1024))) u16 vs[VLDS ? 128 * DP : 8];
  // What each thread keeps here instead of in registers: from 64 channels on none are left, and
  // a spilled one's return from memory would wait for every load under way (with 128 channels
  // the launch took 1026 us instead of 639 when this was changed; 606 now).
  constexpr int KEPT = DP == 128 || DP == 64 ? 2 + 2 * NI : DP > 64 ? 2 : 0;
  __shared__ int kept[KEPT ? KEPT : 1][256];
  const SAttnArgs& a = ga.f;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t BH = (int64_t)a.B * a.Hk;
  int64_t bh;
  int unit, tile, part, rbeg, rend;
  if (!sa_unit(ga.order, &bh, &unit) || !grad_unit(ga, unit, &tile, &part, &rbeg, &rend)) return;
  const int b = (int)sa_div((uint32_t)bh, a.Hk), hk = (int)bh - b * a.Hk;
  rbeg = sa_scalar(rbeg);
  rend = sa_scalar(rend);
  tile = sa_scalar(tile);
  const int k0 = tile * 128, kw = k0 + w * 32, k = kw + (lane & 31), kc = min(k, a.N - 1);
  // Rows that see this lane's state, and those that see all of the wave's.
  const int from = kc * a.G;
  const int to = a.window >= a.N || kc < a.sinks ? a.R : (int)min((int64_t)a.R, ((int64_t)kc + a.window) * a.G);
  const int wfrom = min(kw + 31, a.N - 1) * a.G;
  const int wto = sa_scalar(a.window >= a.N || kw + 31 < a.sinks
                      ? a.R : (int)min((int64_t)a.R, ((int64_t)min(kw, a.N - 1) + a.window) * a.G));
  const int tfrom = min(k0 + 127, a.N - 1) * a.G;  // and of the tile's
  const int tto = sa_scalar(a.window >= a.N || k0 + 127 < a.sinks ? a.R : (int)min((int64_t)a.R, ((int64_t)k0 + a.window) * a.G));

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

  // Fixed offsets of this lane's rows and chunks in a tile that begins with a token.  Groups that
  // do not divide the tile form addresses at every tile instead (2 x 4096 tokens of 128 channels:
  // 24 heads on 8 20.9 us a head, 28 on 4 20.2, 40 on 8 19.8, against 19.7 for 32 on 8).
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
    if constexpr (KEPT > 2) {
      kept[2 + 2 * t][threadIdx.x] = (int)qo[t];
      kept[3 + 2 * t][threadIdx.x] = (int)oo[t];
    }
  }
  if constexpr (KEPT > 0) {
    kept[0][threadIdx.x] = from;
    kept[KEPT ? 1 : 0][threadIdx.x] = to;
  }
  const u16* qbase = sa_scalar(a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh);
  const u16* obase = sa_scalar(ga.dout + ((int64_t)b * a.N * a.H + hk * a.G) * a.D);
  const float* sbase = sa_scalar((w == 0 ? ga.lse : ga.delta) + bh * a.R);
  auto issue = [&](int r0, int st) {
    char* dst = reinterpret_cast<char*>(smem[st][0]) + NI * w * 1024;
    if (near && r0 + RT <= rend) {
      const int i0 = (int)fdiv((uint32_t)r0, a.div_g);
      const i32x4 qr = buffer_rsrc(qbase + (int64_t)i0 * a.q_sn);
      const i32x4 dr = buffer_rsrc(obase + (int64_t)i0 * o_sn);
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        const uint32_t qa = KEPT > 2 ? (uint32_t)kept[KEPT > 2 ? 2 + 2 * t : 0][threadIdx.x] : qo[t];
        const uint32_t oa = KEPT > 2 ? (uint32_t)kept[KEPT > 2 ? 3 + 2 * t : 0][threadIdx.x] : oo[t];
        buf2lds16(qr, qa, dst + t * 1024);
        buf2lds16(dr, oa, dst + t * 1024 + TILE * 2);
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
          qs = qbase + g * a.q_sh + (int64_t)i * a.q_sn + 8 * chunk;
          os = obase + (int64_t)i * o_sn + g * a.D + 8 * chunk;
        }
        g2lds16(qs, dst + t * 1024);
        g2lds16(os, dst + t * 1024 + TILE * 2);
      }
    }
    if (w < 2) {  // wave 0: lse, 1: delta of the tile's rows
      // (Absent rows: no state sees them.)
      sg_lds4(sbase + r0, min(RT, a.R - r0), stats[st][w]);
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
        // Rows whose Q or dO is not finite (of those without a delta): the statistic makes p and
        // dS NaN.  All waves see the same.
        const float de = stats[st][1][lane & (RT - 1)];
        if (__ballot(de != de)) {
          auto mark = [&](int row) { stats[st][0][row] = __builtin_nanf(""); };
          sa_look<DP, NI, false, true>(Q, w, mark);
          sa_look<DP, NI, false, true>(dO, w, mark);
          lds_barrier();
        }
      }
#pragma unroll
      for (int rb = 0; rb < RT / 32; ++rb) {
        const int rr = r0 + 32 * rb;
        const bool whole = rr >= wfrom && rr + 32 <= wto;
        uint32_t bits = ~0u;
        if (!whole) {
          const int first = KEPT ? kept[0][threadIdx.x] : from, end = KEPT ? kept[KEPT ? 1 : 0][threadIdx.x] : to;
          bits = sa_ones32(end - 1 - rr) & ~sa_ones32(first - 1 - rr);
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
          const uint32_t mine = bits >> (4 * h);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!((mine >> (8 * (e >> 2) + (e & 3))) & 1)) s[e] = dp[e] = 0.f;
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
  // A tile's only part is its sum.
  const bool sunk = tile < ga.sunk;
  const bool alone = sunk ? ga.splits == 1 : ga.parts == 1 || (a.window >= a.N && tile >= (ga.parts - 1) * ga.chunk_tiles);
  const int64_t po = (((int64_t)part * BH + bh) * (sunk ? 128 * ga.sunk : a.N) + k) * a.D;
  sg_store<DB>(dk, a.D, ga.dk + b * ga.dk_s[0] + hk * ga.dk_s[1] + (int64_t)k * ga.dk_s[2],
               alone ? nullptr : (sunk ? ga.sunk_k : ga.part_k) + po, ga.scale, !live);
  sg_store<DB>(dv, a.D, ga.dv + b * ga.dv_s[0] + hk * ga.dv_s[1] + (int64_t)k * ga.dv_s[2],
               alone ? nullptr : (sunk ? ga.sunk_v : ga.part_v) + po, 1.f, !live);
}

// Sums the parts of the states' gradients in ascending order, four channels a thread, of the
// first n states; blockIdx.y 0: dK, 1: dV.
__global__ __launch_bounds__(256) void sattn_fold_kernel(SAttnGrad ga, int n) {
  const SAttnArgs& a = ga.f;
  u16* dst = blockIdx.y ? ga.dv : ga.dk;
  const int64_t* st = blockIdx.y ? ga.dv_s : ga.dk_s;
  const float scale = blockIdx.y ? 1.f : ga.scale;
  const int dv = a.D / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, row = t / dv, BH = (int64_t)a.B * a.Hk;
  if (row >= BH * n) return;
  const int d = 4 * (int)(t - row * dv);
  const int64_t bh = row / n;
  const int k = (int)(row - bh * n), b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  if (k >= a.N) return;
  const bool sunk = k < 128 * ga.sunk;
  const int first = a.window >= a.N ? k / 128 / ga.chunk_tiles : 0, end = sunk ? ga.splits : ga.parts;
  if (end - first == 1) return;  // (written at once)
  const float* part = sunk ? (blockIdx.y ? ga.sunk_v : ga.sunk_k) : (blockIdx.y ? ga.part_v : ga.part_k);
  const int64_t rows = sunk ? 128 * ga.sunk : a.N;
  f32x4 o = (f32x4)0.f;
  for (int s = first; s < end; ++s) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + (((int64_t)s * BH + bh) * rows + k) * a.D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += v[e];
  }
  uint2 x;
  x.x = xa_pair<false>(o[0] * scale, o[1] * scale);
  x.y = xa_pair<false>(o[2] * scale, o[3] * scale);
  *reinterpret_cast<uint2*>(dst + b * st[0] + hk * st[1] + (int64_t)k * st[2] + d) = x;
}

// Parts of the rows, so that the dK / dV launch has two workgroups a CU and none of them is
// much longer than the mean.
static int window_grad_plan(SAttnGrad& g, const char* fn) {
  SAttnArgs& a = g.f;
  const int64_t BH = (int64_t)a.B * a.Hk;
  a.tiles = (a.R + 127) / 128;
  a.splits = 1;
  g.ktiles = (a.N + 127) / 128;
  g.sunk = 0;
  g.splits = g.parts = 1;
  g.chunk_tiles = g.ktiles;
  g.rchunk = g.schunk = a.R;
  int64_t units;
  if (a.window >= a.N) {
    int64_t parts = (1024 + BH * (g.ktiles + 1) - 1) / (BH * (g.ktiles + 1));
    if (parts > 16) parts = 16;
    if (parts > 1) {
      g.chunk_tiles = (int)((g.ktiles + parts - 1) / parts);
      g.parts = (g.ktiles + g.chunk_tiles - 1) / g.chunk_tiles;
    }
    units = (int64_t)g.parts * (g.parts - 1) / 2 * g.chunk_tiles + (int64_t)g.parts * g.chunk_tiles;
  } else {
    g.sunk = (int)((((int64_t)a.sinks < a.N ? a.sinks : a.N) + 127) / 128);
    int64_t rows = ((int64_t)a.window + 128) * a.G;
    if (rows > a.R) rows = a.R;
    int64_t parts = 1024 / (BH * g.ktiles);
    if (parts > rows / 512) parts = rows / 512;
    if (parts < 1) parts = 1;
    // Of more parts than run at once the last is half as long as the others and fills the end of the
    // launch (16 heads on 4 of 64, 16384 tokens, window 1024: 212 us against 223).
    const bool uneven = parts > 1 && BH * g.ktiles * parts > 768;
    rows = (2 * rows / (2 * parts - uneven) + 64) / 64 * 64;
    g.parts = (int)parts;
    g.rchunk = (int)rows;
    if (g.sunk) {
      // The sinks' parts are as long as the others, unless more than 2048 would need memory.
      int64_t most = 2048 / (BH * g.sunk);
      if (most < 1) most = 1;
      int64_t chunk = (a.R + most - 1) / most;
      if (chunk < rows) chunk = rows;
      if (chunk < 512) chunk = 512;
      chunk = (chunk + 63) / 64 * 64;
      g.schunk = (int)chunk;
      g.splits = (int)((a.R + chunk - 1) / chunk);
    }
    units = (int64_t)g.sunk * g.splits + (int64_t)(g.ktiles - g.sunk) * g.parts;
  }
  if (BH * (units + 8) > kMaxGroups || (double)BH * a.N * (a.D / 4) / 256 + 1 > (double)kMaxGroups / 2)
    return set_error(TPF_ERR_SHAPE, "%s: too many states", fn);
  a.order = sa_order(BH, a.tiles);
  g.order = sa_order(BH, units);
  return TPF_OK;
}

// Workspace in floats: delta, then the parts.
struct WindowSpace {
  int64_t delta, part, sunk, total;
  explicit WindowSpace(const SAttnGrad& g) {
    const int64_t BH = (int64_t)g.f.B * g.f.Hk;
    delta = (BH * g.f.R + 3) / 4 * 4;
    part = g.parts > 1 ? g.parts * BH * g.f.N * g.f.D : 0;
    sunk = g.sunk && g.splits > 1 ? g.splits * BH * g.sunk * 128 * g.f.D : 0;
    total = delta + 2 * part + 2 * sunk;
  }
};

template <int DP>
static void window_grad_launch(const SAttnGrad& g, hipStream_t s) {
  hipLaunchKernelGGL((sattn_dq_kernel<DP>), dim3((unsigned)g.f.order.groups), dim3(256), 0, s, g);
  hipLaunchKernelGGL((sattn_dkdv_kernel<DP>), dim3((unsigned)g.order.groups), dim3(256), 0, s, g);
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
  g.part_k = w + ws.delta;
  g.part_v = g.part_k + ws.part;
  g.sunk_k = g.part_v + ws.part;
  g.sunk_v = g.sunk_k + ws.sunk;
  hipStream_t s = (hipStream_t)stream;
  if (a.D <= 32) tpf::window_grad_launch<32>(g, s);
  else if (a.D <= 64) tpf::window_grad_launch<64>(g, s);
  else if (a.D <= 96) tpf::window_grad_launch<96>(g, s);
  else tpf::window_grad_launch<128>(g, s);
  if (ws.part || ws.sunk) {
    const int states = ws.part || 128 * g.sunk > a.N ? a.N : 128 * g.sunk;
    const int64_t n = ((int64_t)a.B * a.Hk * states * (a.D / 4) + 255) / 256;
    hipLaunchKernelGGL(tpf::sattn_fold_kernel, dim3((unsigned)n, 2), dim3(256), 0, s, g, states);
  }
  return tpf::check_launch(fn);
}
