// Cross attention: backward.
//
//   p_ij = 2^(c s_ij - lse_i) (with additive masks 2^(c (s_ij + m_j - max_i) -
//   log2 sum_i), whatever the masks' size),  delta_i = dO_i . O_i,  dS = p (dO V^T - delta)
// (O with what its rounding dropped where the forward kept that: dO V^T and delta
// nearly cancel in what the states' values have in common)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = p^T dO
//
// over the rows and states of xattn.hpp, in two launches that each rebuild p
// (7 products of 2 R Nk D operations instead of the 5 that a single pass with
// dQ partials in memory would take; the partials of one pass are R D floats for
// every tile of states).  The first forms dQ and delta, a wave's lanes holding
// rows; the second dK and dV, a wave's lanes holding states.  Both feed the S
// tile back into the matrix cores as it stands.  Sums over rows or states that
// are split over workgroups are folded in ascending order, so results do not
// change from call to call.  32 heads, 4096 x 4096 x 128: 885 us, 777 TFLOP/s of the
// five products (1087 of the seven executed); 64 channels 488 us.
#include "gemm_core.hpp"  // xcd_order
#include "tpf_status.hpp"
#include "xattn.hpp"

namespace tpf {

struct XAttnGrad {
  XAttnArgs f;           // operands; f.splits / f.chunk: states of the dQ launch
  const u16 *o, *res, *dout;  // [B, Nq, H, D]; res null when not kept
  const float *lse, *top;  // log-sum-exp; with additive masks log2 of the sum and the maximum
  float* delta;          // [B, Hk, R]
  u16 *dq, *dk, *dv;
  int64_t dq_s[3], dk_s[3], dv_s[3];
  float scale;
  float* part_q;         // [splits, B*Hk, R, D], null when unsplit
  float *part_k, *part_v;  // [rsplits, B*Hk, Nk, D]
  int rsplits, rchunk;   // row splits of the dK / dV launch, rows per split
  int rkw;               // its groups of four waves
  int ktiles;            // state tiles of the dK / dV launch
};

// 16 zero bytes, then the log-sum-exp (or log2 of the sum) of an absent row: its
// p is 0.
__device__ const float kXaNone[8] = {0.f, 0.f, 0.f, 0.f, __builtin_inff(), 0.f, 0.f, 0.f};

// Direct 4-byte global -> LDS load: lane i writes dst_base + 4 i.
__device__ __forceinline__ void g2lds4(const void* src, void* dst_base) {
  const unsigned lds = __builtin_amdgcn_readfirstlane(lds_offset(dst_base));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :: "v"(src), "s"(lds) : "memory", "m0");
}

// Four consecutive channels of a lane's row or state, as f32 partial or
// rounded with the scale.
template <int DB>
__device__ __forceinline__ void xg_store(const f32x16 (&o)[DB], int D, u16* dst, float* part,
                                         float scale, bool zero) {
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

// dQ and delta: four waves of 32 rows share K and V tiles of 64 states.  KW = 2:
// two groups of four waves take the row tile's states in turn and add their sums in
// LDS, for grids that give a CU one workgroup (as in the forward).
template <int DP, bool ADD, int KW>
__global__ __launch_bounds__(256 * KW, 2) void xattn_dq_kernel(XAttnGrad ga) {
  constexpr int KT = 64, TILE = KT * DP, DS = DP / 16, DB = DP / 32;
  __shared__ __attribute__((aligned(1024))) u16 smem[KW][2][2][TILE];
  const XAttnArgs& a = ga.f;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = KW == 2 ? wave >> 2 : 0, w = wave & 3, lane = threadIdx.x & 63;
  const int64_t T = xcd_order((int64_t)a.B * a.Hk * a.splits * a.tiles);
  if (T < 0) return;
  const int tile = (int)(T % a.tiles);
  const int64_t u = T / a.tiles;
  const int split = (int)(u % a.splits);
  const int64_t bh = u / a.splits;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  const int r = tile * 128 + w * 32 + (lane & 31), rc = min(r, a.R - 1);
  const int kbeg = split * a.chunk, kend = min(a.Nk, kbeg + a.chunk);
  const u16* kp = a.k + b * a.k_sb + hk * a.k_sh;
  const u16* vp = a.v + b * a.v_sb + hk * a.v_sh;

  XTiles<KW> t;
  t.init(a, b, kbeg, kend);
  XTileLoader<DP, KT, 4> lk, lv;
  lk.init(w, a.k_sn, a.D);
  lv.init(w, a.v_sn, a.D);

  bf16x8 q[DS], dO[DS];
  float delta = 0.f;
  int g, i;
  xa_row(a, rc, g, i);
  {
    const u16* qp = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn;
    const int64_t oo = (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
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
        const int d = 16 * s + 8 * (lane >> 5);
        x[s] = d < a.D ? *reinterpret_cast<const bf16x8*>(ga.res + oo + d) : zero8();
      }
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(bf2f(dO[s][e]), bf2f(x[s][e]), delta);
    }
  }
  delta = xor32_sum(delta);
  const float lse = ga.lse[bh * a.R + rc], top = ADD ? ga.top[bh * a.R + rc] : 0.f;
  if (split == 0 && group == 0 && lane < 32 && r < a.R) ga.delta[bh * a.R + r] = delta;

  f32x16 dq[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dq[db] = zero16();

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
    const u16 *K = smem[group][st][0], *V = smem[group][st][1];
    st ^= 1;
    if (KW == 2 && !lc) continue;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int d = 0; d < DS; ++d) s = mfma32(xa_frag<DP>(K, 32 * kb, d), q[d], s);
#pragma unroll
      for (int d = 0; d < DS; ++d) dp = mfma32(xa_frag<DP>(V, 32 * kb, d), dO[d], dp);
      if (lc != ~0ull || vc)
        xa_mask32(s, (uint32_t)(lc >> (32 * kb)), vc ? t.mask.f : nullptr, kc + 32 * kb, a.Nk,
                  a.inv_scale, a.mask_floor);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[e] = fast_exp2(fmaf(ADD ? s[e] - top : s[e], a.c, -lse)) * (dp[e] - delta);
      const bf16x8 p0 = xa_pack8<false>(s, 0), p1 = xa_pack8<false>(s, 8);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        dq[db] = mfma32(xa_frag_t<DP>(K, 32 * kb, 0, db), p0, dq[db]);
        dq[db] = mfma32(xa_frag_t<DP>(K, 32 * kb, 1, db), p1, dq[db]);
      }
    }
  }
  if constexpr (KW == 2) {
    static_assert(sizeof(smem) >= 4 * DB * 4096, "the join fits");
    char* lds = reinterpret_cast<char*>(&smem[0][0][0][0]);
    __syncthreads();
    if (group) xa_give<DB>(lds, w, dq);
    __syncthreads();
    if (group) return;
    xa_take<DB>(lds, w, dq, 1.f, 1.f);
  }
  if (r >= a.R) return;
  const int64_t BH = (int64_t)a.B * a.Hk;
  xg_store<DB>(dq, a.D,
               ga.dq + b * ga.dq_s[0] + (int64_t)(hk * a.G + g) * ga.dq_s[1] + (int64_t)i * ga.dq_s[2],
               ga.part_q ? ga.part_q + (((int64_t)split * BH + bh) * a.R + r) * a.D : nullptr, ga.scale,
               false);
}

// dK and dV: four waves of 32 states each pass over tiles of RT rows of Q and
// dO.  A state's column of the tiles depends on that state alone, so dead
// states are left to run and their gradients written as 0.  Above 64 channels
// V stays in LDS (and at 128 the tiles have 32 rows), so that a wave fits 256
// registers and two run on a SIMD.  A tile inside one query head (all of them when Nq is a
// multiple of RT) is loaded at fixed lane offsets from its first row; others
// find each row's address.  KW = 2: two groups of four waves take the row tiles in
// turn for the same states and add their sums in LDS.
template <int DP, bool ADD, int KW>
__global__ __launch_bounds__(256 * KW, 2) void xattn_dkdv_kernel(XAttnGrad ga) {
  constexpr bool VLDS = DP > 64;
  constexpr int RT = DP == 128 ? 32 : 64, TILE = RT * DP, DS = DP / 16, DB = DP / 32, CPR = DP / 8;
  constexpr int NI = RT * CPR / 256;
  static_assert(RT * CPR % 256 == 0, "whole instructions");
  __shared__ __attribute__((aligned(1024))) u16 smem[KW][2][2][TILE];
  __shared__ __attribute__((aligned(1024))) float stats[KW][2][ADD ? 3 : 2][64];
  __shared__ __attribute__((aligned(1024))) u16 vs[VLDS ? 128 * DP : 8];
  const XAttnArgs& a = ga.f;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = KW == 2 ? wave >> 2 : 0, w = wave & 3, lane = threadIdx.x & 63, h = lane >> 5;
  const int64_t BH = (int64_t)a.B * a.Hk;
  const int64_t T = xcd_order(BH * ga.rsplits * ga.ktiles);
  if (T < 0) return;
  const int tile = (int)(T % ga.ktiles);
  const int64_t u = T / ga.ktiles;
  const int split = (int)(u % ga.rsplits);
  const int64_t bh = u / ga.rsplits;
  const int b = (int)(bh / a.Hk), hk = (int)(bh - (int64_t)b * a.Hk);
  const int k = tile * 128 + w * 32 + (lane & 31), kc = min(k, a.Nk - 1);
  const int rbeg = split * ga.rchunk, rend = min(a.R, rbeg + ga.rchunk);

  bool live = k < a.Nk;
  float add = 0.f;
  if (a.mask_kind == kMaskBool) {
    live = live && ((const uint8_t*)a.mask)[(int64_t)b * a.mask_sb + kc] != 0;
  } else if (a.mask_kind == kMaskF32) {
    const uint32_t m = ((const uint32_t*)a.mask)[(int64_t)b * a.mask_sb + kc];
    live = live && m != 0xff800000u;
    add = live ? xa_raw_mask(m, a.inv_scale, a.mask_floor) : 0.f;
  }
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
      if constexpr (VLDS)  // (both groups write the same values)
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

  // Fixed offsets of this lane's rows and chunks in a tile inside one head.
  const int64_t o_sn = (int64_t)a.H * a.D;
  uint32_t qo[NI], oo[NI];
#pragma unroll
  for (int t = 0; t < NI; ++t) {
    const int p = 64 * (NI * w + t) + lane, row = p / CPR;
    const int chunk = (p - row * CPR) ^ xa_swz<DP>(row);
    qo[t] = 8 * chunk < a.D ? (uint32_t)(row * a.q_sn + 8 * chunk) * 2u : kBufOOB;
    oo[t] = 8 * chunk < a.D ? (uint32_t)(row * o_sn + 8 * chunk) * 2u : kBufOOB;
  }
  const bool near = a.q_sn < (1 << 23) && o_sn < (1 << 23);  // 64 rows within 2 GiB
  auto issue = [&](int r0, int st) {
    char* dst = reinterpret_cast<char*>(smem[group][st][0]) + NI * w * 1024;
    int g0, i0;
    xa_row(a, min(r0, a.R - 1), g0, i0);
    if (near && i0 + RT <= a.Nq && r0 + RT <= rend) {
      const i32x4 qr = buffer_rsrc(a.q + b * a.q_sb + (int64_t)(hk * a.G + g0) * a.q_sh +
                                   (int64_t)i0 * a.q_sn);
      const i32x4 dr = buffer_rsrc(ga.dout + (((int64_t)b * a.Nq + i0) * a.H + hk * a.G + g0) * a.D);
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
        const u16 *qs = (const u16*)kXaNone, *os = (const u16*)kXaNone;
        if (r < rend && 8 * chunk < a.D) {
          int g, i;
          xa_row(a, r, g, i);
          qs = a.q + b * a.q_sb + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn + 8 * chunk;
          os = ga.dout + (((int64_t)b * a.Nq + i) * a.H + hk * a.G + g) * a.D + 8 * chunk;
        }
        g2lds16(qs, dst + t * 1024);
        g2lds16(os, dst + t * 1024 + TILE * 2);
      }
    }
    if (w < (ADD ? 3 : 2)) {  // wave 0: lse, 1: delta, 2: maxima of the tile's rows
      const float* src = w == 0 ? ga.lse : w == 1 ? ga.delta : ga.top;
      g2lds4(lane < RT && r0 + lane < rend ? src + bh * a.R + r0 + lane : kXaNone + (w ? 0 : 4),
             stats[group][st][w]);
    }
  };

  const bool some = __syncthreads_or(live ? 1 : 0);
  if (some) {
    // A group past the last row loads absent rows, whose p is 0: no branch.
    const int mine = RT * group;
    issue(rbeg + mine, 0);
    int st = 0;
    for (int r0 = rbeg; r0 < rend; r0 += RT * KW, st ^= 1) {
      wait_vmcnt<0>();
      lds_barrier();
      if (r0 + RT * KW < rend) issue(r0 + RT * KW + mine, st ^ 1);
      const u16 *Q = smem[group][st][0], *dO = smem[group][st][1];
#pragma unroll
      for (int rb = 0; rb < RT / 32; ++rb) {
        f32x16 s = zero16(), dp = zero16();
#pragma unroll
        for (int d = 0; d < DS; ++d) s = mfma32(xa_frag<DP>(Q, 32 * rb, d), kf[d], s);
#pragma unroll
        for (int d = 0; d < DS; ++d)
          dp = mfma32(xa_frag<DP>(dO, 32 * rb, d),
                      VLDS ? xa_frag<DP>(vs, 32 * w, d) : vf[VLDS ? 0 : d], dp);
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(&stats[group][st][0][32 * rb + 8 * g4 + 4 * h]);
          const f32x4 de = *reinterpret_cast<const f32x4*>(&stats[group][st][1][32 * rb + 8 * g4 + 4 * h]);
          f32x4 tp;
          if (ADD) tp = *reinterpret_cast<const f32x4*>(&stats[group][st][ADD ? 2 : 0][32 * rb + 8 * g4 + 4 * h]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = ADD ? (s[4 * g4 + e] + add) - tp[e] : s[4 * g4 + e];
            const float p = fast_exp2(fmaf(x, a.c, -ls[e]));
            s[4 * g4 + e] = p;
            dp[4 * g4 + e] = p * (dp[4 * g4 + e] - de[e]);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bf16x8 pb = xa_pack8<false>(s, 8 * t), db_ = xa_pack8<false>(dp, 8 * t);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            dv[db] = mfma32(xa_frag_t<DP>(dO, 32 * rb, t, db), pb, dv[db]);
            dk[db] = mfma32(xa_frag_t<DP>(Q, 32 * rb, t, db), db_, dk[db]);
          }
        }
      }
    }
  }
  if constexpr (KW == 2) {
    static_assert(sizeof(smem) >= 4 * DB * 4096, "the join fits");
    char* lds = reinterpret_cast<char*>(&smem[0][0][0][0]);
    __syncthreads();
    if (group) xa_give<DB>(lds, w, dk);
    __syncthreads();
    if (!group) xa_take<DB>(lds, w, dk, 1.f, 1.f);
    __syncthreads();
    if (group) xa_give<DB>(lds, w, dv);
    __syncthreads();
    if (group) return;
    xa_take<DB>(lds, w, dv, 1.f, 1.f);
  }
  if (k >= a.Nk) return;
  const int64_t po = (((int64_t)split * BH + bh) * a.Nk + k) * a.D;
  xg_store<DB>(dk, a.D, ga.dk + b * ga.dk_s[0] + hk * ga.dk_s[1] + (int64_t)k * ga.dk_s[2],
               ga.part_k ? ga.part_k + po : nullptr, ga.scale, !live);
  xg_store<DB>(dv, a.D, ga.dv + b * ga.dv_s[0] + hk * ga.dv_s[1] + (int64_t)k * ga.dv_s[2],
               ga.part_v ? ga.part_v + po : nullptr, 1.f, !live);
}

// Sums the partials [splits, BH, n, D] of the split launches in ascending order,
// four channels a thread: workgroups [0, first_k) dQ, [first_k, first_v) dK, the rest
// dV.
__global__ __launch_bounds__(256) void xattn_fold_kernel(XAttnGrad ga, unsigned first_k,
                                                         unsigned first_v) {
  const XAttnArgs& a = ga.f;
  const int which = blockIdx.x < first_k ? 0 : blockIdx.x < first_v ? 1 : 2;
  const int64_t block = blockIdx.x - (which == 0 ? 0 : which == 1 ? first_k : first_v);
  const float* part = which == 0 ? ga.part_q : which == 1 ? ga.part_k : ga.part_v;
  u16* dst = which == 0 ? ga.dq : which == 1 ? ga.dk : ga.dv;
  const int64_t* st = which == 0 ? ga.dq_s : which == 1 ? ga.dk_s : ga.dv_s;
  const float scale = which == 2 ? 1.f : ga.scale;
  const int n = which ? a.Nk : a.R, splits = which ? ga.rsplits : a.splits, dv = a.D / 4;
  const int64_t t = block * 256 + threadIdx.x, row = t / dv;
  const int64_t BH = (int64_t)a.B * a.Hk;
  if (row >= BH * n) return;
  const int d = 4 * (int)(t - row * dv);
  f32x4 o = (f32x4)0.f;
  for (int s = 0; s < splits; ++s) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + ((int64_t)s * BH * n + row) * a.D + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += v[e];
  }
  const int64_t bh = row / n;
  const int r = (int)(row - bh * n);
  const int b = (int)(bh / a.Hk);
  int head = (int)(bh - (int64_t)b * a.Hk), pos = r;
  if (which == 0) {
    int g, i;
    xa_row(a, r, g, i);
    head = head * a.G + g;
    pos = i;
  }
  uint2 x;
  x.x = xa_pair<false>(o[0] * scale, o[1] * scale);
  x.y = xa_pair<false>(o[2] * scale, o[3] * scale);
  *reinterpret_cast<uint2*>(dst + b * st[0] + head * st[1] + (int64_t)pos * st[2] + d) = x;
}

// A launch that leaves CUs without a workgroup is split, 256 states or rows at least
// to a split; one workgroup a CU has two groups of waves (forward and backward of 32
// heads, 1024 x 1024 x 128: 138 us against 165 with up to 512 workgroups of one).
static void split_axis(int64_t groups, int64_t n, int64_t tile, int* splits, int* chunk, int* kw) {
  int64_t s = 256 / groups;
  if (s > (n + 255) / 256) s = (n + 255) / 256;
  if (s > 16) s = 16;
  if (s < 1) s = 1;
  const int64_t t = (n + tile - 1) / tile;
  *chunk = (int)((t + s - 1) / s * tile);
  *splits = (int)((n + *chunk - 1) / *chunk);
  *kw = groups * *splits <= 256 && *chunk >= 128 ? 2 : 1;
}

static int grad_plan(XAttnGrad& g, const char* fn) {
  XAttnArgs& a = g.f;
  const int64_t BH = (int64_t)a.B * a.Hk;
  if (BH * (((int64_t)a.Nk + 127) / 128) > kXaMaxGroups)
    return set_error(TPF_ERR_SHAPE, "%s: too many states", fn);
  a.tiles = (a.R + 127) / 128;
  g.ktiles = (a.Nk + 127) / 128;
  split_axis(BH * a.tiles, a.Nk, 64, &a.splits, &a.chunk, &a.kw);
  split_axis(BH * g.ktiles, a.R, 64, &g.rsplits, &g.rchunk, &g.rkw);
  return TPF_OK;
}

// Workspace in floats: delta, then the partials of the split launches, each
// rounded up to 16 bytes.
struct GradSpace {
  int64_t delta, q, kv, total;
  explicit GradSpace(const XAttnGrad& g) {
    const XAttnArgs& a = g.f;
    const int64_t BH = (int64_t)a.B * a.Hk;
    delta = (BH * a.R + 3) / 4 * 4;
    q = a.splits > 1 ? a.splits * BH * a.R * a.D : 0;
    kv = g.rsplits > 1 ? g.rsplits * BH * a.Nk * a.D : 0;
    total = delta + q + 2 * kv;
  }
};

template <int DP, bool ADD>
static void grad_launch(const XAttnGrad& g, hipStream_t s) {
  const XAttnArgs& a = g.f;
  const int64_t BH = (int64_t)a.B * a.Hk;
  const int64_t n1 = BH * a.splits * a.tiles, n2 = BH * g.rsplits * g.ktiles;
  const dim3 g1((unsigned)((n1 + 7) / 8 * 8)), g2((unsigned)((n2 + 7) / 8 * 8));
  if (a.kw == 2) hipLaunchKernelGGL((xattn_dq_kernel<DP, ADD, 2>), g1, dim3(512), 0, s, g);
  else hipLaunchKernelGGL((xattn_dq_kernel<DP, ADD, 1>), g1, dim3(256), 0, s, g);
  if (g.rkw == 2) hipLaunchKernelGGL((xattn_dkdv_kernel<DP, ADD, 2>), g2, dim3(512), 0, s, g);
  else hipLaunchKernelGGL((xattn_dkdv_kernel<DP, ADD, 1>), g2, dim3(256), 0, s, g);
}

template <bool ADD>
static void grad_pick(const XAttnGrad& g, hipStream_t s) {
  if (g.f.D <= 32) grad_launch<32, ADD>(g, s);
  else if (g.f.D <= 64) grad_launch<64, ADD>(g, s);
  else if (g.f.D <= 96) grad_launch<96, ADD>(g, s);
  else grad_launch<128, ADD>(g, s);
}

}  // namespace tpf

extern "C" int64_t tpf_xattn_backward_workspace_bytes(const tpf_xattn_shape* shape) {
  tpf::XAttnGrad g{};
  const char* fn = "tpf_xattn_backward_workspace_bytes";
  if (tpf::xattn_check(g.f, shape, 1.0, fn) || tpf::grad_plan(g, fn)) return -1;
  return tpf::GradSpace(g).total * 4;
}

static int xattn_backward_entry(const void* q, const void* k, const void* v, const void* mask,
                                const void* out, const void* residual, const void* dout,
                                const float* lse, void* dq, void* dk, void* dv, void* workspace,
                                int64_t workspace_bytes, const tpf_xattn_shape* shape,
                                const int64_t* grad_strides, double scale, void* stream,
                                const char* fn) {
  if (!q || !k || !v || !out || !dout || !lse || !dq || !dk || !dv || !workspace || !grad_strides)
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  tpf::XAttnGrad g{};
  tpf::XAttnArgs& a = g.f;
  if (int rc = tpf::xattn_check(a, shape, scale, fn)) return rc;
  if (shape->dtype != TPF_BF16) return tpf::set_error(TPF_ERR_ARG, "%s: BF16 only", fn);
  if ((a.mask_kind != 0) != (mask != nullptr))
    return tpf::set_error(TPF_ERR_ARG, "%s: mask pointer and mask kind disagree", fn);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)residual | (uintptr_t)dout |
       (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  for (int i = 0; i < 9; ++i)
    if (grad_strides[i] < 0 || grad_strides[i] % 8)
      return tpf::set_error(TPF_ERR_SHAPE, "%s: gradient strides must be multiples of 8 elements", fn);
  if (int rc = tpf::grad_plan(g, fn)) return rc;
  const tpf::GradSpace ws(g);
  if (workspace_bytes < ws.total * 4)
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.q = (const tpf::u16*)q; a.k = (const tpf::u16*)k; a.v = (const tpf::u16*)v; a.mask = mask;
  g.o = (const tpf::u16*)out; g.res = (const tpf::u16*)residual; g.dout = (const tpf::u16*)dout; g.lse = lse;
  g.top = a.mask_kind == tpf::kMaskF32 ? lse + (int64_t)a.B * a.Hk * a.R : nullptr;
  g.dq = (tpf::u16*)dq; g.dk = (tpf::u16*)dk; g.dv = (tpf::u16*)dv;
  for (int i = 0; i < 3; ++i) {
    g.dq_s[i] = grad_strides[i];
    g.dk_s[i] = grad_strides[3 + i];
    g.dv_s[i] = grad_strides[6 + i];
  }
  g.scale = (float)scale;
  float* w = (float*)workspace;
  g.delta = w;
  g.part_q = ws.q ? w + ws.delta : nullptr;
  g.part_k = ws.kv ? w + ws.delta + ws.q : nullptr;
  g.part_v = ws.kv ? w + ws.delta + ws.q + ws.kv : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (a.mask_kind == tpf::kMaskF32) tpf::grad_pick<true>(g, s);
  else tpf::grad_pick<false>(g, s);
  const int64_t BH = (int64_t)a.B * a.Hk;
  auto blocks = [&](bool some, int64_t n) { return some ? (BH * n * (a.D / 4) + 255) / 256 : 0; };
  const int64_t nq = blocks(g.part_q, a.R), nk = blocks(g.part_k, a.Nk);
  if (nq + nk)
    hipLaunchKernelGGL(tpf::xattn_fold_kernel, dim3((unsigned)(nq + 2 * nk)), dim3(256), 0, s, g,
                       (unsigned)nq, (unsigned)(nq + nk));
  return tpf::check_launch(fn);
}

extern "C" int tpf_xattn_backward_bf16(const void* q, const void* k, const void* v, const void* mask,
                                       const void* out, const void* dout, const float* lse, void* dq,
                                       void* dk, void* dv, void* workspace, int64_t workspace_bytes,
                                       const tpf_xattn_shape* shape, const int64_t* grad_strides,
                                       double scale, void* stream) {
  return xattn_backward_entry(q, k, v, mask, out, nullptr, dout, lse, dq, dk, dv, workspace,
                              workspace_bytes, shape, grad_strides, scale, stream,
                              "tpf_xattn_backward_bf16");
}

extern "C" int tpf_xattn_backward_shadow_bf16(const void* q, const void* k, const void* v,
                                              const void* mask, const void* out, const void* residual,
                                              const void* dout, const float* lse, void* dq, void* dk,
                                              void* dv, void* workspace, int64_t workspace_bytes,
                                              const tpf_xattn_shape* shape, const int64_t* grad_strides,
                                              double scale, void* stream) {
  const char* fn = "tpf_xattn_backward_shadow_bf16";
  if (!residual) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  return xattn_backward_entry(q, k, v, mask, out, residual, dout, lse, dq, dk, dv, workspace,
                              workspace_bytes, shape, grad_strides, scale, stream, fn);
}
