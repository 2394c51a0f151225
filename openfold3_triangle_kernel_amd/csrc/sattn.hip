// Causal self-attention: forward, over a batch's own tokens and over a paged cache.
//
//   s_ij = scale q_i . k_j for the states j that row i sees (sattn.hpp), -inf for others
//   p = softmax_j(s),  o_i = sum_j p_ij v_j;  a row that sees none gives 0
//
// in one pass over the states with a running maximum and sum, as cross attention's
// (xattn.hip): a wave owns 32 QB rows and forms S^T = K Q^T, so a lane holds one row's
// scores, and the S^T tile goes back into the matrix cores as it stands for O^T += V^T
// P^T.  Bound by the matrix cores at many rows (4 D operations a visible pair), by the
// states' bytes at few.
#include "sattn.hpp"

namespace tpf {

constexpr int kSaMaxSplits = 256;

__device__ const uint32_t kSaZeros[4] = {0, 0, 0, 0};

// Loader of the [ROWS][DP] tiles of a cache's K and V by NW waves from the states' rows.
template <int DP, int ROWS, int NW>
struct SPageLoader {
  static constexpr int CPR = DP / 8, NI = ROWS * CPR / 64 / NW;
  static __device__ __forceinline__ void issue(const SAttnArgs& a, uint32_t row, int w, u16* K, u16* V) {
    char *dk = reinterpret_cast<char*>(K), *dv = reinterpret_cast<char*>(V);
    uint64_t ks[NI], vs[NI];
    const uint64_t zeros = (uint64_t)(uintptr_t)kSaZeros;
    const uint64_t apart = (uint64_t)(uintptr_t)a.v - (uint64_t)(uintptr_t)a.k;
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int p = 64 * (NI * w + t) + (int)(threadIdx.x & 63), r = p / CPR;
      const int chunk = (p - r * CPR) ^ xa_swz<DP>(r);
      const uint32_t at = __shfl(row, r);
      uint64_t x = (uint64_t)(uintptr_t)a.k + (uint64_t)at * (uint32_t)(2 * a.D) + 16 * chunk;
      const bool live = at != kSaDead && 8 * chunk < a.D;
      asm volatile("" : "+v"(x));  // (formed by every lane: a branch around it would cost more)
      ks[t] = live ? x : zeros;
      vs[t] = live ? x + apart : zeros;
    }
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      g2lds16((const void*)(uintptr_t)ks[t], dk + (NI * w + t) * 1024);
      g2lds16((const void*)(uintptr_t)vs[t], dv + (NI * w + t) * 1024);
    }
  }
};

// Running softmax state of a wave's rows, as cross attention's XRows: the maximum (in raw
// units) is raised only once a row's scores pass it by 8 powers of two; p enters the
// second product rounded, and the outputs are divided by n, the sum of the rounded p, so
// that what the states' values have in common passes exactly; l, the sum of the unrounded
// ones, is the backward's.
template <int DP, int QB, bool F16, bool STATS>
struct SRows {
  static constexpr int DS = DP / 16, DB = DP / 32;
  bf16x8 q[QB][DS];
  f32x16 o[QB][DB];
  float m[QB], l[QB], n[QB];
  int p[QB];  // the lane's rows' positions

  // Row r of the R from the token at q on: pos, the first token's position.
  __device__ __forceinline__ void init(const SAttnArgs& a, const u16* qp, int hk, int r0, int R, int pos) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = min(r0 + 32 * qb + (lane & 31), R - 1);
      const int i = (int)fdiv((uint32_t)r, a.div_g), g = r - i * a.G;
      const u16* x = qp + (int64_t)(hk * a.G + g) * a.q_sh + (int64_t)i * a.q_sn;
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        q[qb][s] = d < a.D ? *reinterpret_cast<const bf16x8*>(x + d) : zero8();
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) o[qb][db] = zero16();
      m[qb] = kSaLow;
      l[qb] = n[qb] = 0.f;
      p[qb] = max(pos + i, -1);
    }
  }

  // Notes what the rows see of the states `bad` from k0 on (SPoison), whose V is not finite.
  __device__ __forceinline__ void note(const SAttnArgs& a, const u16* V, uint64_t bad, uint64_t live, int k0,
                                       uint32_t* poison) const {
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
      SPoison<DP>::template note<F16>(poison + (32 * qb + (threadIdx.x & 31)) * SPoison<DP>::WORDS, V, bad,
                                      sa_sees(a, p[qb], k0, live));
  }

  // KB blocks of 32 states from k0 on; `whole`: every row sees them all.
  template <int KB>
  __device__ __forceinline__ void step(const SAttnArgs& a, const u16* K, const u16* V, uint64_t live,
                                       int k0, bool whole) {
    uint64_t sees[QB];
    if (!whole) {
      bool some = false;
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        sees[qb] = sa_sees(a, p[qb], k0, live);
        some = some || sees[qb] != 0;
      }
      if (__ballot(some) == 0) return;
          }
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
    if (!whole) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint32_t w = (uint32_t)(sees[qb] >> (32 * kb)) >> (4 * ((threadIdx.x >> 5) & 1));
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!((w >> (8 * (r >> 2) + (r & 3))) & 1)) s[qb][kb][r] = -__builtin_inff();
        }
    }
    bf16x8 pr[QB][2 * KB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float t = whole || sees[qb] ? kSaSeen : kSaLow;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = xa_max(t, s[qb][kb][r]);
      t = xa_max32(t);
      const bool raise = (t - m[qb]) * a.c > 8.f;
      if (__ballot(raise)) {  // (each row by itself: what its neighbours hold changes no bit of it)
        const float mn = raise ? t : m[qb], al = fast_exp2((m[qb] - mn) * a.c);
        m[qb] = mn;
        if constexpr (STATS) l[qb] *= al;
        n[qb] *= al;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[qb][db][r] *= al;
      }
      const float off = xa_min(-m[qb] * a.c, -kSaLow);  // (finite beside a score of -inf)
      float sum = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[qb][kb][r] = fast_exp2(fmaf(s[qb][kb][r], a.c, off));
          if constexpr (STATS) sum += s[qb][kb][r];
        }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) pr[qb][2 * kb + t2] = xa_pack8<F16>(s[qb][kb], 8 * t2);
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
          for (int qb = 0; qb < QB; ++qb) o[qb][db] = xa_mfma<F16>(vf, pr[qb][2 * kb + t], o[qb][db]);
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const u32x4 w = __builtin_bit_cast(u32x4, pr[qb][2 * kb + t]);
#pragma unroll
          for (int e = 0; e < 4; ++e) n[qb] = xa_add_pair<F16>(w[e], n[qb]);
        }
      }
    if constexpr (DP > 96) __builtin_amdgcn_s_setprio(0);
  }
};

// 1 / sum of a row with the maximum m; 0 for a row that sees no state, NaN for one
// whose scores are all -inf.
__device__ __forceinline__ float sa_inverse(float n, float m) {
  return n == 0.f ? (m == kSaLow ? 0.f : __builtin_nanf("")) : 1.f / n;
}
// A row's log-sum-exp in powers of two; +inf for a row that sees no state: its p are 0.  (A row
// that has met scores of NaN alone, or beside others, keeps that maximum too: its sum is NaN.)
__device__ __forceinline__ float sa_lse(const SAttnArgs& a, float m, float l) {
  return l == 0.f && m == kSaLow ? __builtin_inff() : fmaf(m, a.c, __log2f(l));
}

// Writes four channels of a row's output at `at`, and what their rounding drops where
// the backward wants it.
template <bool F16>
__device__ __forceinline__ void sa_store4(const SAttnArgs& a, int64_t at, float x0, float x1, float x2,
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

// A tile of rows: of which sequence (or batch entry), and where its rows lie.
struct STile : PagedRows {
  int pos;  // the first token's position
  // Sequence s_ of a paged batch (S: the rows behind the last one, without states).
  __device__ __forceinline__ void sequence(const SAttnArgs& a, int s_) {
    PagedRows::sequence<PagedWave>(a.t, a.G, s_);
    place(a);
  }
  // Row tile `tile` of RT rows of a paged batch, or its row `at`; false where there is none.
  __device__ __forceinline__ bool find(const SAttnArgs& a, int at, int rt) {
    const bool in = tile<PagedWave>(a.t, a.G, rt, at);
    place(a);
    return in;
  }
  __device__ __forceinline__ bool find(const SAttnArgs& a, int64_t at) {
    const bool in = row<PagedWave>(a.t, a.G, at);
    place(a);
    return in;
  }
  __device__ __forceinline__ void place(const SAttnArgs& a) {
    pos = sa_scalar(s < a.t.S ? (int)paged_length(a.t, s) - fresh : -fresh);
  }
  __device__ __forceinline__ int position(const SAttnArgs& a, int r) const {
    return pos + (int)fdiv((uint32_t)(r < R ? r : R - 1), a.div_g);
  }
};

// Where a unit of rows leaves its results: as outputs, or unnormalised as parts `step` apart,
// row by row from `base` on.
struct SResult {
  bool whole;
  int64_t base;
  int step;
};

// An even share of a paged batch's work.  Sequence s costs c_s = (row tiles) x (state tiles of
// its span); the kv heads' sequences' row tiles' state tiles, in this order, are one axis of
// Hk sum(c) tiles, of which workgroup w takes `share`, from w * share on: as many as every
// other, whatever the lengths are (16 tokens of sequences of 2047 to 8190 states: 89 us with the
// join, 99 with a workgroup a part of a sequence and branches around the pages' addresses).  A unit (head, sequence, row tile) whose tiles
// are all a workgroup's own is finished there; others leave a part in slot 2 w (one that began
// before the workgroup's share) or 2 w + 1, and sattn_even_join_kernel finds the slots by the same sums.  Lane
// l holds sequence l (64 at most).  c_s counts a row tile's own span, and an XCD has
// neighbouring workgroups, whose row tiles pass over the same states, also in the join (8 chunks
// of up to 512 tokens, 16 heads on 4 of 96, window 2048, with the join: 67 us against 74).
struct SEven {
  int first, cost, tiles;  // before the sequence, its own, of its span
  int total, share;        // of a head, of a workgroup
  __device__ __forceinline__ void init(const SAttnArgs& a, int rt) {
    const int l = threadIdx.x & 63;
    const bool in = l < a.t.S;
    const int64_t from = in ? paged_start(a.t, l) : 0, next = in ? paged_start(a.t, l + 1) : 0;
    const int fresh = (int)(next > from ? next - from : 0);
    const int len = in ? (int)paged_length(a.t, l) : 0;
    // (Starts that do not ascend may ask for more rows than there are, and are not served.)
    const bool fits = lanes_sum<64>((float)fresh) <= 1.01f * (float)a.t.T;
    tiles = fresh && fits ? SSpan(len - fresh, len - 1, a.window, a.sinks).n : 0;
    // A row tile's own span, of (rt + G - 2) / G + 1 tokens at most, has at most this many.
    tiles = min(tiles, (a.sinks + 63) / 64 + (a.window + (rt - 2) / a.G + 63) / 64 + 1);
    cost = (fresh * a.G + rt - 1) / rt * tiles;
    int sum = cost;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(sum, o);
      if (l >= o) sum += x;
    }
    first = sum - cost;
    total = sa_scalar(__shfl(sum, 63));
    const int even = (int)(((uint32_t)a.Hk * (uint32_t)total + a.even - 1) / (uint32_t)a.even);
    share = sa_scalar(even > kSaLeast ? even : kSaLeast);
  }
};

// The units that workgroup w of an even share takes: f(head, tile, span, first, end, result)
// for the state tiles [first, end) of each.
template <typename F>
__device__ __forceinline__ void sa_even_units(const SAttnArgs& a, int rt, F f) {
  SEven e;
  e.init(a, rt);
  if (e.total == 0) return;
  // (An XCD's workgroups, blockIdx % 8, take neighbouring runs: row tiles over the same states
  // then find them in its L2.)
  const int w = (int)(blockIdx.x & 7) * (a.even >> 3) + (int)(blockIdx.x >> 3);
  int64_t x = (int64_t)w * e.share;
  const int64_t end = min(x + e.share, (int64_t)a.Hk * e.total);
  while (x < end) {
    const int hk = (int)sa_div((uint32_t)x, (uint32_t)e.total), y = (int)x - hk * e.total;
    const int s = __builtin_ctzll(__ballot(e.first <= y && y < e.first + e.cost));
    const int z = y - sa_scalar(__shfl(e.first, s)), n = sa_scalar(__shfl(e.tiles, s));
    const int tile = (int)sa_div((uint32_t)z, (uint32_t)n), t0 = z - tile * n;
    const int count = (int)min((int64_t)n - t0, end - x);
    STile at;
    at.sequence(a, s);
    at.r0 = tile * rt;
    const SSpan span(sa_scalar(at.position(a, at.r0)), sa_scalar(at.position(a, at.r0 + rt - 1)), a.window,
                     a.sinks);  // (n tiles or fewer)
    f(hk, at, span, min(t0, span.n), min(t0 + count, span.n),
      SResult{count == n, (int64_t)(2 * w + (t0 == 0 ? 1 : 0)) * rt, 1});
    x += count;
  }
}

// A unit of 128 QB rows: four waves of 32 QB rows share K and V tiles of 64 states, the tiles
// [first, end) of the span, two stages deep.
template <int DP, int QB, bool F16, bool STATS, bool PAGED>
__device__ __forceinline__ void sattn_tile(const SAttnArgs& a, u16 (*smem)[2][64 * DP], uint32_t* poison,
                                           uint32_t* bad, int b, int hk, const STile& at, const SSpan& span,
                                           int first, int end, const SResult& result) {
  constexpr int KT = 64, RT = 128 * QB;
  typedef SPoison<DP> Poison;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int pmin = sa_scalar(at.position(a, at.r0)), pmax = sa_scalar(at.position(a, at.r0 + RT - 1));
  const int r0 = at.r0 + w * 32 * QB;
  const int p0 = sa_scalar(at.position(a, r0)), p1 = sa_scalar(at.position(a, r0 + 32 * QB - 1));
  STiles<PAGED, KT, 1> t;
  const u16 *kp = a.k, *vp = a.v;
  XTileLoader<DP, KT, 4> lk, lv;
  if constexpr (PAGED) {
    t.pages.init(a, at.s, hk);
  } else {
    t.mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
    kp = sa_scalar(kp + b * a.k_sb + hk * a.k_sh);
    vp = sa_scalar(vp + b * a.v_sb + hk * a.v_sh);
    lk.init(w, a.k_sn, a.D);
    lv.init(w, a.v_sn, a.D);
  }
  t.init(span, first, end, pmax + 1);
  t.below = pmin - a.window + 1;
  SRows<DP, QB, F16, STATS> rows;
  rows.init(a, a.q + (PAGED ? at.token * a.q_sn : b * a.q_sb), hk, r0, at.R, at.pos);

  auto issue = [&](int st) {
    if constexpr (PAGED) {
      SPageLoader<DP, KT, 4>::issue(a, t.pages.row, w, smem[st][0], smem[st][1]);
    } else {
      lk.issue(kp + (int64_t)t.k0 * a.k_sn, t.live, w, smem[st][0]);
      lv.issue(vp + (int64_t)t.k0 * a.v_sn, t.live, w, smem[st][1]);
    }
  };
  // (A wave's rows are its own: no barrier.)
  for (int i = lane; i < 32 * QB * Poison::WORDS; i += 64) poison[w * 32 * QB * Poison::WORDS + i] = 0;
  if (threadIdx.x < 2) bad[threadIdx.x] = 0;
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
    if (!sa_whole(a, pmin, pmax, kc, KT)) {
      // Rows that do not see a state must not meet its V: it is looked over first.
      constexpr int NI = XTileLoader<DP, KT, 4>::NI;
      u16* V = smem[st][1];
      sa_look<DP, NI, F16, false>(V, w, [&](int row) { atomicOr(&bad[row >> 5], 1u << (row & 31)); });
      lds_barrier();
      const uint64_t rows_ = (uint64_t)(uint32_t)sa_scalar((int)bad[1]) << 32 | (uint32_t)sa_scalar((int)bad[0]);
      if (rows_) {
        rows.note(a, V, rows_, lc, kc, poison + w * 32 * QB * Poison::WORDS);
        lds_barrier();
        sa_look<DP, NI, F16, true>(V, w, [](int) {});
        if (threadIdx.x < 2) bad[threadIdx.x] = 0;
        lds_barrier();
      }
    }
    if (r0 < at.R)
      rows.template step<2>(a, smem[st][0], smem[st][1], lc, kc, lc == ~0ull && sa_whole(a, p0, p1, kc, KT));
    st ^= 1;
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int r = r0 + 32 * qb + (lane & 31);
    const float l = xor32_sum(rows.l[qb]), n = xor32_sum(rows.n[qb]);
    if (r >= at.R) continue;
    const uint32_t* hurt = poison + (w * 32 * QB + 32 * qb + (lane & 31)) * Poison::WORDS;
    uint32_t any = 0;
#pragma unroll
    for (int x = 0; x < Poison::WORDS; ++x) any |= hurt[x];
    if (__ballot(any != 0)) {
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          rows.o[qb][db][e] =
              Poison::apply(hurt, 32 * db + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), rows.o[qb][db][e]);
    }
    const int i = (int)fdiv((uint32_t)r, a.div_g), g = r - i * a.G;
    if (result.whole) {
      const float inv = sa_inverse(n, rows.m[qb]);
      const int64_t o = ((at.token + i) * a.H + hk * a.G + g) * a.D;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int d = 32 * db + 8 * g4 + 4 * (lane >> 5);
          const f32x16& x = rows.o[qb][db];
          if (d < a.D)
            sa_store4<F16>(a, o + d, x[4 * g4] * inv, x[4 * g4 + 1] * inv, x[4 * g4 + 2] * inv,
                           x[4 * g4 + 3] * inv);
        }
      if (STATS && lane < 32) a.lse[((int64_t)b * a.Hk + hk) * a.R + r] = sa_lse(a, rows.m[qb], l);
    } else {
      const int64_t at_ = result.base + (int64_t)(r - at.r0) * result.step;
      if (lane < 32) {
        a.part_ml[3 * at_] = rows.m[qb];
        a.part_ml[3 * at_ + 1] = l;
        a.part_ml[3 * at_ + 2] = n;
      }
      float* po = a.part_o + at_ * a.D;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int d = 32 * db + 8 * g4 + 4 * (lane >> 5);
          if (d < a.D) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = rows.o[qb][db][4 * g4 + e];
            *reinterpret_cast<f32x4*>(po + d) = v;
          }
        }
    }
  }
}

// As many workgroups a CU as the registers hold without spilling (2 x 32 heads on 8, 4096 tokens
// of 64 channels: 190 us with four, 203 with the three that the compiler would leave).  128
// channels, with the backward's statistics: 340 us, 810 TFLOP/s of the two products.  Paged, 8
// chunks of up to 512 tokens, 16 heads on 4 of 96, window 2048: 62 us, with a part's first loads
// and its way out and back through the join (12 us) in each of the two or three units a workgroup.
template <int DP, int QB, bool F16, bool STATS, bool PAGED>
__global__ __launch_bounds__(256, PAGED ? 2 : DP == 64 ? 4 : DP == 96 ? 3 : 2)
void sattn_fwd_kernel(SAttnArgs a) {
  constexpr int RT = 128 * QB;
  __shared__ __attribute__((aligned(1024))) u16 smem[2][2][64 * DP];
  __shared__ uint32_t poison[RT * SPoison<DP>::WORDS], bad[2];
  if constexpr (PAGED) {
    if (a.even) {
      sa_even_units(a, RT, [&](int hk, const STile& at, const SSpan& span, int first, int end,
                               const SResult& result) {
        __syncthreads();  // (the unit before is done with the tiles)
        sattn_tile<DP, QB, F16, STATS, PAGED>(a, smem, poison, bad, 0, hk, at, span, first, end, result);
      });
      return;
    }
  }
  int64_t bh;
  int unit;
  if (!sa_unit(a.order, &bh, &unit)) return;
  const int tile = (int)sa_div(unit, a.splits), split = unit - tile * a.splits;
  const int b = PAGED ? 0 : (int)sa_div((uint32_t)bh, a.Hk), hk = (int)bh - b * a.Hk;
  STile at;
  if constexpr (PAGED) {
    if (!at.find(a, tile, RT)) return;
  } else {
    at.s = b;
    at.r0 = (a.tiles - 1 - tile) * RT;  // (later rows see more states)
    at.R = a.R;
    at.pos = 0;
    at.token = (int64_t)b * a.N;
  }
  const SSpan span(sa_scalar(at.position(a, at.r0)), sa_scalar(at.position(a, at.r0 + RT - 1)), a.window,
                   a.sinks);
  const SParts parts(span.n, a.splits, kSaLeast);
  if (a.splits > 1 && split >= parts.live) return;
  sattn_tile<DP, QB, F16, STATS, PAGED>(
      a, smem, poison, bad, b, hk, at, span, split * parts.per, min(span.n, (split + 1) * parts.per),
      SResult{a.splits == 1, (hk * a.rows + at.token * a.G + at.r0) * a.splits + split, a.splits});
}

// Few rows of a sequence (32 a workgroup; one decoded token above all): the states' bytes
// are the bound.  Every wave streams tiles of 32 states of its own, two stages deep without
// a barrier, and the four waves' results meet in LDS at the end.  16 tokens of 32 heads on 8 of
// 128 over 403 MB of states: 81-85 us, 4.9 TB/s, the rate of a copy (the loads alone: 75-80).
template <int DP, bool F16>
__device__ __forceinline__ void sattn_few(const SAttnArgs& a, u16 (*smem)[2][2][32 * DP], uint32_t* poison,
                                          int hk, const STile& at, const SSpan& span, int first, int end,
                                          const SResult& result) {
  constexpr int KT = 32, RT = 32, NI = KT * DP / 512;
  constexpr int OP = DP + 4;  // pitch of the joined rows (f32)
  typedef SPoison<DP> Poison;
  static_assert(4 * sizeof(smem[0]) >= 4 * 32 * (OP + 2) * 4, "the join fits");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int p0 = sa_scalar(at.position(a, at.r0)), p1 = sa_scalar(at.position(a, at.r0 + RT - 1));
  STiles<true, KT, 4> t;
  t.pages.init(a, at.s, hk);
  t.init(span, 2 * first + w, 2 * end, p1 + 1);
  t.below = p0 - a.window + 1;
  SRows<DP, 1, F16, false> rows;
  rows.init(a, a.q + at.token * a.q_sn, hk, at.r0, at.R, at.pos);

  auto issue = [&](int st) {
    SPageLoader<DP, KT, 1>::issue(a, t.pages.row, 0, smem[w][st][0], smem[w][st][1]);
  };
  for (int i = threadIdx.x; i < RT * Poison::WORDS; i += 256) poison[i] = 0;
  lds_barrier();
  bool more = t.advance(a, span);
  if (more) issue(0);
  int st = 0;
  while (more) {
    const int kc = t.k0;
    const uint64_t lc = t.live;
    more = t.advance(a, span);
    if (more) {
      issue(st ^ 1);
      wait_vmcnt<2 * NI>();  // this tile's loads are older than the next one's
    } else {
      wait_vmcnt<0>();
    }
    const bool whole = lc == 0xffffffffull && sa_whole(a, p0, p1, kc, KT);
    if (!whole) {  // (as in the tile kernel; the tile is this wave's own)
      u16* V = smem[w][st][1];
      const uint32_t bad = sa_bad_rows<DP, F16>(V, 0);
      if (bad) {
        rows.note(a, V, bad, lc, kc, poison);
        sa_look<DP, NI, F16, true>(V, 0, [](int) {});
      }
    }
    rows.template step<1>(a, smem[w][st][0], smem[w][st][1], lc, kc, whole);
    st ^= 1;
  }

  float* O = reinterpret_cast<float*>(&smem[0][0][0][0]);
  float* MN = O + 4 * 32 * OP;
  __syncthreads();
  const float nw = xor32_sum(rows.n[0]);
  float* ow = O + (w * 32 + (lane & 31)) * OP;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = rows.o[0][db][4 * g4 + e];
      *reinterpret_cast<f32x4*>(ow + 32 * db + 8 * g4 + 4 * (lane >> 5)) = v;
    }
  if (lane < 32) {
    MN[2 * (w * 32 + lane)] = rows.m[0];
    MN[2 * (w * 32 + lane) + 1] = nw;
  }
  __syncthreads();
  const int rl = threadIdx.x >> 3, r = at.r0 + rl;
  if (r >= at.R) return;
  float m = kSaLow, n = 0.f, f[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) m = xa_max(m, MN[2 * (x * 32 + rl)]);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    f[x] = fast_exp2((MN[2 * (x * 32 + rl)] - m) * a.c);
    n += f[x] * MN[2 * (x * 32 + rl) + 1];
  }
  const int64_t pr = result.base + (int64_t)rl * result.step;
  const float inv = sa_inverse(n, m);
  const int i = (int)fdiv((uint32_t)r, a.div_g), g = r - i * a.G;
  const int64_t out = ((at.token + i) * a.H + hk * a.G + g) * a.D;
  for (int d = 4 * (threadIdx.x & 7); d < a.D; d += 32) {
    f32x4 o = (f32x4)0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(O + (x * 32 + rl) * OP + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f[x] * v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = Poison::apply(poison + rl * Poison::WORDS, d + e, o[e]);
    if (result.whole) sa_store4<F16>(a, out + d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    else *reinterpret_cast<f32x4*>(a.part_o + pr * a.D + d) = o;
  }
  if (!result.whole && (threadIdx.x & 7) == 0) {
    a.part_ml[3 * pr] = m;
    a.part_ml[3 * pr + 1] = n;
    a.part_ml[3 * pr + 2] = n;
  }
}

template <int DP, bool F16>
__global__ __launch_bounds__(256, 1) void sattn_few_kernel(SAttnArgs a) {
  constexpr int RT = 32;
  __shared__ __attribute__((aligned(1024))) u16 smem[4][2][2][32 * DP];
  __shared__ uint32_t poison[RT * SPoison<DP>::WORDS];
  if (a.even) {
    sa_even_units(a, RT, [&](int hk, const STile& at, const SSpan& span, int first, int end,
                             const SResult& result) {
      __syncthreads();  // (the unit before is done with the tiles)
      sattn_few<DP, F16>(a, smem, poison, hk, at, span, first, end, result);
    });
    return;
  }
  int64_t head;
  int unit;
  if (!sa_unit(a.order, &head, &unit)) return;
  const int hk = (int)head, tile = (int)sa_div(unit, a.splits), split = unit - tile * a.splits;
  STile at;
  if (!at.find(a, tile, RT)) return;
  const SSpan span(sa_scalar(at.position(a, at.r0)), sa_scalar(at.position(a, at.r0 + RT - 1)), a.window,
                   a.sinks);
  const SParts parts(span.n, a.splits, kSaLeast);
  if (a.splits > 1 && split >= parts.live) return;
  sattn_few<DP, F16>(a, smem, poison, hk, at, span, split * parts.per, min(span.n, (split + 1) * parts.per),
                     SResult{a.splits == 1, (hk * a.rows + at.token * a.G + at.r0) * a.splits + split, a.splits});
}

// Joins the parts of a row's states, a wave a row: o = sum_s 2^(c (m_s - m)) o_s / sum_s
// 2^(c (m_s - m)) n_s; the lanes' halves take the parts in turn.
template <bool F16, bool PAGED>
__global__ __launch_bounds__(256) void sattn_join_kernel(SAttnArgs a, int rt) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= a.Hk * a.rows) return;
  const int hk = (int)(item / a.rows);
  const int64_t row = item - hk * a.rows;
  STile at;
  int r;
  if constexpr (PAGED) {
    if (!at.find(a, row)) return;
    r = at.r0;
  } else {
    at.s = (int)(row / a.R);
    at.token = (int64_t)at.s * a.N;
    at.R = a.R;
    at.pos = 0;
    r = (int)(row - at.token * a.G);
  }
  const int r0 = r / rt * rt;
  const SSpan span(at.position(a, r0), at.position(a, r0 + rt - 1), a.window, a.sinks);
  const int live = SParts(span.n, a.splits, kSaLeast).live;
  const int64_t first = item * a.splits;

  float m = kSaLow;
  for (int s = lane; s < live; s += 64) m = xa_max(m, a.part_ml[3 * (first + s)]);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = xa_max(m, __shfl_xor(m, o));
  const int d = 4 * (lane & 31);
  float l = 0.f, n = 0.f;
  f32x4 o = (f32x4)0.f;
  for (int s0 = 0; s0 < live; s0 += 64) {
    const int s = s0 + lane;
    const float f = s < live ? fast_exp2((a.part_ml[3 * (first + s)] - m) * a.c) : 0.f;
    if (s < live) {
      l = fmaf(f, a.part_ml[3 * (first + s) + 1], l);
      n = fmaf(f, a.part_ml[3 * (first + s) + 2], n);
    }
    const int count = min(64, live - s0);
#pragma unroll 4
    for (int x = 0; x < count; x += 2) {
      const float wt = __shfl(f, x + half);  // (0 past the last)
      f32x4 v = (f32x4)0.f;
      if (d < a.D && x + half < count)
        v = *reinterpret_cast<const f32x4*>(a.part_o + (first + s0 + x + half) * a.D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, v[e], o[e]);
    }
  }
  l = lanes_sum<64>(l);
  n = lanes_sum<64>(n);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = xor32_sum(o[e]);
  const float inv = sa_inverse(n, m);
  const int i = (int)fdiv((uint32_t)r, a.div_g), g = r - i * a.G;
  if (half == 0 && d < a.D)
    sa_store4<F16>(a, ((at.token + i) * a.H + hk * a.G + g) * a.D + d, o[0] * inv, o[1] * inv, o[2] * inv,
                   o[3] * inv);
  if (a.lse && lane == 0) a.lse[((int64_t)at.s * a.Hk + hk) * a.R + r] = sa_lse(a, m, l);
}

// The same for an even share.  Of every unit that workgroups share, the join's workgroup that
// has the number of the second of them joins the rows, 32 rows each; the workgroups
// behind them write the
// zeros of tokens that see nothing (of no sequence, or of one without states), a wave a token.
template <bool F16>
__global__ __launch_bounds__(256) void sattn_even_join_kernel(SAttnArgs a, int rt) {
  // (Each XCD joins what its own workgroups left: a.even is a multiple of eight.)
  const int lane = threadIdx.x & 63, each = rt / 32, joins = a.even * each, block = (int)blockIdx.x;
  const int item = block < joins ? (block & 7) * (joins >> 3) + (block >> 3) : block;
  const int w = (int)sa_div((uint32_t)item, (uint32_t)each);
  SEven e;
  e.init(a, rt);
  if (w >= a.even) {
    const int64_t token = (int64_t)(block - joins) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (token >= a.t.T) return;
    const int s = __builtin_amdgcn_readfirstlane(
        paged_search<PagedWave>(a.t.S, [&](int x) { return paged_start(a.t, x) <= token; }));
    if (s < a.t.S && __shfl(e.tiles, s) != 0) return;
    uint2* out = reinterpret_cast<uint2*>(a.out + token * a.H * a.D);
    for (int i = lane; i < a.H * a.D / 4; i += 64) out[i] = uint2{0, 0};
    return;
  }
  const int64_t x = (int64_t)w * e.share;
  if (w == 0 || x >= (int64_t)a.Hk * e.total) return;
  const int hk = (int)sa_div((uint32_t)x, (uint32_t)e.total), y = (int)x - hk * e.total;
  const int s = __builtin_ctzll(__ballot(e.first <= y && y < e.first + e.cost));
  const int z = y - sa_scalar(__shfl(e.first, s)), n = sa_scalar(__shfl(e.tiles, s));
  const int tile = (int)sa_div((uint32_t)z, (uint32_t)n), before = z - tile * n;
  // Tiles of the unit before this workgroup's share: none, or more than the workgroup before has.
  if (before == 0 || before > e.share) return;
  const int parts = 2 + (n - before - 1) / e.share;
  STile at;
  at.sequence(a, s);
  const int rows = min(rt, at.R - tile * rt), d = 4 * (threadIdx.x & 31);
  if (d >= a.D) return;
  // Four rows a thread, whose loads go out together.
  const int first = 32 * (item - w * each) + (int)(threadIdx.x >> 5);
  int r[4];
  float m[4], sum[4];
  f32x4 o[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    r[u] = min(first + 8 * u, rows - 1);
    m[u] = kSaLow;
    sum[u] = 0.f;
    o[u] = (f32x4)0.f;
  }
#pragma unroll 2
  for (int i = 0; i < parts; ++i) {
    // Slot 2 (w - 1) + 1, then 2 w, 2 w + 2, ...
    const int64_t slot = (int64_t)(i ? 2 * (w + i - 1) : 2 * w - 1) * rt;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float mi = a.part_ml[3 * (slot + r[u])], ni = a.part_ml[3 * (slot + r[u]) + 2];
      const f32x4 v = *reinterpret_cast<const f32x4*>(a.part_o + (slot + r[u]) * a.D + d);
      const float to = xa_max(m[u], mi), f = fast_exp2((m[u] - to) * a.c), g = fast_exp2((mi - to) * a.c);
      m[u] = to;
      sum[u] = fmaf(g, ni, f * sum[u]);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[u][c] = fmaf(g, v[c], f * o[u][c]);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (first + 8 * u >= rows) break;
    const float inv = sa_inverse(sum[u], m[u]);
    const int all = tile * rt + r[u], i = (int)fdiv((uint32_t)all, a.div_g), g = all - i * a.G;
    sa_store4<F16>(a, ((at.token + i) * a.H + hk * a.G + g) * a.D + d, o[u][0] * inv, o[u][1] * inv,
                   o[u][2] * inv, o[u][3] * inv);
  }
}

// Sizes that both forms share; 0 or an error code.
static int sattn_check(SAttnArgs& a, int64_t H, int64_t Hk, int64_t D, int64_t window, int64_t sinks,
                       double scale, const char* fn) {
  if (H < 1 || Hk < 1 || H % Hk || H > (1 << 20) || D < 8 || D > 128 || D % 8)
    return set_error(TPF_ERR_SHAPE, "%s: bad shape H=%lld Hk=%lld D=%lld", fn, (long long)H, (long long)Hk,
                     (long long)D);
  if (window < 0 || sinks < 0) return set_error(TPF_ERR_ARG, "%s: window and sinks must not be negative", fn);
  if (!(scale > 1e-30) || !(scale < 1e30))
    return set_error(TPF_ERR_ARG, "%s: the scale must be between 1e-30 and 1e30", fn);
  const int64_t most = (int64_t)1 << 30;  // above every position
  a.window = (int)(window == 0 || window > most ? most : window);
  a.sinks = a.window == most ? 0 : (int)(sinks > most ? most : sinks);
  a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.D = (int)D;
  a.div_g = make_fastdiv((uint32_t)a.G);
  a.c = (float)(scale * 1.4426950408889634);
  return TPF_OK;
}

int window_check(SAttnArgs& a, const tpf_window_shape* s, double scale, const char* fn) {
  if (!s) return set_error(TPF_ERR_ARG, "%s: null shape", fn);
  if (int rc = sattn_check(a, s->H, s->Hk, s->D, s->window, s->sinks, scale, fn)) return rc;
  const int64_t lim = (int64_t)1 << 30;
  if (s->B < 1 || s->N < 1 || s->B > lim || s->N > lim || a.G * s->N > lim ||
      (double)s->B * s->Hk * ((double)(a.G * s->N) / 64 + 1) * 64 > 2e9 ||
      s->B * s->Hk * ((a.G * s->N + 127) / 128 + 8) > kMaxGroups)
    return set_error(TPF_ERR_SHAPE, "%s: too many rows (B=%lld N=%lld)", fn, (long long)s->B, (long long)s->N);
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
  if (s->mask_stride < 0) return set_error(TPF_ERR_ARG, "%s: bad mask", fn);
  a.q_sb = s->q_stride[0]; a.q_sh = s->q_stride[1]; a.q_sn = s->q_stride[2];
  a.k_sb = s->k_stride[0]; a.k_sh = s->k_stride[1]; a.k_sn = s->k_stride[2];
  a.v_sb = s->v_stride[0]; a.v_sh = s->v_stride[1]; a.v_sn = s->v_stride[2];
  a.mask_sb = s->mask_stride;
  a.B = (int)s->B; a.N = (int)s->N; a.R = (int)(a.G * s->N);
  if (a.window >= a.N || a.sinks >= a.N) {  // every token sees all up to itself
    a.window = 1 << 30;
    a.sinks = 0;
  }
  a.rows = (int64_t)a.B * a.R;
  return TPF_OK;
}

// Workgroups of an even share's join: a unit's rows by 32, and a wave a token.
static int64_t sattn_even_joins(const SAttnArgs& a, int rt) { return (int64_t)a.even * (rt / 32) + (a.t.T + 3) / 4; }

// Rows of the parts in memory.
static int64_t sattn_part_rows(const SAttnArgs& a, int rt) {
  return a.even ? (int64_t)2 * a.even * rt : a.splits > 1 ? a.Hk * a.rows * a.splits : 0;
}

// Parts of the states so that `units` workgroups become `target`, of 256 states at least.
static int sattn_splits(int64_t units, int64_t target, int64_t states) {
  int64_t s = target / units;
  if (s > states / 256) s = states / 256;
  if (s > kSaMaxSplits) s = kSaMaxSplits;
  return (int)(s < 1 ? 1 : s);
}

// 128 rows a workgroup, 256 up to 32 channels where those fill the chip twice: each K and V
// fragment then feeds two products (16 heads on 4, 16384 tokens, window 1024: 76 us against 81
// with 32 channels).  With 64 channels 128 rows are faster, whose registers let more waves run on
// a SIMD (2 x 32 heads on 8, 4096 tokens: 203 us with three against 213 with 256 rows).
static int window_plan(SAttnArgs& a) {
  const int64_t BH = (int64_t)a.B * a.Hk;
  const int qb = a.D <= 32 && BH * ((a.R + 255) / 256) >= 512 ? 2 : 1;
  a.tiles = (a.R + 128 * qb - 1) / (128 * qb);
  a.splits = sattn_splits(BH * a.tiles, 256, a.N);
  a.order = sa_order(BH, (int64_t)a.tiles * a.splits);
  return qb;
}

template <int DP, bool F16, bool STATS>
static void window_launch(const SAttnArgs& a, int qb, hipStream_t s) {
  const dim3 grid((unsigned)a.order.groups);
  if constexpr (DP <= 32) {
    if (qb == 2) {
      hipLaunchKernelGGL((sattn_fwd_kernel<DP, 2, F16, STATS, false>), grid, dim3(256), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((sattn_fwd_kernel<DP, 1, F16, STATS, false>), grid, dim3(256), 0, s, a);
}

template <bool F16, bool STATS>
static void window_pick(const SAttnArgs& a, int qb, hipStream_t s) {
  if (a.D <= 32) window_launch<32, F16, STATS>(a, qb, s);
  else if (a.D <= 64) window_launch<64, F16, STATS>(a, qb, s);
  else if (a.D <= 96) window_launch<96, F16, STATS>(a, qb, s);
  else window_launch<128, F16, STATS>(a, qb, s);
}

template <bool F16, bool PAGED>
static void sattn_join(const SAttnArgs& a, int rt, hipStream_t s) {
  if (a.even)
    hipLaunchKernelGGL((sattn_even_join_kernel<F16>), dim3((unsigned)sattn_even_joins(a, rt)), dim3(256), 0, s, a,
                       rt);
  if (a.splits > 1)
    hipLaunchKernelGGL((sattn_join_kernel<F16, PAGED>), dim3((unsigned)((a.Hk * a.rows + 3) / 4)), dim3(256), 0,
                       s, a, rt);
}

static int paged_attn_check(SAttnArgs& a, const tpf_paged_shape* s, const tpf_paged_batch* batch, double scale,
                            const char* fn) {
  if (!s) return set_error(TPF_ERR_ARG, "%s: null shape", fn);
  if (int rc = paged_check(a.t, batch, fn)) return rc;
  if (int rc = sattn_check(a, s->H, s->Hk, s->D, s->window, s->sinks, scale, fn)) return rc;
  if (s->dtype != TPF_BF16 && s->dtype != TPF_F16)
    return set_error(TPF_ERR_ARG, "%s: dtype must be TPF_BF16 or TPF_F16", fn);
  for (int i = 0; i < 2; ++i)
    if (s->q_stride[i] < 0 || s->q_stride[i] % 8)
      return set_error(TPF_ERR_SHAPE, "%s: strides must be multiples of 8 elements", fn);
  if ((double)batch->pages * s->Hk * batch->page > (double)((int64_t)1 << 30))
    return set_error(TPF_ERR_SHAPE, "%s: a cache holds 2^30 states of all kv heads at most", fn);
  a.q_sn = s->q_stride[0]; a.q_sh = s->q_stride[1];
  a.B = a.t.S;
  a.rows = a.t.T * a.G;
  if (a.rows > ((int64_t)1 << 30) || ((double)a.rows / 32 + a.t.S + 9) * a.Hk > (double)kMaxGroups / 2 ||
      (double)a.rows * a.Hk / 4 + 1 > (double)kMaxGroups)
    return set_error(TPF_ERR_SHAPE, "%s: too many rows", fn);
  return TPF_OK;
}

// Up to 32 rows a sequence on the mean run on the streaming kernel.  Up to 64 sequences share
// their work evenly over the workgroups that run at once, if a sequence can have 1024 states;
// otherwise tiles are counted for the most that the tokens can be and the parts for those
// that are likely.  (One token of each of 64 sequences of 512 to 8191 states, 32 heads on 8 of
// 128: 250 us, 5.1 TB/s; of 65: 280, 4.0 TB/s.  77 states in a table for 8192: 13 us, in a short
// one 7: the host does not read the lengths.)
static int paged_plan(SAttnArgs& a) {
  const int rt = a.rows <= 32 * (int64_t)a.t.S ? 32 : 128;
  const int64_t states = (int64_t)a.t.width * a.t.page;
  a.tiles = (int)(a.rows / rt) + a.t.S + 1;
  a.splits = 1;
  a.even = 0;
  if (a.t.S <= 64 && states >= 1024 &&
      ((double)a.rows / rt + a.t.S) * ((double)states / 64 + 1) * a.Hk < (double)((int64_t)1 << 30)) {
    // Workgroups that a CU runs at once: the streaming kernel's by their LDS, the tile kernel's by
    // their registers.
    a.even = 256 * (a.D > 64 ? (rt == 128 ? 2 : 1) : a.D > 32 ? (rt == 128 ? 3 : 2) : 4);
    if (sattn_even_joins(a, rt) <= kMaxGroups) return rt;
    a.even = 0;
  }
  int64_t units = a.rows / rt > a.t.S ? a.rows / rt : a.t.S;
  units *= a.Hk;
  a.splits = sattn_splits(units < 1 ? 1 : units, 512, states);
  while (a.splits > 1 && (double)a.tiles * a.Hk * a.splits > (double)kMaxGroups / 2) a.splits /= 2;
  a.order = sa_order(a.Hk, (int64_t)a.tiles * a.splits);
  return rt;
}

template <int DP, bool F16>
static void paged_launch(const SAttnArgs& a, int rt, hipStream_t s) {
  const dim3 grid((unsigned)(a.even ? a.even : a.order.groups));
  if (rt == 32) hipLaunchKernelGGL((sattn_few_kernel<DP, F16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((sattn_fwd_kernel<DP, 1, F16, false, true>), grid, dim3(256), 0, s, a);
}

template <bool F16>
static void paged_pick(const SAttnArgs& a, int rt, hipStream_t s) {
  if (a.D <= 32) paged_launch<32, F16>(a, rt, s);
  else if (a.D <= 64) paged_launch<64, F16>(a, rt, s);
  else if (a.D <= 96) paged_launch<96, F16>(a, rt, s);
  else paged_launch<128, F16>(a, rt, s);
  sattn_join<F16, true>(a, rt, s);
}

}  // namespace tpf

extern "C" int64_t tpf_window_forward_workspace_bytes(const tpf_window_shape* shape) {
  tpf::SAttnArgs a{};
  if (tpf::window_check(a, shape, 1.0, "tpf_window_forward_workspace_bytes")) return -1;
  const int qb = tpf::window_plan(a);
  return tpf::sattn_part_rows(a, 128 * qb) * (a.D + 3) * 4;
}

extern "C" int tpf_window_forward(const void* q, const void* k, const void* v, const void* mask, void* out,
                                  float* lse, void* residual, void* workspace, int64_t workspace_bytes,
                                  const tpf_window_shape* shape, double scale, void* stream) {
  const char* fn = "tpf_window_forward";
  if (!q || !k || !v || !out) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  tpf::SAttnArgs a{};
  if (int rc = tpf::window_check(a, shape, scale, fn)) return rc;
  if ((lse || residual) && shape->dtype != TPF_BF16)
    return tpf::set_error(TPF_ERR_ARG, "%s: a backward needs BF16", fn);
  if (residual && !lse) return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)residual |
       (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  const int qb = tpf::window_plan(a);
  const int64_t parts = tpf::sattn_part_rows(a, 128 * qb);
  if (parts && (!workspace || workspace_bytes < parts * (a.D + 3) * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.q = (const tpf::u16*)q; a.k = (const tpf::u16*)k; a.v = (const tpf::u16*)v;
  a.mask = (const uint8_t*)mask;
  a.out = (tpf::u16*)out; a.res = (tpf::u16*)residual; a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_ml = parts ? a.part_o + parts * a.D : nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (shape->dtype == TPF_F16) {
    tpf::window_pick<true, false>(a, qb, s);
    tpf::sattn_join<true, false>(a, 128 * qb, s);
  } else {
    if (lse) tpf::window_pick<false, true>(a, qb, s);
    else tpf::window_pick<false, false>(a, qb, s);
    tpf::sattn_join<false, false>(a, 128 * qb, s);
  }
  return tpf::check_launch(fn);
}

extern "C" int64_t tpf_paged_attention_workspace_bytes(const tpf_paged_shape* shape,
                                                       const tpf_paged_batch* batch) {
  tpf::SAttnArgs a{};
  if (tpf::paged_attn_check(a, shape, batch, 1.0, "tpf_paged_attention_workspace_bytes")) return -1;
  const int rt = tpf::paged_plan(a);
  return tpf::sattn_part_rows(a, rt) * (a.D + 3) * 4;
}

extern "C" int tpf_paged_attention(const void* q, const void* k_cache, const void* v_cache, void* out,
                                   void* workspace, int64_t workspace_bytes, const tpf_paged_shape* shape,
                                   const tpf_paged_batch* batch, double scale, void* stream) {
  const char* fn = "tpf_paged_attention";
  tpf::SAttnArgs a{};
  if (int rc = tpf::paged_attn_check(a, shape, batch, scale, fn)) return rc;
  if (!q || !out || (a.t.pages && (!k_cache || !v_cache)))
    return tpf::set_error(TPF_ERR_ARG, "%s: null pointer", fn);
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) % 16)
    return tpf::set_error(TPF_ERR_ARG, "%s: tensors must start on 16 bytes", fn);
  const int rt = tpf::paged_plan(a);
  const int64_t parts = tpf::sattn_part_rows(a, rt);
  if (parts && (!workspace || workspace_bytes < parts * (a.D + 3) * 4))
    return tpf::set_error(TPF_ERR_ARG, "%s: workspace too small", fn);
  a.q = (const tpf::u16*)q; a.k = (const tpf::u16*)k_cache; a.v = (const tpf::u16*)v_cache;
  a.out = (tpf::u16*)out;
  a.part_o = (float*)workspace;
  a.part_ml = parts ? a.part_o + parts * a.D : nullptr;
  if (shape->dtype == TPF_F16) tpf::paged_pick<true>(a, rt, (hipStream_t)stream);
  else tpf::paged_pick<false>(a, rt, (hipStream_t)stream);
  return tpf::check_launch(fn);
}
