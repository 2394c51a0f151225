// Shared pieces of causal self-attention (sattn.hip, sattn_bwd.hip): over a batch's own
// tokens, or the new tokens of sequences over a paged cache.
//
// Rows and states.  The queries of the G query heads on a kv head are one row axis, token
// by token: row r is token r / G under query head hk * G + r % G.  A tile of rows then
// spans few tokens, and its states end close behind the last of them.  The token that is
// state p sees the states j <= p with p - j < window or j < sinks, of those that live (the
// key mask; a page that the cache has).  A tile of rows passes over the 64-state tiles
// that any of its tokens may see: those of the sinks, then those from the first token's
// window to the last token.
//
// Operand tiles in LDS are cross attention's (xattn.hpp).  A row's scores of states that it
// does not see are -inf by bit, whatever they are.  Such a state's V is another matter: a
// product takes 0 p times it, which infinities and NaN survive.  Blocks that some row sees
// in part are looked over for them first, and they are kept from those rows.
#pragma once

#include "gemm_core.hpp"  // xcd_order
#include "paged.hpp"
#include "tpf_status.hpp"
#include "xattn.hpp"

namespace tpf {

// The maximum of a row before its first visible state, and the least one after it.
constexpr float kSaLow = -3.402823466e38f, kSaSeen = -3.3e38f;

// Order of `units` units of work of every head over the XCDs (sa_unit): 2^shift sub-sequences of
// a head's units; those of an XCD, and how many of them at a time; units of a sub-sequence.
struct SOrder {
  int units;
  uint32_t shift, subs, together, each;
  int64_t groups;  // workgroups in all
};

struct SAttnArgs {
  const u16 *q, *k, *v;
  int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;  // element strides
  const uint8_t* mask;  // [B, N], null without
  int64_t mask_sb;
  u16* out;    // [tokens, H, D]
  u16* res;    // what its rounding drops, laid out the same; null when not wanted
  float* lse;  // [B, Hk, R] log-sum-exp of the rows; null when no backward follows
  int B, H, Hk, G, N, D, R;  // R = G * N rows of a kv head
  FastDiv div_g;
  float c;             // scale * log2(e)
  int window, sinks;   // window above every position where there is none, then no sinks
  int splits, tiles;   // most parts of a tile's states; row tiles of a batch entry
  int even;            // workgroups that share a paged batch's state tiles evenly (SEven), or 0
  SOrder order;        // of the forward's or dQ's units
  int64_t rows;        // rows of a kv head in all
  float* part_o;       // [Hk, rows, splits, D] (or SEven's) unnormalised outputs of the parts
  float* part_ml;      // the same by 3: their maxima and the two sums (SRows)
  PagedTables t;
};

// ones(n): the n + 1 lowest bits, none below 0.
__device__ __forceinline__ uint64_t sa_ones(int n) {
  return n < 0 ? 0 : n >= 63 ? ~0ull : (2ull << n) - 1;
}
__device__ __forceinline__ uint32_t sa_ones32(int n) {
  return n < 0 ? 0 : n >= 31 ? ~0u : (2u << n) - 1;
}

// The states that rows at positions pmin .. pmax may see, as tiles of 64: `n` in all, the
// first `heads` of them the sinks' (from state 0), the others from state `low` on.
struct SSpan {
  int low, heads, n;
  __host__ __device__ __forceinline__ SSpan(int pmin, int pmax, int window, int sinks) {
    const int first = pmin - window + 1;  // (both below 2^30)
    low = first > 0 ? first / 64 * 64 : 0;
    heads = (sinks + 63) / 64;
    if (heads > low / 64) heads = low / 64;
    n = heads + (pmax >= low ? (pmax - low) / 64 + 1 : 0);
    if (pmax < 0) n = 0;
  }
  __host__ __device__ __forceinline__ int state(int t) const { return t < heads ? 64 * t : low + 64 * (t - heads); }
};

// Parts of a tile's n state tiles: `per` each, the last one shorter; `live` of them.
struct SParts {
  int per, live;
  __host__ __device__ __forceinline__ SParts(int n, int splits, int least) {
    per = (n + splits - 1) / splits;
    if (per < least) per = least;
    live = (n + per - 1) / per;
  }
};
constexpr int kSaLeast = 4;  // state tiles of a part, at least

// The bits of the 64 states from k0 on that the row at position p sees, of the `live`.
__device__ __forceinline__ uint64_t sa_sees(const SAttnArgs& a, int p, int k0, uint64_t live) {
  const int rel = p - k0;
  return live & sa_ones(rel) & (~sa_ones(rel - a.window) | sa_ones(a.sinks - 1 - k0));
}

// Whether rows at positions pmin .. pmax see all of the `count` states from k0 on.
__device__ __forceinline__ bool sa_whole(const SAttnArgs& a, int pmin, int pmax, int k0, int count) {
  return k0 + count - 1 <= pmin && (k0 > pmax - a.window || k0 + count <= a.sinks);
}

// A quotient of uniform values, on the scalar side (the compiler forms it in vector registers
// and leaves all that follows from it there).
__device__ __forceinline__ uint32_t sa_div(uint32_t n, uint32_t d) {
  return __builtin_amdgcn_readfirstlane(n / d);
}

__device__ __forceinline__ int sa_scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename T>
__device__ __forceinline__ const T* sa_scalar(const T* p) {
  const uint64_t x = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
  return (const T*)(uintptr_t)((uint64_t)hi << 32 | lo);
}

// This workgroup's kv head of a batch entry, and its unit of work there, of those that the
// host counted (SOrder); false past the last one.  Units are numbered from the longest on
// and start in that order; an XCD (workgroup L runs on XCD L % 8) has whole heads, whose
// K and V its L2 then holds, one after the other or two at a time, or, where their number
// is none of eight's, every second, fourth or eighth unit of one.
__device__ __forceinline__ bool sa_unit(const SOrder& o, int64_t* head, int* unit) {
  const uint32_t x = blockIdx.x & 7, j = blockIdx.x >> 3;
  const uint32_t run = o.together * o.each, group = sa_div(j, run), rest = j - group * run;
  const uint32_t at = o.together == 2 ? rest / 2 : rest;
  const uint32_t sub = x * o.subs + group * o.together + (rest - at * o.together);
  const uint32_t bh = sub >> o.shift;
  *head = bh;
  *unit = (int)((at << o.shift) + (sub - (bh << o.shift)));
  return *unit < o.units;
}

constexpr uint32_t kSaDead = 0xffffffffu;

// Where states lie in the pages of sequence s under kv head hk: lane l holds the page of
// table entry `first + l`, read once for 64 entries.
template <int ROWS>
struct SPages {
  const int32_t* table;
  int first, page, hk;
  uint32_t row;  // of the lane's state: (page Hk + hk) P + place, kSaDead where none lives
  __device__ __forceinline__ void init(const SAttnArgs& a, int s, int hk_) {
    table = a.t.tables + s * a.t.table_ld;
    first = -1 - 64;
    page = -1;
    hk = hk_;
  }
  // The states k0 + lane % ROWS below `end`: their rows, and which live.
  __device__ __forceinline__ uint64_t at(const SAttnArgs& a, int k0, int end) {
    const int lane = threadIdx.x & 63;
    const int e0 = (int)fdiv((uint32_t)k0, a.t.div_page);
    const int e1 = (int)fdiv((uint32_t)min(k0 + ROWS - 1, end - 1), a.t.div_page);
    if (e0 < first || e1 > first + 63) {
      first = e0;
      page = first + lane < a.t.width ? table[first + lane] : -1;
      // (Waited for here: at its use the compiler would wait for every load under way.)
      asm volatile("" : "+v"(page));
    }
    const int j = min(k0 + lane % ROWS, end - 1);
    const int e = (int)fdiv((uint32_t)j, a.t.div_page);
    const int p = __shfl(page, e - first);
    const bool live = k0 + lane % ROWS < end && p >= 0 && p < a.t.pages;
    row = ((uint32_t)p * (uint32_t)a.Hk + (uint32_t)hk) * (uint32_t)a.t.page + (uint32_t)(j - e * a.t.page);
    row = live ? row : kSaDead;
    return __ballot(live && lane < ROWS);
  }
};

// The tiles of 64 states (or of 32: ROWS) that a wave walks over, from part [t, t1) of a
// span; ones without a live state are passed over.
template <bool PAGED, int ROWS, int STEP>
struct STiles {
  SPages<ROWS> pages;
  const uint8_t* mask;
  int t, t1, end, k0;
  int below = 0;  // states below this, but the sinks, are seen by no row (whose span is wider)
  uint32_t raw;
  uint64_t live;
  __device__ __forceinline__ int state(const SSpan& span, int i) const {
    if constexpr (ROWS == 64) return span.state(i);
    else return span.state(i >> 1) + 32 * (i & 1);
  }
  __device__ __forceinline__ uint32_t load(const SSpan& span, int i) const {
    const int k = state(span, i) + (int)(threadIdx.x & 63);
    return i < t1 && k < end ? mask[k] : 0;
  }
  __device__ __forceinline__ void init(const SSpan& span, int t_, int t1_, int end_) {
    t = t_ - STEP;
    t1 = t1_;
    end = end_;
    if (!PAGED && mask) raw = load(span, t_);
  }
  __device__ __forceinline__ bool advance(const SAttnArgs& a, const SSpan& span) {
    for (;;) {
      t += STEP;
      if (t >= t1) return false;
      k0 = state(span, t);
      if constexpr (PAGED) {
        live = k0 < end && (k0 + ROWS > below || k0 < a.sinks) ? pages.at(a, k0, end) : 0;
      } else if (mask) {
        live = __ballot(raw != 0);
        raw = load(span, t + STEP);
      } else {
        live = sa_ones(end - 1 - k0);
      }
      if (live) return true;
    }
  }
};

// The larger exponents of the pairs of x and `most`, whose two halves tell whether any of the
// values that passed is not finite.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <bool F16>
struct SExponents {
  static constexpr uint16_t top = F16 ? 0x7c00u : 0x7f80u;
  u16x2 most = {0, 0};
  __device__ __forceinline__ void add(bf16x8 f) {
    const u32x4 x = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[e] & (top * 0x10001u)));
  }
  __device__ __forceinline__ bool bad() const { return most[0] == top || most[1] == top; }
};

// Which of the 32 tile rows from rbase on hold a value that is not finite.
template <int DP, bool F16>
__device__ __forceinline__ uint32_t sa_bad_rows(const u16* T, int rbase) {
  SExponents<F16> x;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) x.add(xa_frag<DP>(T, rbase, s));
  const uint64_t rows = __ballot(x.bad());
  return (uint32_t)(rows | rows >> 32);
}
// A fragment with zeros in the place of values that are not finite.
template <bool F16>
__device__ __forceinline__ bf16x8 sa_finite(bf16x8 f) {
  constexpr uint32_t top = F16 ? 0x7c00u : 0x7f80u;
  u32x4 x = __builtin_bit_cast(u32x4, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((x[e] & top) == top) x[e] &= 0xffff0000u;
    if (((x[e] >> 16) & top) == top) x[e] &= 0xffffu;
  }
  return __builtin_bit_cast(bf16x8, x);
}

// Calls mark(row) for the rows of a tile's chunks (64 (n w + t) + lane, as its loader put them
// there) that hold a value that is not finite; CLEAN: and puts zeros in the values' place.
template <int DP, int NI, bool F16, bool CLEAN, typename F>
__device__ __forceinline__ void sa_look(u16* T, int w, F mark) {
  bf16x8* at = reinterpret_cast<bf16x8*>(T) + 64 * NI * w + (threadIdx.x & 63);
  SExponents<F16> all;
#pragma unroll
  for (int t = 0; t < NI; ++t) all.add(at[64 * t]);
  if (__ballot(all.bad()) == 0) return;
#pragma unroll 1
  for (int t = 0; t < NI; ++t) {
    SExponents<F16> x;
    x.add(at[64 * t]);
    if (x.bad()) {
      if constexpr (CLEAN) at[64 * t] = sa_finite<F16>(at[64 * t]);
      mark((64 * (NI * w + t) + (int)(threadIdx.x & 63)) / (DP / 8));
    }
  }
}

// What rows see that is not finite, beside their sums: two bits a channel, 1 +inf, 2 -inf,
// both NaN, 16 channels a word.
template <int DP>
struct SPoison {
  static constexpr int WORDS = DP / 16;  // a row
  // Adds what the lane's row sees (`sees`) of the tile rows `bad`.
  template <bool F16>
  static __device__ __forceinline__ void note(uint32_t* row, const u16* T, uint64_t bad, uint64_t sees) {
    constexpr uint32_t top = F16 ? 0x7c00u : 0x7f80u;
    const int h = (threadIdx.x >> 5) & 1;
    while (bad) {  // (uniform)
      const int r = __builtin_ctzll(bad);
      bad &= bad - 1;
#pragma unroll 1
      for (int d = 4 * h; d < DP; d += 8) {
        const int slot = (d >> 3) ^ xa_swz<DP>(r);
        const uint2 x = *reinterpret_cast<const uint2*>(T + r * DP + slot * 8 + (d & 7));
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t v = ((e & 2 ? x.y : x.x) >> (16 * (e & 1))) & 0xffffu;
          if ((v & top) == top) bits |= ((v & 0x7fffu) > top ? 3u : v & 0x8000u ? 2u : 1u) << (2 * e);
        }
        if (bits && ((sees >> r) & 1)) atomicOr(row + (d >> 4), bits << (2 * (d & 15)));
      }
    }
  }
  // The value x of channel d of a row.
  static __device__ __forceinline__ float apply(const uint32_t* row, int d, float x) {
    const uint32_t b = (row[d >> 4] >> (2 * (d & 15))) & 3;
    if (b & 1) x += __builtin_inff();
    if (b & 2) x -= __builtin_inff();
    return x;
  }
};

// Sizes, strides and scale of a windowed call into `a` (sattn.hip); 0 or an error code.
int window_check(SAttnArgs& a, const tpf_window_shape* s, double scale, const char* fn);

inline SOrder sa_order(int64_t heads, int64_t units) {
  int64_t shared = 8;
  while (heads % shared) shared /= 2;
  SOrder o;
  o.units = (int)units;
  o.shift = shared == 8 ? 0 : shared == 4 ? 1 : shared == 2 ? 2 : 3;
  o.subs = (uint32_t)(heads / shared);
  o.together = o.subs == 2 ? 2 : 1;
  o.each = (uint32_t)((units + (8 / shared) - 1) / (8 / shared));
  o.groups = 8 * (int64_t)o.subs * o.each;
  return o;
}

}  // namespace tpf
