// Sequences over a paged cache: where a batch's new tokens lie, and where a state's
// row is.
//
// A batch packs the new tokens of S sequences: those of sequence s are the rows
// starts[s] .. starts[s + 1] of T, and are the last of its lengths[s] states.  State j
// lies in page tables[s][j / P] at place j % P.  The tables are device data that the
// host never reads, so the kernels take any value: starts are held to [0, T], lengths
// to the table's width, and a page that the cache does not have holds no state.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"
#include "tpf_amd.h"

namespace tpf {

struct PagedTables {
  const int32_t* tables;   // [S, width], sequences table_ld apart
  const int32_t* starts;   // [S + 1]
  const int32_t* lengths;  // [S]
  int64_t table_ld;
  int64_t T;               // rows of the batch
  int S, width, page, pages;
  FastDiv div_page;
};

// starts[s] held to [0, T]; the first sequence begins with row 0.
__host__ __device__ inline int64_t paged_start(const PagedTables& t, int s) {
  const int64_t v = s ? t.starts[s] : 0;
  return v < 0 ? 0 : v > t.T ? t.T : v;
}

// lengths[s] held to what the table can hold.
__host__ __device__ inline int64_t paged_length(const PagedTables& t, int s) {
  const int64_t v = t.lengths[s], most = (int64_t)t.width * t.page;
  return v < 0 ? 0 : v > most ? most : v;
}

// Page and place of state j of sequence s; false where there is none: outside the
// table, or in a page that the cache does not have.
__host__ __device__ inline bool paged_place(const PagedTables& t, int s, int64_t j, int64_t* page,
                                            int64_t* place) {
  if (j < 0 || j >= (int64_t)t.width * t.page) return false;
  const uint32_t at = (uint32_t)j / (uint32_t)t.page;  // (a table holds 2^30 states at most)
  const int64_t p = t.tables[s * t.table_ld + at];
  *page = p;
  *place = (uint32_t)j - at * (uint32_t)t.page;
  return p >= 0 && p < t.pages;
}

// How the 64 numbers of a search are asked about, and a uniform value kept: by a wave, or
// one after the other on the host.
struct PagedWave {
  // Of the numbers first + l * step below end, l = 0 .. 63, how many hold; `last` is asked
  // about in the place of others.
  template <typename F>
  static __device__ __forceinline__ int count(int first, int step, int end, int last, F holds) {
    const int s = first + (int)(threadIdx.x & 63) * step;
    return __popcll(__ballot(s < end && holds(s < end ? s : last)));
  }
  static __device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
};
struct PagedHost {
  template <typename F>
  static int count(int first, int step, int end, int, F holds) {
    int c = 0;
    for (int64_t l = 0, s = first; l < 64 && s < end; ++l, s += step) c += holds((int)s) ? 1 : 0;
    return c;
  }
  static int scalar(int x) { return x; }
};

// The last s in [0, last] for which before(s) holds, where before ascends from true (s = 0
// is taken to hold) to false, 64 comparisons at a time; for any other before some s in
// [0, last], before or behind what is looked for.
template <typename W, typename F>
__host__ __device__ __forceinline__ int paged_search(int last, F before) {
  int lo = 0, hi = last + 1;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64;
    const int c = W::count(lo + 1, step, hi, last, before);
    const int next = c ? lo + 1 + (c - 1) * step : lo;
    hi = c ? (hi < next + step ? hi : next + step) : lo + 1;
    lo = next;
  }
  return lo;
}

// Rows of a batch with G of them a token (the query heads of a kv head): of which sequence,
// and where there.  Sequence S has the rows behind the last one.
struct PagedRows {
  int s, r0, R, fresh;  // first row, of all in the sequence, its new tokens
  int64_t token;        // the sequence's first token in the batch
  template <typename W>
  __host__ __device__ __forceinline__ void sequence(const PagedTables& t, int G, int s_) {
    s = s_;
    token = paged_start(t, s);
    const int64_t next = s < t.S ? paged_start(t, s + 1) : t.T;
    fresh = (int)(next > token ? next - token : 0);
    R = W::scalar(fresh * G);
  }
  // Row tile `tile` of rt rows (a power of two); false where no sequence has it: the search
  // ends before it, past a sequence's rows, or, where starts do not ascend, behind it.
  // Sequence s has the tiles from starts[s] G / rt + s on, enough for its rows whatever its
  // length.
  template <typename W>
  __host__ __device__ __forceinline__ bool tile(const PagedTables& t, int G, int rt, int tile) {
    // (T G + S rt is below 2^31.)
    auto before = [&](int x) { return (int)((uint32_t)paged_start(t, x) * (uint32_t)G / (uint32_t)rt) + x; };
    sequence<W>(t, G, W::scalar(paged_search<W>(t.S, [&](int x) { return before(x) <= tile; })));
    r0 = W::scalar((tile - before(s)) * rt);
    return r0 >= 0 && r0 < R;
  }
  // Row `row` of the batch, likewise.
  template <typename W>
  __host__ __device__ __forceinline__ bool row(const PagedTables& t, int G, int64_t row) {
    const int64_t at = row / G;
    sequence<W>(t, G, W::scalar(paged_search<W>(t.S, [&](int x) { return paged_start(t, x) <= at; })));
    r0 = (int)(row - token * G);
    return r0 >= 0 && r0 < R;
  }
};

// The batch of a call into t; 0 or an error code (rotary.hip).
int paged_check(PagedTables& t, const tpf_paged_batch* batch, const char* fn);

}  // namespace tpf
