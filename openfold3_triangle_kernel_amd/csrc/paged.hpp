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

// The last s in [0, last] for which before(s) holds; before ascends from true (s = 0 is
// taken to hold) to false.  A wave compares 64 at a time.
template <typename F>
__device__ __forceinline__ int paged_search(int last, F before) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = last + 1;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 63) / 64, s = lo + 1 + lane * step;
    const int c = __popcll(__ballot(s < hi && before(s < hi ? s : last)));
    const int next = c ? lo + 1 + (c - 1) * step : lo;
    hi = c ? min(hi, next + step) : lo + 1;
    lo = next;
  }
  return lo;
}

// The batch of a call into t; 0 or an error code (rotary.hip).
int paged_check(PagedTables& t, const tpf_paged_batch* batch, const char* fn);

}  // namespace tpf
