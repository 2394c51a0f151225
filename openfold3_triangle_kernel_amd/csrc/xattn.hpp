// Shared pieces of the cross-attention kernels (xattn.hip, xattn_bwd.hip).
//
// Rows and states.  The key mask does not depend on the query, so the queries
// of the G query heads that share a kv head are one row axis: row r = g * Nq + i
// of kv head (b, hk) is query i of head hk * G + g, and every kernel works on
// R = G * Nq rows against Nk states.
//
// Tiles.  K, V, Q and dO tiles are rows of DP channels (D rounded up to 32, 64,
// 96 or 128) in LDS, loaded there directly 16 bytes a lane; absent rows, dead
// states and the channels past D read as zeros.  Chunk c (16 bytes) of row r
// sits at slot c ^ xa_swz(r).  A row-wise fragment read (16 rows, one chunk)
// then meets 16 different slots of the 256 bytes that LDS serves at a time,
// and a transposing read (4 rows, two chunks) meets four different pairs.
#pragma once

#include "common.hpp"
#include "tpf_amd.h"

namespace tpf {

enum { kMaskNone = 0, kMaskBool = 1, kMaskF32 = 2 };

struct XAttnArgs {
  const u16 *q, *k, *v;
  int64_t q_sb, q_sh, q_sn, k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;  // element strides
  const void* mask;
  int64_t mask_sb;
  int mask_kind;
  u16* out;    // [B, Nq, H, D]
  u16* res;    // what its rounding drops, laid out the same; null when not wanted
  float* lse;  // the rows' statistics (xa_store_stats); null when no backward follows
  int B, H, Hk, G, Nq, Nk, D, R;
  FastDiv div_nq;
  float c;          // scale * log2(e)
  float inv_scale;  // additive masks enter the raw scores divided by the scale
  float mask_floor; // lowest finite raw mask value, its negative the highest
  int splits, chunk, tiles;  // state splits, states per split (a multiple of 64), row tiles
  int qb;           // blocks of 32 rows a wave
  int kw;           // groups of four waves that share a row tile's states
  float* part_o;    // [B*Hk, splits, R, D] unnormalised outputs of the splits
  float* part_ml;   // [B*Hk, splits, R, 3] their raw maxima and the two sums (XRows)
};

template <int DP>
__device__ __forceinline__ int xa_swz(int r) {
  if constexpr (DP == 128) return ((r & 7) << 1) | ((r >> 3) & 1);
  else if constexpr (DP == 64) return ((r & 6) | ((r >> 3) & 1));
  else return (r >> 2) & 3;  // 32, 96: four rows fill the 256 bytes
}

// 16 x 32 x 32 matrix step of the operands' type.
template <bool F16>
__device__ __forceinline__ f32x16 xa_mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  if constexpr (F16) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    return mfma32(a, b, c);
  }
}

// Two f32 rounded to nearest as a pair of 16-bit operands.
template <bool F16>
__device__ __forceinline__ uint32_t xa_pair(float lo, float hi) {
  if constexpr (F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    f16x2 p;
    p[0] = (_Float16)lo;
    p[1] = (_Float16)hi;
    return __builtin_bit_cast(uint32_t, p);
  } else {
    bf16x2 p;
    p[0] = f2bf(lo);
    p[1] = f2bf(hi);
    return __builtin_bit_cast(uint32_t, p);
  }
}
// Registers r0 .. r0 + 7 of a C tile as an MFMA operand.
template <bool F16>
__device__ __forceinline__ bf16x8 xa_pack8(const f32x16& c, int r0) {
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = xa_pair<F16>(c[r0 + 2 * e], c[r0 + 2 * e + 1]);
  return __builtin_bit_cast(bf16x8, o);
}

// The larger of two values, NaN where one is (v_maximum3_f32: three values a step, and
// no quieting of its operands first): a NaN score makes its row's maximum NaN.
__device__ __forceinline__ float xa_max(float x, float y) {
  return __builtin_elementwise_maximum(x, y);
}
__device__ __forceinline__ float xa_min(float x, float y) {
  return __builtin_elementwise_minimum(x, y);
}
// The larger of a lane's and lane ^ 32's value.
__device__ __forceinline__ float xa_max32(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return xa_max(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Adds the two 16-bit values of a pair to acc, in 32 bits.
template <bool F16>
__device__ __forceinline__ float xa_add_pair(uint32_t pair, float acc) {
  if constexpr (F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair),
                                  __builtin_bit_cast(f16x2, 0x3c003c00u), acc, false);
  } else {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
  }
}

// Row-wise fragment: row rbase + lane % 32, channels 16 s + 8 (lane / 32) .. + 8.
template <int DP>
__device__ __forceinline__ bf16x8 xa_frag(const u16* T, int rbase, int s) {
  const int l = threadIdx.x & 63;
  const int r = rbase + (l & 31), slot = (2 * s + (l >> 5)) ^ xa_swz<DP>(r);
  return *reinterpret_cast<const bf16x8*>(T + r * DP + slot * 8);
}

// Transposed fragment: channel 32 db + lane % 32 of the eight rows that
// registers 8 t .. 8 t + 7 of a C tile hold in this lane (rows 16 t + 4 h + e and
// 16 t + 8 + 4 h + e, h = lane / 32, e < 4), relative to rbase.
template <int DP>
__device__ __forceinline__ bf16x8 xa_frag_t(const u16* T, int rbase, int t, int db) {
  const int l = threadIdx.x & 63, g = l >> 4, ip = l & 15;
  const int col = 32 * db + 16 * (g & 1) + 4 * (ip & 3);
  bf16x4 h[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = rbase + 16 * t + 8 * e + 4 * (g >> 1) + (ip >> 2);
    const int slot = (col >> 3) ^ xa_swz<DP>(r);
    h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (lds_bf16x4*)(T + r * DP + slot * 8 + (col & 7)));
  }
  return cat8(h[0], h[1]);
}

// Loader of a [ROWS][DP] tile of K or V by NW waves (w: this wave's number).
// The lane's offsets are fixed; the tile's first row is the buffer's base, in
// 64 bits.
template <int DP, int ROWS, int NW>
struct XTileLoader {
  static constexpr int CPR = DP / 8, NI = ROWS * CPR / 64 / NW;
  static_assert(ROWS * CPR % (64 * NW) == 0, "whole instructions");
  uint32_t off[NI];
  __device__ __forceinline__ int row(int w, int t) const {
    return (64 * (NI * w + t) + (int)(threadIdx.x & 63)) / CPR;
  }
  __device__ __forceinline__ void init(int w, int64_t sn, int D) {
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const int p = 64 * (NI * w + t) + (int)(threadIdx.x & 63), r = p / CPR;
      const int chunk = (p - r * CPR) ^ xa_swz<DP>(r);
      off[t] = 8 * chunk < D ? (uint32_t)(r * sn + 8 * chunk) * 2u : kBufOOB;
    }
  }
  // Rows whose bit of `live` is clear read as zeros.
  __device__ __forceinline__ void issue(const u16* base, uint64_t live, int w, u16* T) const {
    const i32x4 rsrc = buffer_rsrc(base);
    char* dst = reinterpret_cast<char*>(T);
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const uint32_t o = (live >> row(w, t)) & 1 ? off[t] : kBufOOB;
      buf2lds16(rsrc, o, dst + (NI * w + t) * 1024);
    }
  }
};

// A live additive value, given by its bits, in raw score units: finite ones within
// +-floor_, so that they stay finite beside any score.  NaN and infinity are told by the
// bits and pass as they are: their rows are NaN, as the formula's.  (A clamp alone would
// turn a NaN into the floor, a state without weight.)
__device__ __forceinline__ float xa_raw_mask(uint32_t m, float inv_scale, float floor_) {
  const float x = __builtin_amdgcn_fmed3f(__uint_as_float(m) * inv_scale, floor_, -floor_);
  return (m & 0x7fffffffu) < 0x7f800000u ? x : __uint_as_float(m);
}

// The masks of the 64 states from k0 on: lane l holds state k0 + l.  What a
// dead or absent state gives is 0 in `live`.  Additive values are held as
// bits: -inf is a dead state, a NaN is not.
struct XMask {
  const uint8_t* b = nullptr;
  const float* f = nullptr;
  int kind, Nk;
  __device__ __forceinline__ void init(const XAttnArgs& a, int batch) {
    kind = a.mask_kind;
    Nk = a.Nk;
    if (kind == kMaskBool) b = (const uint8_t*)a.mask + (int64_t)batch * a.mask_sb;
    if (kind == kMaskF32) f = (const float*)a.mask + (int64_t)batch * a.mask_sb;
  }
  // The lane's raw value: 0 / 1, or the float's bits.
  __device__ __forceinline__ uint32_t load(int k0, int kend) const {
    const int k = k0 + (int)(threadIdx.x & 63);
    if (k >= kend) return kind == kMaskF32 ? 0xff800000u : 0u;
    if (kind == kMaskBool) return b[k];
    if (kind == kMaskF32) return __float_as_uint(f[k]);
    return 1u;
  }
  __device__ __forceinline__ uint64_t live(uint32_t raw) const {
    return __ballot(kind == kMaskF32 ? raw != 0xff800000u : raw != 0u);
  }
  // Whether an additive mask has values other than 0 and -inf here.
  __device__ __forceinline__ bool values(uint32_t raw) const {
    return kind == kMaskF32 && __ballot(raw != 0xff800000u && (raw << 1) != 0u) != 0;
  }
};

// Applies the masks of 32 states from k0 on to a C tile whose registers are
// states: dead ones to -inf (by bit, whatever the score is), additive values
// in raw units.
__device__ __forceinline__ void xa_mask32(f32x16& s, uint32_t live, const float* f, int k0, int Nk,
                                          float inv_scale, float floor_) {
  const int h = (threadIdx.x >> 5) & 1;
  if (f) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int k = k0 + 8 * (r >> 2) + 4 * h + (r & 3);
      const uint32_t m = k < Nk ? reinterpret_cast<const uint32_t*>(f)[k] : 0u;
      s[r] += xa_raw_mask(m, inv_scale, floor_);
    }
  }
  const uint32_t w = live >> (4 * h);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (!((w >> (8 * (r >> 2) + (r & 3))) & 1)) s[r] = -__builtin_inff();
}

// The tiles of 64 states that a workgroup walks over, KW at a time (one for each
// group of four waves), in the order of the states; rounds without a live state are
// passed over.  Every wave keeps the same state, so all take the same turns.
template <int KW>
struct XTiles {
  XMask mask;
  int k0, kend;
  uint32_t raw[KW];
  uint64_t live[KW];
  bool values[KW];
  __device__ __forceinline__ void init(const XAttnArgs& a, int batch, int kbeg, int kend_) {
    mask.init(a, batch);
    k0 = kbeg - 64 * KW;
    kend = kend_;
#pragma unroll
    for (int t = 0; t < KW; ++t) raw[t] = mask.load(kbeg + 64 * t, kend);
  }
  // To the next round with a live state; false past the end.
  __device__ __forceinline__ bool advance() {
    for (;;) {
      k0 += 64 * KW;
      if (k0 >= kend) return false;
      uint64_t any = 0;
#pragma unroll
      for (int t = 0; t < KW; ++t) {
        live[t] = mask.live(raw[t]);
        values[t] = mask.values(raw[t]);
        raw[t] = mask.load(k0 + 64 * (KW + t), kend);
        any |= live[t];
      }
      if (any) return true;
    }
  }
};

// Hands N blocks of a wave's accumulators from the second group of four waves to
// the first through LDS (4 waves x N x 4 KiB); `w`: the wave's number in its group.
template <int N>
__device__ __forceinline__ void xa_give(char* lds, int w, const f32x16 (&o)[N]) {
  f32x4* p = reinterpret_cast<f32x4*>(lds) + w * N * 256 + (threadIdx.x & 63);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[n][4 * q + e];
      p[(4 * n + q) * 64] = v;
    }
}
// o = mine * o + other * (what the second group's wave gave).
template <int N>
__device__ __forceinline__ void xa_take(const char* lds, int w, f32x16 (&o)[N], float mine,
                                        float other) {
  const f32x4* p = reinterpret_cast<const f32x4*>(lds) + w * N * 256 + (threadIdx.x & 63);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 v = p[(4 * n + q) * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][4 * q + e] = mine * o[n][4 * q + e] + other * v[e];
    }
}

// Address of row r (already split) in a [B, H, Nq, D] operand.
__device__ __forceinline__ void xa_row(const XAttnArgs& a, int r, int& g, int& i) {
  g = (int)fdiv((uint32_t)r, a.div_nq);
  i = r - g * a.Nq;
}

// Sizes, strides and scale of a call into `a` (xattn.hip); 0 or an error code.
int xattn_check(XAttnArgs& a, const tpf_xattn_shape* s, double scale, const char* fn);

}  // namespace tpf
