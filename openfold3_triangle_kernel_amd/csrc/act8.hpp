// Rows of 32-, 16-bit types in chunks of eight channels, and the 8-bit form of
// activations.
//
// 8-bit form.  32 channels of a row share a power of two 2^k, k the smallest
// whole number from -120 on for which round(max |x| / 2^k) is at most 127, but at
// most 121 (9 for FP16 rows), so that 127 2^k is finite: a larger quotient there
// is held as 127.  A value is held as the byte 128 + round(x / 2^k) (ties to even)
// and the block's scale as the byte k + 127 (255: the block had an infinity or NaN, and every
// value of it decodes to NaN).  With a power of two the quotient is exact, so
// codes do not depend on how a kernel rounds, and a decoded value (seven bits
// times 2^k) is exact in BF16 and FP32: it goes into the matrix cores as it is.
// Codes are stored at a pitch of whole blocks, the rest of the last block
// holding 0 (byte 128).
#pragma once

#include "common.hpp"

namespace tpf {

constexpr int kActBlock = 32;

// Element types of a row: 0 BF16, 1 FP16, 2 FP32 (TPF_BF16, TPF_F16, TPF_F32).
template <int DT> struct ActType;
template <> struct ActType<0> { typedef __bf16 T; };
template <> struct ActType<1> { typedef _Float16 T; };
template <> struct ActType<2> { typedef float T; };
template <int DT> constexpr int act_bytes() { return DT == 2 ? 4 : 2; }

// Eight channels as loaded.
template <int DT> struct Raw8 { u32x4 v[DT == 2 ? 2 : 1]; };

// Loads `n` (at most 8; fewer only at a row's end) channels from p, which need
// only be aligned to the element: rows of an odd width start anywhere.
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p, int n) {
  Raw8<DT> r;
  if (n >= 8) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
    typedef typename ActType<DT>::T T;
    T e[8] = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) e[i] = reinterpret_cast<const T*>(p)[i];
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void to_f32(const Raw8<DT>& r, float (&f)[8]) {
  typedef typename ActType<DT>::T T;
  T e[8];
  __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(e[i]);
}
template <int DT>
__device__ __forceinline__ void store8(void* p, const float (&f)[8], int n) {
  typedef typename ActType<DT>::T T;
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = static_cast<T>(f[i]);
  if (n >= 8) {
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) reinterpret_cast<T*>(p)[i] = e[i];
  }
}

// Maximum over aligned groups of four lanes.
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, dpp_f<kDppXor1>(x));
  return fmaxf(x, dpp_f<kDppXor2>(x));
}

// Encodes a block whose 32 values lie in four lanes, eight each (0 past the
// row's end); returns this lane's eight bytes and the block's scale byte.
constexpr int kActTop = 121, kActTopF16 = 9;
template <int KMAX = kActTop>
__device__ __forceinline__ u32x2 encode8(const float (&f)[8], uint32_t& scale) {
  float top = 0.f;
  uint32_t odd = 0;  // an infinity or NaN among the values, by its exponent
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    top = fmaxf(top, fabsf(f[i]));
    odd |= ((__float_as_uint(f[i]) & 0x7f800000u) == 0x7f800000u) ? 1u : 0u;
  }
  top = quad_max(odd ? __builtin_inff() : top);
  u32x2 out;
  if (top == __builtin_inff()) {
    scale = 255u;
    out[0] = out[1] = 0x80808080u;
    return out;
  }
  // floor(log2 top) - 6 puts the largest into [64, 128); 127.5 and above would
  // round to 128 and takes the next power.
  int k = (int)(__float_as_uint(top) >> 23) - 127 - 6;
  k = k < -120 ? -120 : k > KMAX ? KMAX : k;
  float inv = __uint_as_float((uint32_t)(127 - k) << 23);
  if (top * inv >= 127.5f && k < KMAX) {
    ++k;
    inv *= 0.5f;
  }
  scale = (uint32_t)(k + 127);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b |= (uint32_t)((int)__builtin_amdgcn_fmed3f(__builtin_rintf(f[4 * j + i] * inv), -127.f, 127.f) +
                      128) << (8 * i);
    out[j] = b;
  }
  return out;
}

// Values of eight bytes with the scale byte of their block: (byte - 128) 2^k in
// one exact fused multiply-add; a scale of 255 gives NaN.  128 2^k passes FP32's
// range from k = 121 on: such a block is formed at half its size and doubled.
__device__ __forceinline__ void decode8(u32x2 b, uint32_t scale, float (&f)[8]) {
  const bool big = scale >= 248u && scale < 255u;
  const float s = __uint_as_float((big ? scale - 1u : scale) << 23), off = -128.f * s;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[4 * j + i] = fmaf((float)((b[j] >> (8 * i)) & 0xffu), s, off);
  if (big) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += f[i];
  }
}

}  // namespace tpf
