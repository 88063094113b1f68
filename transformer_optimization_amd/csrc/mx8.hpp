// 8-bit cache rows: e4m3 codes and one scale 2^(byte - 127) (e8m0) for every 32
// elements of a head.
//
// The scale is the smallest power of two that keeps the block's largest
// magnitude within e4m3's 448, so no element saturates: one that is 2^-14 of the
// largest or more is off by at most 2^-4 of itself, smaller ones by 2^-10 of the
// code step at the bottom.  Powers of two, because a code has 4 significant bits:
// code x scale is then exact in bf16 and, with the two bounds below, in fp16, and
// the 16-bit matrix instructions work on the very values that the cache stands
// for.  A scale byte of 255 stands for NaN (its block's values are NaN).
#pragma once

#include "common.hpp"

namespace tx {

constexpr int MX_BLOCK = 32;

template <typename T> struct Mx;
template <> struct Mx<bf16> {
  // The smallest code step, 2^(LOWEST - 9), is the smallest normal value.
  static constexpr int LOWEST = -117;
  static constexpr float TOP = 0x1.ep127f;  // the largest magnitude that rounds to 4 bits within the type
};
template <> struct Mx<f16> {
  static constexpr int LOWEST = -15;  // 2^-24, the smallest subnormal value
  static constexpr float TOP = 61440.f;
};

// Exponent of the scale of a block whose largest magnitude is amax (finite).
template <typename T> __device__ __forceinline__ int mx_exponent(float amax) {
  const uint32_t x = __builtin_bit_cast(uint32_t, amax);
  // 448 = 1.75 * 2^8
  const int e = (int)(x >> 23) - 127 - 8 + ((x & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > Mx<T>::LOWEST ? e : Mx<T>::LOWEST;
}
__device__ __forceinline__ float mx_power(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// What of x a block's maximum counts: finite magnitudes, no more than TOP.
template <typename T> __device__ __forceinline__ float mx_magnitude(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_inff() ? fminf(a, Mx<T>::TOP) : 0.f;
}
// x as it is held: magnitudes above TOP count as that; NaN for what is not finite.
template <typename T> __device__ __forceinline__ float mx_within(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_inff() ? __builtin_copysignf(fminf(a, Mx<T>::TOP), x) : __builtin_nanf("");
}
// Codes of four values times inv = 2^-e: rounded to nearest even.
__device__ __forceinline__ uint32_t mx_codes(const float* x, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inv, x[3] * inv, r, true);
  return (uint32_t)r;
}

// Eight codes -> eight 16-bit values (exact; beyond fp16's range infinite).
template <typename T> __device__ __forceinline__ u32x4 mx_values(uint32_t lo, uint32_t hi, float scale) {
  u32x4 r;
  if constexpr (std::is_same<T, bf16>::value) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
  }
  return r;
}

}  // namespace tx
