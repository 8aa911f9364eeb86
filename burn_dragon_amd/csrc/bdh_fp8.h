// 8-bit values of kept activations: e4m3 with one power of two for 32 neighbours.
//
// Of a block with the largest finite magnitude a the power is 2^e, e the least
// integer with a <= 448 * 2^e (448 = 1.75 * 2^8 is e4m3's largest) and at least
// kLeastExp.  A value x is held as e4m3(x * 2^-e), to nearest, ties to even: off by at most
// half a step, 2^-4 of it, or 2^-10 * 2^e where it is below 2^-6 * 2^e.  The
// product by a power of two is exact and so is the way back, to f32 and to bf16.
// With the largest power, 2^120, the codes past 240 would stand for 2^128 and more:
// finite values past 240 * 2^120 are held as that.  Infinities and NaN are held as NaN.
// The power is kept as the byte e + 127.
#pragma once

#include "bdh_common.h"

namespace bdh {

constexpr int kFp8Block = 32;
// Below it the least step, 2^-9 * 2^e, would leave f32's (and bf16's) normal range.
constexpr int kLeastExp = -117;

typedef float floatx2 __attribute__((ext_vector_type(2)));

// |x|'s bits where x is finite, else 0: the largest of these is a's.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// The block's byte e + 127 from a's bits: a = m 2^k has e = k - 8, one more where
// m > 1.75 (the carry of the sum).
__device__ __forceinline__ int fp8_scale(uint32_t bits) {
  const int e = (int)((bits + 0x1fffffu) >> 23) - 8;
  return e > kLeastExp + 127 ? e : kLeastExp + 127;
}
__device__ __forceinline__ float fp8_power(int scale) { return __uint_as_float((uint32_t)scale << 23); }
// The largest of the finite magnitudes of a lane's values, as bits: one instruction for two
// values (three where they are signed) unless a lane of the wave has an infinity or a NaN.
template <bool SIGNED, int N, typename V>
__device__ __forceinline__ uint32_t finite_top(const V& x) {
  constexpr uint32_t magnitude = SIGNED ? 0x7fffffffu : 0xffffffffu;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const uint32_t a = __float_as_uint(x[j]) & magnitude, b = __float_as_uint(x[j + 1]) & magnitude;
    top = max(max(top, a), b);
  }
  if (__ballot(top >= 0x7f800000u) != 0) {
    top = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) top = max(top, finite_bits(x[j]));
  }
  return top;
}
// Values of a block of the largest power stay finite.
template <int N>
__device__ __forceinline__ void fp8_keep_finite(float (&x)[N], int scale) {
  if (scale < 247) return;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (fabsf(x[j]) > 0x1.ep127f && fabsf(x[j]) < INFINITY) x[j] = copysignf(0x1.ep127f, x[j]);
}
// Four values of a block, first in the lowest byte.  (The conversions take the power's
// exponent, and give NaN past 464 times it, so for an infinity too.)
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float power) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, power, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, power, true);
  return __builtin_bit_cast(uint32_t, w);
}
__device__ __forceinline__ void fp8_unpack4(uint32_t w, float power, float (&x)[4]) {
  const floatx2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, power, false);
  const floatx2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, power, true);
  x[0] = lo.x;
  x[1] = lo.y;
  x[2] = hi.x;
  x[3] = hi.y;
}

}  // namespace bdh
