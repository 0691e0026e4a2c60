// The 4-bit KV encoding: arithmetic shared by its kernels (gfx950).
//
// 128 values of a (token, kv head) row are 64 bytes of codes and four bytes of
// powers.  A code is a 4-bit float (one sign, two exponent, one mantissa bit:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6), dim 2 j in the low half of byte j; byte g of the
// powers is the exponent + 127 of the power of two that scales dims 32 g .. 32 g
// + 31.  It is the smallest that takes the run's largest magnitude to 6 or
// less, so no value saturates below the top of the range: rounding the exponent
// down instead (magnitudes up to 8 saturating at 6) would cost the largest
// value of a run up to a quarter, and in keys the largest are what a score
// hangs on.  The format is one that the card converts in hardware, both ways:
// v_cvt_scalef32_pk_fp4_bf16 rounds to nearest, ties to the even mantissa, and
// v_cvt_scalef32_pk_bf16_fp4 is exact (two significant bits and a power of two).
#pragma once

#include "kvc_internal.h"

namespace kvc {

constexpr int kFp4RowBytes = 64;
constexpr int kFp4Powers = 4;
constexpr int kPowerNaN = 255;    // a run that held an infinity or a NaN (codes 0)
constexpr int kPowerLow = 1;      // 2^-126
constexpr int kPowerHigh = 252;   // 2^125: 6 times that is still finite

// The power byte of a run whose largest magnitude has the bf16 bits `top`.
// top = m 2^x with 1 <= m < 2; 6 is 1.5 x 2^2, so the exponent is x - 2, and one
// more for m > 1.5 (mantissa field > 64 of 128).
__device__ __forceinline__ int power_of_top(uint32_t top) {
  if (top >= 0x7f80u) return kPowerNaN;
  const int e = int(top >> 7) - 2 + ((top & 127u) > 64u ? 1 : 0);
  return min(max(e, kPowerLow), kPowerHigh);
}

__device__ __forceinline__ float power_f32(int byte) {
  return __uint_as_float(byte == kPowerNaN ? 0x7fc00000u : uint32_t(byte) << 23);
}

// Eight bf16 values (two to a dword) as codes.
__device__ __forceinline__ uint32_t quant_fp4x8(const u32x4_t& x, float power) {
  // (by value: a bit cast of a vector's element in place takes element 0)
  const uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, x0), power, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, x1), power, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, x2), power, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, x3), power, 3);
  return c;
}

// Eight codes as bf16.
__device__ __forceinline__ u32x4_t dequant_fp4x8(uint32_t c, float power) {
  return u32x4_t{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, power, 3))};
}

// The largest magnitude (bf16 bits) of a lane's eight values.
__device__ __forceinline__ uint32_t top_bits(const u32x4_t& x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  return top;
}

}  // namespace kvc
