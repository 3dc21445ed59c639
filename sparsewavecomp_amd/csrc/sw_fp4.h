// Rows of 4-bit codes with a scale a block of 32 elements (E2M1 and E8M0): a
// code is a sign and one of the sizes 0, 1/2, 1, 3/2, 2, 3, 4, 6; the scale
// byte b stands for 2^(b - 127), 255 for NaN.  A row of d elements is d / 2
// bytes of codes, element 2 j in the low half of byte j, and d / 32 scales.
//
// A value has two significant bits, so fp32 and bf16 hold it exactly, and so
// do the products of the bf16 matrix cores with it.
#pragma once

#include "sw_heads.h"

namespace swd {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// The scale that the conversion instructions take: they read its exponent, 255
// of which makes NaN and 0 a factor of 2^-127.
__device__ __forceinline__ float fp4_scale(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// The eight values of four bytes of codes, as bf16.
__device__ __forceinline__ v4u fp4_values(uint32_t codes, float scale) {
  return v4u{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                       codes, scale, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                       codes, scale, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                       codes, scale, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                       codes, scale, 3))};
}

// The four values of two bytes of codes, as fp32.
__device__ __forceinline__ v4u fp4_values_f32(uint32_t codes, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  return __builtin_bit_cast(v4u, v4f{a[0], a[1], b[0], b[1]});
}

// The scale byte of a block whose largest size has these bits: the smallest
// power of two from 2^-125 to 2^125 that 7 times covers it (from 6 to 7 a value
// rounds to 6 as it would if there were an 8), 255 where a value is not finite.
// Of the limits that a power of two can keep, 7 gives normal values the
// smallest error (root of the mean square: 0.1118 of their deviation; 0.1155
// at 6, where no value is cut, 0.1149 at 8).
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t top) {
  // (2^k m: k - 2 where m is at most 7/4, else k - 1)
  const uint32_t byte = (top + 0x1FFFFFu) >> 23;
  return top >= 0x7F800000u ? 255u : byte < 4 ? 2u : byte > 254 ? 252u : byte - 2;
}

// The codes of eight bf16 or four fp32 values, each rounded to nearest, ties to the even code and
// sizes past 6 to 6, as the conversion instructions do.
__device__ __forceinline__ uint32_t fp4_codes(v4u x, float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      c, __builtin_bit_cast(bf16x2, (uint32_t)x[0]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      c, __builtin_bit_cast(bf16x2, (uint32_t)x[1]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      c, __builtin_bit_cast(bf16x2, (uint32_t)x[2]), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      c, __builtin_bit_cast(bf16x2, (uint32_t)x[3]), scale, 3);
}
__device__ __forceinline__ uint32_t fp4_codes(v4f x, float scale) {
  const uint32_t c =
      __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[0], x[1], scale, 0);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
}

} // namespace swd
