// 8-bit (e4m3) values with a scale per block of 128: the quantisation rule and
// the conversions shared by the kernels that write and read them.
//
// A block is 128 consecutive columns of a row (activations) or 128 x 128
// elements (weights).  Its scale is the smallest power of two s with
// max|v| / s <= 448 over the block's finite v (1 for a block of zeros, never
// below 2^-126), so v / s is exact and each stored value is one rounding (half
// to even) of it.  A non-finite v is stored as NaN.
#pragma once

#include "tm_mfma.h"

constexpr int kFp8Block = 128;

// max|v| of a block over its finite elements, from fp32 bit patterns: for
// non-negative floats the integer order is the float order.
__device__ __forceinline__ uint32_t tm_fp8_amax(uint32_t m, float v) {
  const uint32_t a = __float_as_uint(v) & 0x7fffffffu;
  return a < 0x7f800000u && a > m ? a : m;
}

// Maximum over each 16-lane row of the wave, in every lane of it.
__device__ __forceinline__ uint32_t tm_row16_max(uint32_t v) {
  v = max(v, tm_dpp<0xB1>(v, v));   // quad_perm [1,0,3,2]
  v = max(v, tm_dpp<0x4E>(v, v));   // quad_perm [2,3,0,1]
  v = max(v, tm_dpp<0x141>(v, v));  // row_half_mirror
  v = max(v, tm_dpp<0x140>(v, v));  // row_mirror
  return v;
}

// The block scale of max|v| (bits): a / s <= 448 = 1.75 * 2^8 with a = m 2^e,
// 1 <= m < 2, asks for s = 2^(e - 8), or 2^(e - 7) where m > 1.75.  Subnormal
// a gives the smallest scale.  `inv` receives 1 / s (exact).
__device__ __forceinline__ float tm_fp8_scale(uint32_t amax, float &inv) {
  int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased exponent of s
  b = b < 1 ? 1 : b;
  b = amax == 0 ? 127 : b;
  inv = __uint_as_float((uint32_t)(254 - b) << 23);
  return __uint_as_float((uint32_t)b << 23);
}

// The quotient to be rounded: non-finite values become NaN.
__device__ __forceinline__ float tm_fp8_quot(float v, float inv) {
  return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u ? v * inv : __uint_as_float(0x7fc00000u);
}

// Four values to e4m3, packed in order.
__device__ __forceinline__ uint32_t tm_fp8_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

typedef __bf16 tm_bf16x2 __attribute__((ext_vector_type(2)));

// Eight e4m3 values, times a power of two, as bf16 (exact: 4 significant bits;
// apart from products under 2^-126, which blocks of max|v| < 2^-108 alone can have,
// and of values within 3 % of 2^128, whose e4m3 neighbour is 2^128).
__device__ __forceinline__ uint4 tm_fp8_to_bf16x8(uint32_t lo, uint32_t hi, float s = 1.f) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true));
  return r;
}

// Matrix product of 32 x 64 by 64 x 32 e4m3 values: lane l holds row (column)
// l % 32 and 32 of the 64, the same ones in both operands; D as in the 32x32x16
// form.
typedef int tm_i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ tm_f32x16 tm_mfma32x32x64_fp8(const uint4 (&a)[2], const uint4 (&b)[2], tm_f32x16 c) {
  const tm_i32x8 x = {(int)a[0].x, (int)a[0].y, (int)a[0].z, (int)a[0].w,
                      (int)a[1].x, (int)a[1].y, (int)a[1].z, (int)a[1].w};
  const tm_i32x8 y = {(int)b[0].x, (int)b[0].y, (int)b[0].z, (int)b[0].w,
                      (int)b[1].x, (int)b[1].y, (int)b[1].z, (int)b[1].w};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);
}

// The 16 x 128 by 128 x 16 form: row (column) l % 16, 32 of the 128; D as in the
// 16x16x32 form.
__device__ __forceinline__ tm_f32x4 tm_mfma16x16x128_fp8(const uint4 (&a)[2], const uint4 (&b)[2], tm_f32x4 c) {
  const tm_i32x8 x = {(int)a[0].x, (int)a[0].y, (int)a[0].z, (int)a[0].w,
                      (int)a[1].x, (int)a[1].y, (int)a[1].z, (int)a[1].w};
  const tm_i32x8 y = {(int)b[0].x, (int)b[0].y, (int)b[0].z, (int)b[0].w,
                      (int)b[1].x, (int)b[1].y, (int)b[1].z, (int)b[1].w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);
}
