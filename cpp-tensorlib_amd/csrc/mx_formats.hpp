// The microscaled formats: rows in blocks of 32 elements, e2m1 (MXFP4, two to a byte, the even element in the low nibble) or
// e4m3 (MXFP8), with a scale byte each that stands for 2^(byte - 127); 255 is NaN.
#pragma once

#include "common.hpp"

namespace tlhip {

constexpr int kMxBlock = 32;
constexpr int kMx4Exp = 2, kMx8Exp = 8;            // exponents of the largest elements, 6 and 448
constexpr float kMx8Max = 448.f;

// What every entry point over these formats asks of a row: whole blocks. Scale bytes need no alignment.
inline bool mx_row(int64_t K) { return K > 0 && K % kMxBlock == 0; }

#if defined(__HIPCC__)
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// The scale byte of a block: the exponent of its largest magnitude less that of the element type's largest. `big` is that magnitude's
// bit pattern (compared as integers: a NaN is the largest of all, so a block with an infinity or a NaN gets 255).
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t big, int largest) {
  const uint32_t field = big >> 23;
  return field == 255u ? 255u : (uint32_t)max((int)field - largest, 0);
}
// 2^(127 - s), what elements are multiplied by (exact: a power of two; s <= 252 here)
__device__ __forceinline__ float mx_up(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127): a subnormal for 0, NaN for 255
__device__ __forceinline__ float mx_scale(uint32_t s) {
  return __uint_as_float(s == 0u ? 0x00400000u : s == 255u ? 0x7fc00000u : s << 23);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Elements from scaled values, rounded to nearest even, saturating (the conversion to e2m1 does so by itself, the one to e4m3
// would give NaN).
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&v)[8]) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
}
__device__ __forceinline__ float e4m3_range(float v) { return __builtin_amdgcn_fmed3f(v, -kMx8Max, kMx8Max); }
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(a), e4m3_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(c), e4m3_range(d), r, true);
}
#endif

}  // namespace tlhip
