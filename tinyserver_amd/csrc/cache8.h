// 8-bit K/V caches: how a row of a kv head is held, and the conversions.
//
// A row x of D values is held as D codes and one float32 scale:
//   scale = max|x| / Q, Q = 448 (e4m3's largest) or 127 (int8), in float32;
//   code = x / scale, in float32, rounded once to the type (ties to even).
// A row of zeros (or one whose scale underflows to 0) has scale 0 and codes 0;
// a row that holds a NaN or an infinity has scale NaN and codes 0, so that it
// reads back as NaN. One scale per row and kv head, not per tensor or channel:
// it is found while the row is in registers, stays right whatever is written
// later, and costs 4 bytes beside 128.
#pragma once

#include "tsa_common.h"

namespace tsa {

struct e4m3_t { uint8_t x; };
struct i8_t { int8_t x; };

template <typename C> constexpr float kLargest8 = 0.f;
template <> inline constexpr float kLargest8<e4m3_t> = 448.f;
template <> inline constexpr float kLargest8<i8_t> = 127.f;

__device__ __forceinline__ float to_float(e4m3_t v) { return __builtin_amdgcn_cvt_f32_fp8(v.x, 0); }
__device__ __forceinline__ float to_float(i8_t v) { return static_cast<float>(v.x); }

// The scale of a row whose largest |x| has these bits (a NaN's bits are above
// an infinity's, and both above every number's).
template <typename C> __device__ __forceinline__ float scale8(uint32_t amax_bits) {
  return amax_bits >= 0x7F800000u ? __builtin_nanf("") : __builtin_bit_cast(float, amax_bits) / kLargest8<C>;
}

// x / scale within the type's range (0 for a scale of 0 or NaN). The quotient
// can pass the largest code where the scale is subnormal.
template <typename C> __device__ __forceinline__ float quotient8(float x, float scale) {
  return scale > 0.f ? fminf(fmaxf(x / scale, -kLargest8<C>), kLargest8<C>) : 0.f;
}

// Four quotients as codes, the first in the low byte.
template <typename C> __device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t codes4<e4m3_t>(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}
template <> __device__ __forceinline__ uint32_t codes4<i8_t>(float a, float b, float c, float d) {
  auto q = [](float x) { return static_cast<uint32_t>(static_cast<int>(rintf(x))) & 0xFFu; };
  return q(a) | q(b) << 8 | q(c) << 16 | q(d) << 24;
}

// Four codes as numbers.
template <typename C> __device__ __forceinline__ void values4(uint32_t w, float (&v)[4]);
template <> __device__ __forceinline__ void values4<e4m3_t>(uint32_t w, float (&v)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}
template <> __device__ __forceinline__ void values4<i8_t>(uint32_t w, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
}

// code * scale, rounded to fp32 before any rounding to 16 bits (the compiler
// would otherwise round an f16's product once, from its full width, and a
// bf16's twice).
__device__ __forceinline__ float product8(float code, float scale) {
  float x = code * scale;
  asm volatile("" : "+v"(x));
  return x;
}

}  // namespace tsa
