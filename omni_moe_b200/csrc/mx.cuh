// MX blocks: 32 neighbouring values of a row share one power-of-two scale 2^s (stored as the byte s + 127, e8m0), each
// value is held as e4m3.
//   s     the smallest exponent >= -127 for which the largest finite magnitude of the block is <= 448 * 2^s
//   code  e4m3 of v * 2^-s, to nearest, ties to even (exact scaling: the only rounding is that of the 3 mantissa bits,
//         at most 2^-4 of the value); a value that is not finite becomes NaN and does not count for the scale
// A decoded value needs 4 significant bits, so it is exact in bf16, fp32 and fp16 wherever their ranges hold it.
#pragma once

#include "common.cuh"

namespace omni {
namespace mx {

constexpr int kBlock = 32;

// |v| if finite, else 0: what the block maximum is taken over.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}

// s for a block maximum: 448 = 1.75 * 2^8, so for top = m * 2^e with m in [1, 2) it is e - 8, one more if m > 1.75.
__device__ __forceinline__ int exponent_of(float top) {
  const uint32_t u = __float_as_uint(top);
  const int s = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return s < -127 ? -127 : s;  // zero and subnormal maxima end here too
}
__device__ __forceinline__ float pow2(int s) {  // 2^s, -127 <= s <= 127
  return s == -127 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(s + 127) << 23);
}
// The scale that byte b stands for: 2^(b - 127), and NaN for 255, which no block of ours holds but others may.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7fffffffu : b << 23); }

// Codes of two values (the first in the low byte); inv = 2^-s.  v - v is 0 for a finite v and NaN otherwise.
__device__ __forceinline__ uint32_t encode2(float v0, float v1, float inv) {
  const float a = __fmaf_rn(v0, inv, v0 - v0), b = __fmaf_rn(v1, inv, v1 - v1);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t encode4(float v0, float v1, float v2, float v3, float inv) {
  return encode2(v0, v1, inv) | (encode2(v2, v3, inv) << 16);
}

// The same where no value is infinite: NaN converts to the NaN code by itself.
__device__ __forceinline__ uint32_t encode_finite4(float v0, float v1, float v2, float v3, float inv) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v1 * inv), "f"(v0 * inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v3 * inv), "f"(v2 * inv));
  return lo | (static_cast<uint32_t>(hi) << 16);
}

// The two e4m3 values in the low 16 bits of r.
__device__ __forceinline__ float2 decode2(uint32_t r) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(r)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

}  // namespace mx
}  // namespace omni
