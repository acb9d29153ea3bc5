// The 8-bit form of cached rows: an e4m3 code per element and, per row and head, one power of two 2^(byte - 127) -- the least that takes the head's largest
// finite element to 448 or below.  A power of two costs a float format no precision (only the lowest codes' range), its product with a code is exact, and
// it is a byte: 1 / dim of the codes.  Infinities and NaN become the NaN code and do not change the row's power.
// Codes: [pages, page, heads * size]; bytes: [pages, heads, page], so that a tile of one head's keys finds its powers side by side.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace cache8 {

// the byte for a head whose largest finite magnitude has these bits: 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t power_of(uint32_t abs_bits) {
  const int e = static_cast<int>(abs_bits >> 23) - 127 - 8 + ((abs_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, -127) + 127);
}
__device__ __forceinline__ float value_of_power(uint32_t byte) { return __uint_as_float(byte != 0 ? byte << 23 : 0x00400000u); }       // 2^(byte - 127)
__device__ __forceinline__ float inverse_of_power(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }                       // 2^(127 - byte), byte <= 247
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// two codes, a in the low byte: to the nearest, ties to even; NaN is kept, infinities are not for this (they would become 448)
__device__ __forceinline__ uint32_t codes_of(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// two codes -> two halves (exact), the low byte's in the low half
__device__ __forceinline__ uint32_t halves_of(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}

}  // namespace cache8
