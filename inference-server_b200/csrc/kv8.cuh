// The 8-bit page cache: what its kernels (kv8_append.cu, kv8_decode.cu, kv8_prefill.cu) share.
//
// Pools [num_blocks, num_kv_heads, 16, head_dim] hold e4m3 numbers; a page and kv head has one scale for its keys and one for its values,
// 2^(byte - 127) ([num_blocks, num_kv_heads] bytes, the e8m0 format), with exponents from kScaleLow to kScaleHigh.  Powers of two cost
// an e4m3 number nothing (its relative precision does not depend on the scale) and make every step with a scale exact but the one
// rounding to e4m3: a page whose scale grows is rounded anew by a factor 2^-n, which changes only what becomes subnormal, and the
// attention kernels multiply scores and weights by scales without an error.  The range is bounded so that sums of weights, which carry
// a value scale, stay far inside fp32 (kv8_decode.cu).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

constexpr int kKvPage = 16;
constexpr int kScaleLow = -32, kScaleHigh = 31;

__device__ __forceinline__ int scale_exponent(int byte) { return min(max(byte - 127, kScaleLow), kScaleHigh); }
// 2^e for a normal result.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
// Smallest exponent e in range with top <= 448 * 2^e, from the bits of top >= 0: 448 = 1.75 * 2^8.
__device__ __forceinline__ int fit_exponent(uint32_t top) {
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleLow), kScaleHigh);
}
// Four e4m3 numbers as f16 (exact): bytes 0, 1 and bytes 2, 3.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// Two fp32 numbers to e4m3, to nearest; beyond +-448 to the largest, NaN to the NaN code.  `a` goes to the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Four of them, the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Two products in one instruction.
__device__ __forceinline__ float2 mul_pair(float a, float b, float by) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %4};\n\t"
      "mul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a), "f"(b), "f"(by));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 16 or 8 bytes of shared memory.
template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t* w) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

}  // namespace b200
