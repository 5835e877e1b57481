// The 8-bit KV cache: e4m3 codes [.., C, D] and one fp32 scale per (row, KV head, block of
// `block` slots); code * scale is the value. Shared by the append (cache_q8.cu) and the
// attention (attention_q8.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace fb {
namespace q8 {

constexpr float kE4M3Max = 448.f;
// Scale of a block whose slots are all zero: small enough that any later token's scale replaces
// it, large enough that 1 / scale and code * scale stay normal fp32 numbers.
constexpr float kLeastScale = 7.888609052210118e-31f;  // 2^-100

// The least power of two s with largest <= 448 s. 448 = 0.875 * 2^9, so with largest = f * 2^x,
// f in [0.5, 1), s = 2^(x - 9) for f <= 0.875, else 2^(x - 8). Powers of two make the rescaling of
// a block exact (down to e4m3's subnormals), and cost no precision: the codes are floating point.
__device__ __forceinline__ float least_scale(float largest) {
  int x;
  const float f = frexpf(largest, &x);
  const float s = ldexpf(1.f, f <= 0.875f ? x - 9 : x - 8);
  return largest > kE4M3Max * kLeastScale ? s : kLeastScale;
}

// Two values to packed e4m3 codes, round to nearest even, lo in the low byte. Anything that is
// not finite becomes the NaN code.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  const float nan = __int_as_float(0x7fffffff);
  lo = fabsf(lo) < INFINITY ? lo : nan;
  hi = fabsf(hi) < INFINITY ? hi : nan;
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Two packed e4m3 codes (low 16 bits) to f16x2: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t h;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(h) : "r"(codes));
  return h;
}

// Four packed codes to two f16x2.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}

__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t codes) {
  const uint32_t h = e4m3x2_to_f16x2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; "
      "fma.rn.f32x2 z, x, y, z; mov.b64 {%0, %1}, z; }"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
constexpr bool valid_block(int block) { return block == 16 || block == 32 || block == 64; }

}  // namespace q8
}  // namespace fb
