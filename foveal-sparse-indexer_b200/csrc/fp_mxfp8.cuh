// MXFP8 copies of activations: 32 consecutive elements (row-major order) share a power of two 2^k, the
// smallest with max|x| <= 448 * 2^k over the block's finite elements (k clamped to [-118, 120]); an element is
// e4m3, x * 2^-k rounded to nearest even, and NaN for a NaN or an infinity.
//
// The scale is a power of two because e4m3 is a floating-point format: scaling by 2^-k is exact, so the only
// rounding is the one to e4m3 (at most 2^-4 of the value, or 2^-10 of 2^k below the smallest normal), and a
// copy does not depend on how the scale was computed.  Choosing the smallest k that fits 448 * 2^k never
// clips the block's largest element (rounding its exponent down would clip mantissas above 1.75).  The upper
// and lower clamp keep 2^k, 2^-k and every dequantised value (a multiple of 2^(k-9)) normal in fp32 and exact
// in bf16.  The scale is stored as the byte k + 127.  Magnitudes of at least 248 * 2^120 would round to 2^128,
// past fp32's range: they are held as 240 * 2^120, so that a finite value stays finite.
#pragma once
#include "fp_internal.cuh"

namespace fp {

constexpr int kMxBlock = 32;
constexpr int kMxMin = -118, kMxMax = 120;
constexpr uint32_t kF32Inf = 0x7F800000u;
constexpr float kMxHuge = 0x1.fp127f;     // 248 * 2^120
constexpr float kMxLargest = 0x1.ep127f;  // 240 * 2^120

// Scale byte from the bits of the block's largest finite magnitude: 448 = 1.75 * 2^8, so k is the exponent
// minus 8, plus one when the mantissa exceeds 1.75; adding 0x1FFFFF carries into the exponent exactly then.
__device__ __forceinline__ int mx_scale_byte(uint32_t amax_bits) {
  const int b = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
  return min(max(b, kMxMin + 127), kMxMax + 127);
}
__device__ __forceinline__ float mx_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }            // 2^k
__device__ __forceinline__ float mx_inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }  // 2^-k

// Two e4m3 codes, lo in the low byte (NaN in: NaN code).
__device__ __forceinline__ uint16_t mx_pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// The values of two e4m3 codes (every e4m3 value is exact in fp16).
__device__ __forceinline__ float2 mx_unpack2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  float2 v;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}"
      : "=f"(v.x), "=f"(v.y)
      : "r"(h));
  return v;
}

template <typename T>
__device__ __forceinline__ T mx_from_f32(float v);
template <>
__device__ __forceinline__ float mx_from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 mx_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One block per warp, one element per lane.  Returns the lane's code; `byte` is the block's scale.
__device__ __forceinline__ uint8_t mx_quantize_lane(float v, int& byte) {
  const uint32_t bits = __float_as_uint(v) & 0x7FFFFFFFu;
  const bool finite = bits < kF32Inf;
  byte = mx_scale_byte(__reduce_max_sync(0xffffffffu, finite ? bits : 0u));
  if (fabsf(v) >= kMxHuge) v = copysignf(kMxLargest, v);
  const float s = finite ? v * mx_inv_scale(byte) : __uint_as_float(0x7FC00000u);
  return (uint8_t)(mx_pack2(s, 0.f) & 0xFF);
}
__device__ __forceinline__ float mx_value(uint8_t code, int byte) { return mx_unpack2(code).x * mx_scale(byte); }

}  // namespace fp
