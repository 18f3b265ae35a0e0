// MXFP8 copies of activations: 32 consecutive elements (row-major order) share a power of two 2^k, the
// smallest with max|x| <= 448 * 2^k over the block's finite elements (k clamped to [-118, 120]); an element is
// e4m3, x * 2^-k rounded to nearest even, and NaN for a NaN or an infinity.
//
// The scale is a power of two because e4m3 is a floating-point format: scaling by 2^-k is exact, so the only
// rounding is the one to e4m3 (at most 2^-4 of the value, or 2^-10 of 2^k below the smallest normal), and a
// copy does not depend on how the scale was computed.  Choosing the smallest k that fits 448 * 2^k never
// clips the block's largest element (rounding its exponent down would clip mantissas above 1.75).  The upper
// and lower clamp keep 2^k and 2^-k normal in fp32 and every dequantised value, a multiple of 2^(k-9), exact in
// fp32 and bf16.  At k = -118 those are subnormal down to 2^-127: the kernels need a build that does not flush
// subnormals to zero.  The scale is stored as the byte k + 127.  Magnitudes of at least 248 * 2^120 would round
// to 2^128, past fp32's range: they are held as 240 * 2^120, so that a finite value stays finite.
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

// For blocks that hold a NaN, an infinity or a magnitude near 2^128 (rare): makes v what its code shall stand
// for, and returns the bits of its magnitude for the block's maximum, 0 where it is not finite.
__device__ __forceinline__ uint32_t mx_finite(float& v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  if (b >= kF32Inf) {
    v = __uint_as_float(0x7FC00000u);
    return 0;
  }
  if (b >= __float_as_uint(kMxHuge)) v = copysignf(kMxLargest, v);
  return b;
}

template <typename T>
__device__ __forceinline__ T mx_from_f32(float v);
template <>
__device__ __forceinline__ float mx_from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 mx_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of a tensor: kV elements in a thread, kGroup neighbouring lanes to a block of 32.
template <typename T>
struct MxVec {
  static constexpr int kV = 16 / (int)sizeof(T);
  static constexpr int kGroup = kMxBlock / kV;

  // elements [i, i + kV) of the n, zeros past the end
  static __device__ __forceinline__ uint4 load(const T* __restrict__ p, int64_t i, int64_t n) {
    if (i + kV <= n) return __ldg(reinterpret_cast<const uint4*>(p + i));
    T t[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) t[e] = i + e < n ? p[i + e] : T(0.f);
    return *reinterpret_cast<const uint4*>(t);
  }
  static __device__ __forceinline__ void store(T* __restrict__ p, int64_t i, int64_t n, const float (&v)[kV]) {
    if (i + kV <= n) {
      uint4 w;
      if constexpr (kV == 4) {
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      } else {
        uint32_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
          r[e] = *reinterpret_cast<const uint32_t*>(&b);
        }
        w = make_uint4(r[0], r[1], r[2], r[3]);
      }
      *reinterpret_cast<uint4*>(p + i) = w;
    } else {
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (i + e < n) p[i + e] = mx_from_f32<T>(v[e]);
    }
  }
  static __device__ __forceinline__ void unpack(const uint4& w, float (&v)[kV]) {
    const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kV == 4) {
        v[e] = __uint_as_float(r[e]);
      } else {
        v[2 * e] = __uint_as_float(r[e] << 16);
        v[2 * e + 1] = __uint_as_float(r[e] & 0xFFFF0000u);
      }
    }
  }
  // fp32 bits of the largest magnitude (a NaN or an infinity wins)
  static __device__ __forceinline__ uint32_t amax_bits(const uint4& w) {
    if constexpr (kV == 4) {
      constexpr uint32_t m = 0x7FFFFFFFu;
      return max(max(w.x & m, w.y & m), max(w.z & m, w.w & m));
    } else {
      constexpr uint32_t m = 0x7FFF7FFFu;
      const uint32_t a = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
      return max(a & 0xFFFF0000u, a << 16);
    }
  }
  static __device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int o = 1; o < kGroup; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }

  // codes of elements [i, i + kV) and, by the group's first lane, the block's scale byte.  All lanes of the
  // warp call this together; vectors past the end are zeros and write nothing.
  static __device__ __forceinline__ void quantize(const uint4& w, int64_t i, int64_t n, uint8_t* __restrict__ codes,
                                                  uint8_t* __restrict__ scales) {
    float v[kV];
    unpack(w, v);
    uint32_t top = group_max(amax_bits(w));
    if (__any_sync(0xffffffffu, top >= __float_as_uint(kMxHuge))) {  // rare: NaN, infinity or a value near 2^128
      uint32_t fin = 0;
#pragma unroll
      for (int e = 0; e < kV; ++e) fin = max(fin, mx_finite(v[e]));
      top = group_max(fin);
    }
    const int byte = mx_scale_byte(top);
    const float inv = mx_inv_scale(byte);
    uint32_t c[kV / 4];
#pragma unroll
    for (int e = 0; e < kV / 4; ++e)
      c[e] = (uint32_t)mx_pack2(v[4 * e] * inv, v[4 * e + 1] * inv) |
             ((uint32_t)mx_pack2(v[4 * e + 2] * inv, v[4 * e + 3] * inv) << 16);
    if (i + kV <= n) {
      if constexpr (kV == 4) *reinterpret_cast<uint32_t*>(codes + i) = c[0];
      else *reinterpret_cast<uint2*>(codes + i) = make_uint2(c[0], c[1]);
    } else {
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (i + e < n) codes[i + e] = (uint8_t)(c[e / 4] >> (8 * (e & 3)));
    }
    if (i < n && (i & (kMxBlock - 1)) == 0) scales[i / kMxBlock] = (uint8_t)byte;
  }

  struct Codes {
    uint32_t c[kV / 4];
    uint32_t byte;
  };
  static __device__ __forceinline__ Codes load_codes(const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, int64_t i, int64_t n) {
    Codes r;
    if (i + kV <= n) {
      if constexpr (kV == 4) {
        r.c[0] = __ldg(reinterpret_cast<const uint32_t*>(codes + i));
      } else {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(codes + i));
        r.c[0] = w.x;
        r.c[1] = w.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kV / 4; ++e) r.c[e] = 0;
#pragma unroll
      for (int e = 0; e < kV; ++e)
        if (i + e < n) r.c[e / 4] |= (uint32_t)codes[i + e] << (8 * (e & 3));
    }
    r.byte = i < n ? __ldg(scales + i / kMxBlock) : 127u;
    return r;
  }
  static __device__ __forceinline__ void values(const Codes& q, float (&v)[kV]) {
    const float s = mx_scale((int)q.byte);
#pragma unroll
    for (int e = 0; e < kV / 2; ++e) {
      const float2 f = mx_unpack2((uint16_t)(q.c[e / 2] >> (16 * (e & 1))));
      v[2 * e] = f.x * s;
      v[2 * e + 1] = f.y * s;
    }
  }
};

}  // namespace fp
