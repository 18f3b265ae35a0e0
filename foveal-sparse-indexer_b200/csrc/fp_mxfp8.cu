// 8-bit activation copies (format: fp_mxfp8.cuh) and the SwiGLU whose backward pass reads them.
//
//   h  = silu(g) u                                   from g and u themselves
//   du = dh silu(g^),  dg = dh u^ s (1 + g^ (1 - s)),  s = sigmoid(g^)      from their copies g^, u^
//
// The forward therefore leaves 2 * (1 + 1/32) bytes per element pair for the backward pass where keeping g
// and u takes 4 (bf16) or 8 (fp32).
#include "fp_mxfp8.cuh"

namespace fp {
namespace {

// All four kernels stream: a thread takes a few vectors of 16 bytes, a CTA's width apart, and issues all of their
// loads before the first use.  HBM bound, but for the SwiGLU forward, which the exact division and exponential
// of fp_swiglu_fwd (whose bits it keeps) hold at 0.92 of a copy's rate: with the hardware's approximations it
// took 278 us where it takes 318 (16384 x 14336 bf16).  Vectors to a thread, measured there (GB/s moved; torch's
// copy 6500): copy 4 / 8: 6470 / 6810 (fp32, 16384 x 4096: 47 / 52 us); restore 2 / 4: 6680 / 6310; forward
// 1 / 2 / 4: 5470 / 5960 / 5020; backward 1 / 2 / 4: 5970 / 5650 / 4800 (fp32, 16384 x 1536: 71 / 65 us for 1 / 2).
// 256 threads; 512 lost 5 to 15 %, 128 gained nothing sure.
constexpr int kThreads = 256;
template <typename T>
constexpr int kUnrollCopy = sizeof(T) == 2 ? 8 : 4;
template <typename T>
constexpr int kUnrollBwd = sizeof(T) == 2 ? 1 : 2;
constexpr int kUnrollRestore = 2, kUnrollFwd = 2;

template <typename T, int U>
__device__ __forceinline__ int64_t first_element() {
  return ((int64_t)blockIdx.x * (kThreads * U) + threadIdx.x) * MxVec<T>::kV;
}
template <typename T>
constexpr int kStep = kThreads * MxVec<T>::kV;

template <typename T>
__global__ void __launch_bounds__(kThreads)
mxfp8_quantize_kernel(const T* __restrict__ x, int64_t n, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  using V = MxVec<T>;
  const int64_t i = first_element<T, kUnrollCopy<T>>();
  uint4 w[kUnrollCopy<T>];
#pragma unroll
  for (int k = 0; k < kUnrollCopy<T>; ++k) w[k] = V::load(x, i + k * kStep<T>, n);
#pragma unroll
  for (int k = 0; k < kUnrollCopy<T>; ++k) V::quantize(w[k], i + k * kStep<T>, n, codes, scales);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
mxfp8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n,
                        T* __restrict__ y) {
  using V = MxVec<T>;
  const int64_t i = first_element<T, kUnrollRestore>();
  typename V::Codes q[kUnrollRestore];
#pragma unroll
  for (int k = 0; k < kUnrollRestore; ++k) q[k] = V::load_codes(codes, scales, i + k * kStep<T>, n);
#pragma unroll
  for (int k = 0; k < kUnrollRestore; ++k) {
    float v[V::kV];
    V::values(q[k], v);
    V::store(y, i + k * kStep<T>, n, v);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu_fwd_mxfp8_kernel(const T* __restrict__ g, const T* __restrict__ u, int64_t n, T* __restrict__ h,
                        uint8_t* __restrict__ gc, uint8_t* __restrict__ gs, uint8_t* __restrict__ uc,
                        uint8_t* __restrict__ us) {
  using V = MxVec<T>;
  const int64_t i0 = first_element<T, kUnrollFwd>();
  uint4 gw[kUnrollFwd], uw[kUnrollFwd];
#pragma unroll
  for (int k = 0; k < kUnrollFwd; ++k) {
    gw[k] = V::load(g, i0 + k * kStep<T>, n);
    uw[k] = V::load(u, i0 + k * kStep<T>, n);
  }
#pragma unroll
  for (int k = 0; k < kUnrollFwd; ++k) {
    const int64_t i = i0 + k * kStep<T>;
    V::quantize(gw[k], i, n, gc, gs);
    V::quantize(uw[k], i, n, uc, us);
    float gv[V::kV], uv[V::kV];
    V::unpack(gw[k], gv);
    V::unpack(uw[k], uv);
#pragma unroll
    for (int e = 0; e < V::kV; ++e) gv[e] = gv[e] / (1.0f + expf(-gv[e])) * uv[e];  // as fp_swiglu_fwd
    V::store(h, i, n, gv);
  }
}

// sigmoid(g).  For bf16 gradients the hardware exponential and reciprocal do: the exponential is off by up to
// 2 + 1.2 |g| steps of 2^-23 (2^-16 of the value at |g| = 80, and only where g is negative does it reach the
// sigmoid whole), far below the gradients' own rounding (2^-9 to 2^-8), and the exact forms made the backward
// kernel issue bound (446 us, 340 without them, 16384 x 14336).
template <typename T>
__device__ __forceinline__ float sigmoid_for(float g) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-g)));
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu_bwd_mxfp8_kernel(const T* __restrict__ dout, const uint8_t* __restrict__ gc, const uint8_t* __restrict__ gs,
                        const uint8_t* __restrict__ uc, const uint8_t* __restrict__ us, int64_t n,
                        T* __restrict__ dg, T* __restrict__ du, T* __restrict__ h) {
  using V = MxVec<T>;
  const int64_t i0 = first_element<T, kUnrollBwd<T>>();
  uint4 dw[kUnrollBwd<T>];
  typename V::Codes gq[kUnrollBwd<T>], uq[kUnrollBwd<T>];
#pragma unroll
  for (int k = 0; k < kUnrollBwd<T>; ++k) {
    dw[k] = V::load(dout, i0 + k * kStep<T>, n);
    gq[k] = V::load_codes(gc, gs, i0 + k * kStep<T>, n);
    uq[k] = V::load_codes(uc, us, i0 + k * kStep<T>, n);
  }
#pragma unroll
  for (int k = 0; k < kUnrollBwd<T>; ++k) {
    const int64_t i = i0 + k * kStep<T>;
    float d[V::kV], gv[V::kV], uv[V::kV];
    V::unpack(dw[k], d);
    V::values(gq[k], gv);
    V::values(uq[k], uv);
    float a[V::kV], b[V::kV], c[V::kV];
#pragma unroll
    for (int e = 0; e < V::kV; ++e) {
      const float sig = sigmoid_for<T>(gv[e]);
      const float silu = gv[e] * sig;
      a[e] = d[e] * uv[e] * (sig * (1.0f + gv[e] * (1.0f - sig)));
      b[e] = d[e] * silu;
      c[e] = silu * uv[e];
    }
    V::store(dg, i, n, a);
    V::store(du, i, n, b);
    if (h) V::store(h, i, n, c);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// CTAs of kThreads * unroll vectors for n elements; 0 when the grid would pass its limit.
template <typename T>
unsigned grid_for(int64_t n, int unroll) {
  const int64_t per = (int64_t)kStep<T> * unroll, want = (n + per - 1) / per;
  return want <= INT32_MAX ? (unsigned)want : 0u;
}

int launched() { return cudaGetLastError() == cudaSuccess ? FP_OK : FP_ERR_CUDA; }

// f(T{}) with the element type of `dtype`, once the current device is known to run these kernels.
template <typename F>
int by_type(int dtype, F f) {
  int sms;
  if (const int rc = device_info(sms)) return rc;
  return dtype == FP_DTYPE_BF16 ? f(__nv_bfloat16{}) : f(float{});
}

bool known(int dtype) { return dtype == FP_DTYPE_F32 || dtype == FP_DTYPE_BF16; }

}  // namespace
}  // namespace fp

using namespace fp;

extern "C" {

int fp_mxfp8_quantize(const void* x, int dtype, int64_t n, void* codes, void* scales, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!x || !codes || !scales || !al16(x) || !al16(codes)) return FP_ERR_INVALID_ARG;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned grid = grid_for<T>(n, kUnrollCopy<T>);
    if (!grid) return FP_ERR_UNSUPPORTED;
    mxfp8_quantize_kernel<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const T*)x, n, (uint8_t*)codes,
                                                                         (uint8_t*)scales);
    return launched();
  });
}

int fp_mxfp8_dequantize(const void* codes, const void* scales, int dtype, int64_t n, void* y, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!y || !codes || !scales || !al16(y) || !al16(codes)) return FP_ERR_INVALID_ARG;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned grid = grid_for<T>(n, kUnrollRestore);
    if (!grid) return FP_ERR_UNSUPPORTED;
    mxfp8_dequantize_kernel<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const uint8_t*)codes,
                                                                           (const uint8_t*)scales, n, (T*)y);
    return launched();
  });
}

int fp_swiglu_fwd_mxfp8(const void* g, const void* u, int dtype, int64_t n, void* h, void* g_codes, void* g_scales,
                        void* u_codes, void* u_scales, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!g || !u || !h || !g_codes || !g_scales || !u_codes || !u_scales) return FP_ERR_INVALID_ARG;
  if (!al16(g) || !al16(u) || !al16(h) || !al16(g_codes) || !al16(u_codes)) return FP_ERR_INVALID_ARG;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned grid = grid_for<T>(n, kUnrollFwd);
    if (!grid) return FP_ERR_UNSUPPORTED;
    swiglu_fwd_mxfp8_kernel<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>(
        (const T*)g, (const T*)u, n, (T*)h, (uint8_t*)g_codes, (uint8_t*)g_scales, (uint8_t*)u_codes,
        (uint8_t*)u_scales);
    return launched();
  });
}

int fp_swiglu_bwd_mxfp8(const void* dout, const void* g_codes, const void* g_scales, const void* u_codes,
                        const void* u_scales, int dtype, int64_t n, void* dg, void* du, void* h, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!dout || !dg || !du || !g_codes || !g_scales || !u_codes || !u_scales) return FP_ERR_INVALID_ARG;
  if (!al16(dout) || !al16(dg) || !al16(du) || !al16(h) || !al16(g_codes) || !al16(u_codes)) return FP_ERR_INVALID_ARG;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned grid = grid_for<T>(n, kUnrollBwd<T>);
    if (!grid) return FP_ERR_UNSUPPORTED;
    swiglu_bwd_mxfp8_kernel<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>(
        (const T*)dout, (const uint8_t*)g_codes, (const uint8_t*)g_scales, (const uint8_t*)u_codes,
        (const uint8_t*)u_scales, n, (T*)dg, (T*)du, (T*)h);
    return launched();
  });
}

}  // extern "C"
