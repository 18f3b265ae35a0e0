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

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
mxfp8_quantize_kernel(const T* __restrict__ x, int64_t n, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 31;
  const int64_t nb = (n + kMxBlock - 1) / kMxBlock;
  for (int64_t b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); b < nb; b += (int64_t)gridDim.x * kWarps) {
    const int64_t i = b * kMxBlock + lane;
    int byte;
    const uint8_t c = mx_quantize_lane(i < n ? to_f32(x[i]) : 0.f, byte);
    if (i < n) codes[i] = c;
    if (lane == 0) scales[b] = (uint8_t)byte;
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
mxfp8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n,
                        T* __restrict__ y) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    y[i] = mx_from_f32<T>(mx_value(codes[i], scales[i / kMxBlock]));
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
swiglu_fwd_mxfp8_kernel(const T* __restrict__ g, const T* __restrict__ u, int64_t n, T* __restrict__ h,
                        uint8_t* __restrict__ gc, uint8_t* __restrict__ gs, uint8_t* __restrict__ uc,
                        uint8_t* __restrict__ us) {
  const int lane = threadIdx.x & 31;
  const int64_t nb = (n + kMxBlock - 1) / kMxBlock;
  for (int64_t b = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); b < nb; b += (int64_t)gridDim.x * kWarps) {
    const int64_t i = b * kMxBlock + lane;
    const float gv = i < n ? to_f32(g[i]) : 0.f, uv = i < n ? to_f32(u[i]) : 0.f;
    int gb, ub;
    const uint8_t cg = mx_quantize_lane(gv, gb), cu = mx_quantize_lane(uv, ub);
    if (i < n) {
      h[i] = mx_from_f32<T>(gv / (1.0f + expf(-gv)) * uv);
      gc[i] = cg;
      uc[i] = cu;
    }
    if (lane == 0) {
      gs[b] = (uint8_t)gb;
      us[b] = (uint8_t)ub;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
swiglu_bwd_mxfp8_kernel(const T* __restrict__ dout, const uint8_t* __restrict__ gc, const uint8_t* __restrict__ gs,
                        const uint8_t* __restrict__ uc, const uint8_t* __restrict__ us, int64_t n,
                        T* __restrict__ dg, T* __restrict__ du, T* __restrict__ h) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const float d = to_f32(dout[i]);
    const float gv = mx_value(gc[i], gs[i / kMxBlock]), uv = mx_value(uc[i], us[i / kMxBlock]);
    const float sig = 1.0f / (1.0f + expf(-gv));
    const float silu = gv * sig;
    du[i] = mx_from_f32<T>(d * silu);
    dg[i] = mx_from_f32<T>(d * uv * (sig * (1.0f + gv * (1.0f - sig))));
    if (h) h[i] = mx_from_f32<T>(silu * uv);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int grid_for(int64_t units, int64_t per_block, int sms) {
  const int64_t want = (units + per_block - 1) / per_block;
  return (int)(want < (int64_t)sms * 16 ? want : (int64_t)sms * 16);
}

int launched() { return cudaGetLastError() == cudaSuccess ? FP_OK : FP_ERR_CUDA; }

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
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = grid_for(n, kWarps * 32, sms);
  if (dtype == FP_DTYPE_BF16)
    mxfp8_quantize_kernel<<<grid, kWarps * 32, 0, st>>>((const __nv_bfloat16*)x, n, (uint8_t*)codes, (uint8_t*)scales);
  else
    mxfp8_quantize_kernel<<<grid, kWarps * 32, 0, st>>>((const float*)x, n, (uint8_t*)codes, (uint8_t*)scales);
  return launched();
}

int fp_mxfp8_dequantize(const void* codes, const void* scales, int dtype, int64_t n, void* y, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!y || !codes || !scales || !al16(y) || !al16(codes)) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = grid_for(n, kWarps * 32, sms);
  if (dtype == FP_DTYPE_BF16)
    mxfp8_dequantize_kernel<<<grid, kWarps * 32, 0, st>>>((const uint8_t*)codes, (const uint8_t*)scales, n,
                                                         (__nv_bfloat16*)y);
  else
    mxfp8_dequantize_kernel<<<grid, kWarps * 32, 0, st>>>((const uint8_t*)codes, (const uint8_t*)scales, n, (float*)y);
  return launched();
}

int fp_swiglu_fwd_mxfp8(const void* g, const void* u, int dtype, int64_t n, void* h, void* g_codes, void* g_scales,
                        void* u_codes, void* u_scales, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!g || !u || !h || !g_codes || !g_scales || !u_codes || !u_scales) return FP_ERR_INVALID_ARG;
  if (!al16(g) || !al16(u) || !al16(h) || !al16(g_codes) || !al16(u_codes)) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = grid_for(n, kWarps * 32, sms);
  if (dtype == FP_DTYPE_BF16)
    swiglu_fwd_mxfp8_kernel<<<grid, kWarps * 32, 0, st>>>(
        (const __nv_bfloat16*)g, (const __nv_bfloat16*)u, n, (__nv_bfloat16*)h, (uint8_t*)g_codes, (uint8_t*)g_scales,
        (uint8_t*)u_codes, (uint8_t*)u_scales);
  else
    swiglu_fwd_mxfp8_kernel<<<grid, kWarps * 32, 0, st>>>((const float*)g, (const float*)u, n, (float*)h,
                                                         (uint8_t*)g_codes, (uint8_t*)g_scales, (uint8_t*)u_codes,
                                                         (uint8_t*)u_scales);
  return launched();
}

int fp_swiglu_bwd_mxfp8(const void* dout, const void* g_codes, const void* g_scales, const void* u_codes,
                        const void* u_scales, int dtype, int64_t n, void* dg, void* du, void* h, void* stream) {
  if (n < 0) return FP_ERR_INVALID_ARG;
  if (!known(dtype)) return FP_ERR_UNSUPPORTED;
  if (n == 0) return FP_OK;
  if (!dout || !dg || !du || !g_codes || !g_scales || !u_codes || !u_scales) return FP_ERR_INVALID_ARG;
  if (!al16(dout) || !al16(dg) || !al16(du) || !al16(h) || !al16(g_codes) || !al16(u_codes)) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = grid_for(n, kWarps * 32, sms);
  if (dtype == FP_DTYPE_BF16)
    swiglu_bwd_mxfp8_kernel<<<grid, kWarps * 32, 0, st>>>(
        (const __nv_bfloat16*)dout, (const uint8_t*)g_codes, (const uint8_t*)g_scales, (const uint8_t*)u_codes,
        (const uint8_t*)u_scales, n, (__nv_bfloat16*)dg, (__nv_bfloat16*)du, (__nv_bfloat16*)h);
  else
    swiglu_bwd_mxfp8_kernel<<<grid, kWarps * 32, 0, st>>>(
        (const float*)dout, (const uint8_t*)g_codes, (const uint8_t*)g_scales, (const uint8_t*)u_codes,
        (const uint8_t*)u_scales, n, (float*)dg, (float*)du, (float*)h);
  return launched();
}

}  // extern "C"
