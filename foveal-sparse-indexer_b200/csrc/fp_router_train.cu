// Training of the 16-D router: the gradient of its scores, and the load-balance loss over the routed blocks.
//
// Scores (forward in fp_router.cu):  q = x Wq^T,  r = (mean(q^2) + eps)^-1/2,  n = r q,  S = n K^T / 4.
// Gradient from dS:
//   a = dS K / 4            dK = dS^T n / 4
//   dq = r (a - n mean(a n))
//   dWq = dq^T x            dx = dq Wq
//
// Balance loss over the R = NB - base remote blocks, n counted rows:
//   p_t = softmax(S_t[base:] / T),  f_e = c_e / sum c  with c_e the routed slots of block e,
//   L = R sum_e f_e (1/n) sum_t p_te,    dL/dS_te = R / (T n) p_te (f_e - sum_j f_j p_tj).
// A constant added to f cancels in the gradient, so it is computed from f_e - 1/R (exact integer numerators):
// near balance f_e and its mean agree in most of their bits and their difference would be rounding error.
#include "fp_mxfp8.cuh"

#include <algorithm>

namespace fp {
namespace {

constexpr int kIdx = 16;  // the router's width

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int launched() { return cudaGetLastError() == cudaSuccess ? FP_OK : FP_ERR_CUDA; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ------------------------------------------------------------------ gradient of the scores
// dq, one warp per token.
template <typename T>
__global__ void __launch_bounds__(256)
router_dq_kernel(const float* __restrict__ ds, const T* __restrict__ k16, const float* __restrict__ q16,
                 const float* __restrict__ rnorm, int64_t M, int NB, float* __restrict__ dq) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < M; t += (int64_t)gridDim.x * 8) {
    float a[kIdx] = {};
    for (int b = lane; b < NB; b += 32) {
      const float s = ds[t * NB + b];
#pragma unroll
      for (int j = 0; j < kIdx; ++j) a[j] = fmaf(s, to_f32(k16[b * kIdx + j]), a[j]);
    }
    float dot = 0.f, n[kIdx];
#pragma unroll
    for (int j = 0; j < kIdx; ++j) {
      a[j] = warp_sum(a[j]) * 0.25f;
      n[j] = q16[t * kIdx + j];
      dot = fmaf(a[j], n[j], dot);
    }
    dot *= 1.0f / kIdx;
    const float r = rnorm[t];
#pragma unroll
    for (int j = 0; j < kIdx; ++j)
      if (lane == j) dq[t * kIdx + j] = r * (a[j] - n[j] * dot);
  }
}

// Partial sums over the token range of blockIdx.y: dK, one thread per element.
__global__ void __launch_bounds__(256)
router_dk_kernel(const float* __restrict__ ds, const float* __restrict__ q16, int64_t M, int NB, int64_t chunk,
                 float* __restrict__ part) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= NB * kIdx) return;
  const int b = i / kIdx, j = i % kIdx;
  const int64_t t0 = blockIdx.y * chunk, t1 = min(t0 + chunk, M);
  float s = 0.f;
  for (int64_t t = t0; t < t1; ++t) s = fmaf(ds[t * NB + b], q16[t * kIdx + j], s);
  part[(int64_t)blockIdx.y * NB * kIdx + i] = s * 0.25f;
}

// dWq over the token range of blockIdx.y, one thread per column; x from its 8-bit copy when codes are given.
template <typename T>
__global__ void __launch_bounds__(256)
router_dw_kernel(const T* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                 const float* __restrict__ dq, int64_t M, int D, int64_t chunk, float* __restrict__ part) {
  const int d = blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= D) return;
  const int64_t t0 = blockIdx.y * chunk, t1 = min(t0 + chunk, M);
  float acc[kIdx] = {};
  for (int64_t t = t0; t < t1; ++t) {
    const int64_t i = t * D + d;
    const float v = codes ? mx_value(codes[i], scales[i / kMxBlock]) : to_f32(x[i]);
#pragma unroll
    for (int j = 0; j < kIdx; ++j) acc[j] = fmaf(dq[t * kIdx + j], v, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < kIdx; ++j) part[((int64_t)blockIdx.y * kIdx + j) * D + d] = acc[j];
}

template <typename T>
__global__ void __launch_bounds__(256)
router_dx_kernel(const float* __restrict__ dq, const T* __restrict__ wq, int64_t M, int D, T* __restrict__ dx) {
  const int64_t n = M * D;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / D;
    const int d = (int)(i - t * D);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kIdx; ++j) s = fmaf(dq[t * kIdx + j], to_f32(wq[(int64_t)j * D + d]), s);
    dx[i] = mx_from_f32<T>(s);
  }
}

// out[i] = sum over the partials in their order.
template <typename T>
__global__ void __launch_bounds__(256)
sum_partials_kernel(const float* __restrict__ part, int parts, int64_t n, T* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += part[p * n + i];
  out[i] = mx_from_f32<T>(s);
}

struct BwdPlan {
  int64_t chunk;  // tokens per partial sum
  int parts;
  size_t dq, dw, dk, total;
};
BwdPlan bwd_plan(int64_t M, int D, int NB) {
  BwdPlan p{};
  p.chunk = std::max<int64_t>(64, (M + 31) / 32);
  p.parts = (int)((M + p.chunk - 1) / p.chunk);
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  p.dq = 0;
  p.dw = p.dq + up((size_t)M * kIdx * 4);
  p.dk = p.dw + up((size_t)p.parts * kIdx * D * 4);
  p.total = p.dk + up((size_t)p.parts * kIdx * NB * 4);
  return p;
}

template <typename T>
int router_bwd(const float* ds, const T* x, const uint8_t* codes, const uint8_t* scales, const T* wq, const T* k16,
               const float* q16, const float* rnorm, int64_t M, int D, int NB, T* dx, void* dwq, void* dk16,
               int grad_dtype, char* ws, int sms, cudaStream_t st) {
  const BwdPlan p = bwd_plan(M, D, NB);
  float* dq = reinterpret_cast<float*>(ws + p.dq);
  float* pw = reinterpret_cast<float*>(ws + p.dw);
  float* pk = reinterpret_cast<float*>(ws + p.dk);
  if (dx || dwq)
    router_dq_kernel<T><<<(int)std::min<int64_t>((M + 7) / 8, sms * 8), 256, 0, st>>>(ds, k16, q16, rnorm, M, NB, dq);
  if (dk16) {
    const int n = NB * kIdx;
    router_dk_kernel<<<dim3((n + 255) / 256, p.parts), 256, 0, st>>>(ds, q16, M, NB, p.chunk, pk);
    if (grad_dtype == FP_DTYPE_BF16)
      sum_partials_kernel<<<(n + 255) / 256, 256, 0, st>>>(pk, p.parts, n, (__nv_bfloat16*)dk16);
    else
      sum_partials_kernel<<<(n + 255) / 256, 256, 0, st>>>(pk, p.parts, n, (float*)dk16);
  }
  if (dwq) {
    const int64_t n = (int64_t)kIdx * D;
    router_dw_kernel<T><<<dim3((D + 255) / 256, p.parts), 256, 0, st>>>(x, codes, scales, dq, M, D, p.chunk, pw);
    if (grad_dtype == FP_DTYPE_BF16)
      sum_partials_kernel<<<(int)((n + 255) / 256), 256, 0, st>>>(pw, p.parts, n, (__nv_bfloat16*)dwq);
    else
      sum_partials_kernel<<<(int)((n + 255) / 256), 256, 0, st>>>(pw, p.parts, n, (float*)dwq);
  }
  if (dx)
    router_dx_kernel<T><<<(int)std::min<int64_t>((M * D + 255) / 256, sms * 16), 256, 0, st>>>(dq, wq, M, D, dx);
  return launched();
}

// ------------------------------------------------------------------ balance loss
constexpr int kBalWarps = 8;
constexpr int kBalMaxCtas = 296;

// One row's remote scores in a warp's registers, divided by T; returns whether the row is counted, and turns
// the scores into probabilities.  A row whose remote scores are all -inf has no distribution and is not
// counted; a NaN makes the whole row NaN.
template <int E>
__device__ __forceinline__ bool balance_row(const float* __restrict__ row, int NB, int base, float temperature,
                                            int lane, float (&p)[E]) {
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int b = lane + 32 * i;
    float z = -INFINITY;
    if (b >= base && b < NB) {
      z = row[b];
      if (temperature != 1.0f) z = __fdiv_rn(z, temperature);
    }
    nan |= z != z;
    top = fmaxf(top, z);
    p[i] = z;
  }
  top = warp_max(top);
  if (top == -INFINITY && !__any_sync(0xffffffffu, nan)) return false;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int b = lane + 32 * i;
    p[i] = b >= base && b < NB ? expf(p[i] - top) : 0.f;
    sum += p[i];
  }
  const float inv = __fdiv_rn(1.0f, warp_sum(sum));
#pragma unroll
  for (int i = 0; i < E; ++i) p[i] *= inv;
  return true;
}

// Per CTA: column sums of p over its rows, the number of counted rows, and the blocks' slot counts.
// scores may be NULL (counts only); idx may be NULL (counts given).
template <int E>
__global__ void __launch_bounds__(kBalWarps * 32)
balance_partial_kernel(const float* __restrict__ scores, int64_t M, int NB, int base, float temperature,
                       const uint8_t* __restrict__ valid, const int32_t* __restrict__ idx,
                       const int32_t* __restrict__ cnt, int capacity, float* __restrict__ psum,
                       int32_t* __restrict__ rows, int32_t* __restrict__ hist) {
  extern __shared__ float sm[];  // [kBalWarps][NB] column sums, then [NB] slot counts
  int* sh = reinterpret_cast<int*>(sm + kBalWarps * NB);
  __shared__ int s_rows;
  for (int i = threadIdx.x; i < NB; i += blockDim.x) sh[i] = 0;
  if (threadIdx.x == 0) s_rows = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.f;
  int counted = 0;
  for (int64_t t = (int64_t)blockIdx.x * kBalWarps + warp; t < M; t += (int64_t)gridDim.x * kBalWarps) {
    if (valid && !valid[t]) continue;
    if (idx) {
      const int n = min(cnt[t], capacity);
      for (int k = lane; k < n; k += 32) {
        const int b = idx[t * capacity + k];
        if (b >= 0 && b < NB) atomicAdd(&sh[b], 1);
      }
    }
    if (scores) {
      float p[E];
      if (balance_row<E>(scores + t * NB, NB, base, temperature, lane, p)) {
        ++counted;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] += p[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (lane + 32 * i < NB) sm[warp * NB + lane + 32 * i] = acc[i];
  if (lane == 0) atomicAdd(&s_rows, counted);
  __syncthreads();
  for (int b = threadIdx.x; b < NB; b += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kBalWarps; ++w) s += sm[w * NB + b];
    psum[(int64_t)blockIdx.x * NB + b] = s;
    hist[(int64_t)blockIdx.x * NB + b] = sh[b];
  }
  if (threadIdx.x == 0) rows[blockIdx.x] = s_rows;
}

// One CTA: joins the partials in their order, writes the counts, the loss and what the gradient needs:
// state[b] = f_b - 1/R (0 when nothing was routed) and state[NB] = R / (T n).
__global__ void __launch_bounds__(1024)
balance_join_kernel(const float* __restrict__ psum, const int32_t* __restrict__ rows,
                    const int32_t* __restrict__ hist, int parts, int NB, int base, float temperature,
                    const int64_t* __restrict__ counts_in, int64_t* __restrict__ counts, float* __restrict__ loss,
                    float* __restrict__ state) {
  __shared__ unsigned long long s_total;
  __shared__ long long s_rows;
  __shared__ double s_loss[32];
  const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
  if (b == 0) {
    s_total = 0;
    long long r = 0;
    for (int i = 0; i < parts; ++i) r += rows[i];
    s_rows = r;
  }
  __syncthreads();
  int64_t c = 0;
  double ps = 0.0;
  if (b < NB) {
    if (counts_in) c = counts_in[b];
    for (int i = 0; i < parts; ++i) {
      if (!counts_in) c += hist[(int64_t)i * NB + b];
      ps += (double)psum[(int64_t)i * NB + b];
    }
    if (counts) counts[b] = c;
    if (c) atomicAdd(&s_total, (unsigned long long)c);
  }
  __syncthreads();
  if (!loss) return;
  const int64_t total = (int64_t)s_total, n = s_rows;
  const int R = NB - base;
  const bool remote = b >= base && b < NB;
  const double f = total > 0 && remote ? (double)c / (double)total : 0.0;
  double part = remote ? f * ps : 0.0;
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) s_loss[warp] = part;
  __syncthreads();
  if (b == 0) {
    double s = 0.0;
    for (int w = 0; w < 32; ++w) s += s_loss[w];
    *loss = n > 0 ? (float)(s * R / (double)n) : (float)s;
    state[NB] = n > 0 ? (float)((double)R / ((double)temperature * (double)n)) : 0.f;
  }
  if (b < NB)
    state[b] = total > 0 && remote ? (float)((double)(c * R - total) / ((double)total * R)) : 0.f;
}

template <int E>
__global__ void __launch_bounds__(kBalWarps * 32)
balance_grad_kernel(const float* __restrict__ scores, int64_t M, int NB, int base, float temperature,
                    const uint8_t* __restrict__ valid, const float* __restrict__ state,
                    const float* __restrict__ dloss, float* __restrict__ ds) {
  const int lane = threadIdx.x & 31;
  const float scale = state[NB] * *dloss;
  float f[E];
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = lane + 32 * i < NB ? state[lane + 32 * i] : 0.f;
  for (int64_t t = (int64_t)blockIdx.x * kBalWarps + (threadIdx.x >> 5); t < M; t += (int64_t)gridDim.x * kBalWarps) {
    float p[E];
    const bool counted = (!valid || valid[t]) && balance_row<E>(scores + t * NB, NB, base, temperature, lane, p);
    float inner = 0.f;
    if (counted) {
#pragma unroll
      for (int i = 0; i < E; ++i) inner = fmaf(p[i], f[i], inner);
      inner = warp_sum(inner);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int b = lane + 32 * i;
      if (b < NB) ds[t * NB + b] = counted && b >= base ? p[i] * (f[i] - inner) * scale : 0.f;
    }
  }
}

int balance_ctas(int64_t M) { return (int)std::max<int64_t>(1, std::min<int64_t>((M + kBalWarps - 1) / kBalWarps, kBalMaxCtas)); }

template <int E>
void balance_fwd_go(const float* scores, int64_t M, int NB, int base, float temperature, const uint8_t* valid,
                    const int32_t* idx, const int32_t* cnt, int capacity, float* psum, int32_t* rows, int32_t* hist,
                    cudaStream_t st) {
  const size_t smem = (size_t)(kBalWarps + 1) * NB * 4;  // at most 36 KB
  balance_partial_kernel<E><<<balance_ctas(M), kBalWarps * 32, smem, st>>>(
      scores, M, NB, base, temperature, valid, idx, cnt, capacity, psum, rows, hist);
}

}  // namespace
}  // namespace fp

using namespace fp;

#define FP_BY_WIDTH(NB, CALL)                 \
  do {                                        \
    if ((NB) <= 32) { constexpr int E = 1; CALL; }        \
    else if ((NB) <= 64) { constexpr int E = 2; CALL; }   \
    else if ((NB) <= 128) { constexpr int E = 4; CALL; }  \
    else if ((NB) <= 256) { constexpr int E = 8; CALL; }  \
    else if ((NB) <= 512) { constexpr int E = 16; CALL; } \
    else { constexpr int E = 32; CALL; }      \
  } while (0)

extern "C" {

int fp_router_scores_train(const void* x, const void* q_proj, const void* block_keys, int dtype, int64_t M, int D,
                           int NB, float* scores, float* q16, float* rnorm, void* codes, void* scales, void* stream) {
  if (dtype != FP_DTYPE_F32 && dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (M < 0 || D <= 0 || NB <= 0) return FP_ERR_INVALID_ARG;
  if (D % 8 != 0 || NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if ((codes == nullptr) != (scales == nullptr)) return FP_ERR_INVALID_ARG;
  if (M == 0) return FP_OK;
  if (!x || !q_proj || !block_keys || !scores || !q16 || !rnorm) return FP_ERR_INVALID_ARG;
  if (!al16(x) || !al16(q_proj) || !al16(codes)) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  if (const int rc = launch_router_scores(x, q_proj, block_keys, dtype, M, D, NB, 1.0f, scores, q16,
                                          (cudaStream_t)stream, nullptr, rnorm))
    return rc;
  return codes ? fp_mxfp8_quantize(x, dtype, M * D, codes, scales, stream) : FP_OK;
}

size_t fp_router_scores_bwd_workspace_size(int64_t M, int D, int NB) {
  return M > 0 && D > 0 && NB > 0 ? bwd_plan(M, D, NB).total : 256;
}

int fp_router_scores_bwd(const float* dscores, const void* x, const void* codes, const void* scales,
                         const void* q_proj, const void* block_keys, const float* q16, const float* rnorm, int dtype,
                         int64_t M, int D, int NB, void* dx, void* dq_proj, void* dblock_keys, int grad_dtype,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != FP_DTYPE_F32 && dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (grad_dtype != FP_DTYPE_F32 && grad_dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (M <= 0 || D <= 0 || NB <= 0) return FP_ERR_INVALID_ARG;
  if (D % 8 != 0 || NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if (!dscores || !q_proj || !block_keys || !q16 || !rnorm || !workspace) return FP_ERR_INVALID_ARG;
  if (dq_proj && !x && !codes) return FP_ERR_INVALID_ARG;
  if ((codes == nullptr) != (scales == nullptr)) return FP_ERR_INVALID_ARG;
  if (!al16(x) || !al16(codes) || !al16(q_proj) || !al16(dx) || !al16(dscores) || !al16(q16) || !al16(workspace))
    return FP_ERR_INVALID_ARG;
  if (workspace_bytes < bwd_plan(M, D, NB).total) return FP_ERR_WORKSPACE;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FP_DTYPE_BF16)
    return router_bwd(dscores, (const __nv_bfloat16*)x, (const uint8_t*)codes, (const uint8_t*)scales,
                      (const __nv_bfloat16*)q_proj, (const __nv_bfloat16*)block_keys, q16, rnorm, M, D, NB,
                      (__nv_bfloat16*)dx, dq_proj, dblock_keys, grad_dtype, ws, sms, st);
  return router_bwd(dscores, (const float*)x, (const uint8_t*)codes, (const uint8_t*)scales, (const float*)q_proj,
                    (const float*)block_keys, q16, rnorm, M, D, NB, (float*)dx, dq_proj, dblock_keys, grad_dtype, ws,
                    sms, st);
}

size_t fp_balance_workspace_size(int64_t M, int NB) {
  return M >= 0 && NB > 0 ? (size_t)balance_ctas(M) * (8 * (size_t)NB + 4) + 256 : 256;
}

int fp_balance_loss_fwd(const float* scores, int64_t M, int NB, int base_blocks, float temperature,
                        const uint8_t* valid, const int32_t* remote_indices, const int32_t* remote_counts,
                        int capacity, const int64_t* counts_in, int64_t* counts, float* loss, float* state,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || NB <= 0 || base_blocks < 0 || capacity < 0) return FP_ERR_INVALID_ARG;
  if (NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if ((remote_indices == nullptr) != (remote_counts == nullptr)) return FP_ERR_INVALID_ARG;
  if ((loss == nullptr) != (state == nullptr)) return FP_ERR_INVALID_ARG;
  if (loss && ((M > 0 && !scores) || base_blocks >= NB || !(temperature > 0.f))) return FP_ERR_INVALID_ARG;
  if (!loss && !counts) return FP_ERR_INVALID_ARG;
  if (M > 0 && !remote_indices && !counts_in) return FP_ERR_INVALID_ARG;
  if (!workspace || !al16(workspace)) return FP_ERR_INVALID_ARG;
  if (workspace_bytes < fp_balance_workspace_size(M, NB)) return FP_ERR_WORKSPACE;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int parts = balance_ctas(M);
  float* psum = (float*)workspace;
  int32_t* hist = (int32_t*)(psum + (size_t)parts * NB);
  int32_t* rows = hist + (size_t)parts * NB;
  const int32_t* idx = counts_in ? nullptr : remote_indices;
  FP_BY_WIDTH(NB, balance_fwd_go<E>(loss ? scores : nullptr, M, NB, base_blocks, temperature, valid, idx,
                                    remote_counts, capacity, psum, rows, hist, st));
  balance_join_kernel<<<1, 1024, 0, st>>>(psum, rows, hist, parts, NB, base_blocks, temperature, counts_in, counts, loss,
                                          state);
  return launched();
}

int fp_balance_loss_bwd(const float* scores, int64_t M, int NB, int base_blocks, float temperature,
                        const uint8_t* valid, const float* state, const float* dloss, float* dscores, void* stream) {
  if (M < 0 || NB <= 0 || base_blocks < 0 || base_blocks >= NB || !(temperature > 0.f)) return FP_ERR_INVALID_ARG;
  if (NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if (M == 0) return FP_OK;
  if (!scores || !state || !dloss || !dscores) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int grid = (int)std::min<int64_t>((M + kBalWarps - 1) / kBalWarps, (int64_t)sms * 8);
  FP_BY_WIDTH(NB, (balance_grad_kernel<E><<<grid, kBalWarps * 32, 0, st>>>(scores, M, NB, base_blocks, temperature,
                                                                          valid, state, dloss, dscores)));
  return launched();
}

}  // extern "C"
