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
#include <atomic>

namespace fp {
namespace {

constexpr int kIdx = 16;  // the router's width
constexpr int kMaxWidth = 1 << 24;

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int launched() { return cudaGetLastError() == cudaSuccess ? FP_OK : FP_ERR_CUDA; }

// Lets `kern` use up to `bytes` of dynamic shared memory on the current device (asked for once per device).
template <auto kern>
bool allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ uint32_t tf32_of(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void tf32_split(float v, uint32_t& hi, uint32_t& lo) {
  hi = tf32_of(v);
  lo = tf32_of(v - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero accumulators.
__device__ __forceinline__ void mma_bf16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// ------------------------------------------------------------------ scores of the training forward
// fp_router_scores' bf16 kernel (same products in the same order, so the same bits) for whole batches: a CTA
// stays for many tiles of 32 tokens, with the block keys in shared memory once (loaded per 16 tokens they took
// as long as the projection), a key serves four tokens from registers, and the normalisation factor and
// (kKeep) the MXFP8 copy of x leave in the same pass over x.  Warp: one quarter of D, 16 tokens; then 4
// tokens' scores.  Bound by latency (16384 x 4096: 37 us, 3.6 TB/s at 29 % issue; 16384 x 8192 with the copy: 102 us,
// 3.9 TB/s at 53 %): 128 registers leave 16 warps to an SM.
// With the copy, x comes by TMA (64 columns x 16 tokens) into a ring that a warp keeps for itself and that runs
// on through the scores of a tile (55 us; loads into registers 59 us: the quantisation leaves too few in
// flight).  Without it, plain loads of two steps at a time do better (36 us; the ring 42 us: W_q's fragments
// come through L1, which the ring shrinks).
constexpr int kFwWarps = 8;
constexpr int kFwTokens = 32;
constexpr int kFwStages = 4;
constexpr int kFwRing = kFwWarps * kFwStages * 2048;

// MXFP8 codes of 16 consecutive bf16 values (w: in order); the lane's neighbour (lane ^ 1) holds the other half of
// the block.  All lanes of the warp call this together.
__device__ __forceinline__ void mx_quantize16(const uint32_t (&w)[8], uint4& codes, int& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
  uint32_t top = max(m & 0xFFFF0000u, m << 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  float v[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  if (__any_sync(0xffffffffu, top >= __float_as_uint(kMxHuge))) {
    uint32_t fin = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) fin = max(fin, mx_finite(v[i]));
    top = max(fin, __shfl_xor_sync(0xffffffffu, fin, 1));
  }
  byte = mx_scale_byte(top);
  const float inv = mx_inv_scale(byte);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = (uint32_t)mx_pack2(v[4 * i] * inv, v[4 * i + 1] * inv) |
           ((uint32_t)mx_pack2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
  codes = make_uint4(c[0], c[1], c[2], c[3]);
}

__device__ __forceinline__ void load32(const __nv_bfloat16* p, uint32_t (&w)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
}

// 32 bytes as two pieces of shared memory.
__device__ __forceinline__ void lds32(const uint8_t* p, const uint8_t* q, uint32_t (&w)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p), v = *reinterpret_cast<const uint4*>(q);
  w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
}

template <bool kKeep>
__global__ void __launch_bounds__(kFwWarps * 32, 2)
router_fwd_kernel(const __grid_constant__ CUtensorMap map, const __nv_bfloat16* __restrict__ x,
                  const __nv_bfloat16* __restrict__ wq, const __nv_bfloat16* __restrict__ k16, int64_t M, int D,
                  int NB, float* __restrict__ scores, float* __restrict__ q16, float* __restrict__ rnorm,
                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  extern __shared__ uint8_t fw_dyn[];
  uint8_t* ring = fw_dyn + (1024 - (smem_u32(fw_dyn) & 1023)) % 1024;  // [warp][stage] tiles of x
  float* skeys = reinterpret_cast<float*>(ring + (kKeep ? kFwRing : 0));  // [16][NB] block keys
  __shared__ uint64_t bars[kFwWarps][kFwStages];
  __shared__ float sq[2][4][16 * 17];            // [token group][quarter of D] partial projections
  __shared__ float4 sv[kFwTokens * 4];           // [token][16] projections
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int quarter = warp & 3, group = warp >> 2, dpart = D / 4, kbeg = quarter * dpart;
  const int tiles = (int)((M + kFwTokens - 1) / kFwTokens);
  uint8_t* xs = ring + warp * kFwStages * 2048;
  int f_tile = blockIdx.x, f_k = 0, f_stage = 0;  // the next copy (lane 0)
  const auto fetch = [&] {
    if (f_tile >= tiles) return;
    mbar_arrive_expect_tx(&bars[warp][f_stage], 2048);
    tma_load_2d(xs + f_stage * 2048, &map, &bars[warp][f_stage], kbeg + f_k, f_tile * kFwTokens + 16 * group);
    f_stage = (f_stage + 1) % kFwStages;
    f_k += 64;
    if (f_k == dpart) {
      f_k = 0;
      f_tile += gridDim.x;
    }
  };
  if (kKeep && lane == 0) {
    for (int k = 0; k < kFwStages; ++k) mbar_init(&bars[warp][k], 1);
    fence_mbar_init();
    for (int k = 0; k < kFwStages; ++k) fetch();
  }
  for (int i = threadIdx.x; i < NB * kIdx; i += blockDim.x) {
    const int j = i / NB, b = i - j * NB;
    skeys[i] = __bfloat162float(k16[b * kIdx + j]);
  }
  __syncthreads();  // keys and barriers
  const __nv_bfloat16* wa = wq + (int64_t)g * D + kbeg + 16 * t;
  const __nv_bfloat16* wb = wa + (int64_t)8 * D;
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  uint32_t B0[8], B1[8];  // kKeep: W_q's fragments of the step to come
  if constexpr (kKeep) {
    load32(wa, B0);
    load32(wb, B1);
  }
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t tok0 = (int64_t)tile * kFwTokens;
    const int64_t ta = tok0 + 16 * group + g, tb = ta + 8;
    float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (kKeep) {
#pragma unroll 1
      for (int k0 = 0; k0 < dpart && ok; k0 += 64) {
        uint32_t A0[8], A1[8];
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][stage], parity, nullptr, 0));
        if (!ok) break;
        // 128-byte swizzle: 16-byte piece ^ row % 8; rows g and g + 8, pieces 2 t and 2 t + 1
        const uint8_t* r = xs + stage * 2048 + g * 128;
        const int p0 = ((2 * t) ^ g) << 4, p1 = ((2 * t + 1) ^ g) << 4;
        lds32(r + p0, r + p1, A0);
        lds32(r + 1024 + p0, r + 1024 + p1, A1);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          mma_bf16(c0, A0[2 * st], A1[2 * st], A0[2 * st + 1], A1[2 * st + 1], B0[2 * st], B0[2 * st + 1]);
          mma_bf16(c1, A0[2 * st], A1[2 * st], A0[2 * st + 1], A1[2 * st + 1], B1[2 * st], B1[2 * st + 1]);
        }
        const int kn = k0 + 64 < dpart ? k0 + 64 : 0;
        load32(wa + kn, B0);
        load32(wb + kn, B1);
        __syncwarp();  // the tile is in every lane's registers
        if (lane == 0) fetch();
        if (++stage == kFwStages) {
          stage = 0;
          parity ^= 1;
        }
        const int64_t col = kbeg + k0 + 16 * t;
        uint4 q;
        int byte;
        mx_quantize16(A0, q, byte);
        if (ta < M) {
          *reinterpret_cast<uint4*>(codes + ta * D + col) = q;
          if (!(t & 1)) scales[(ta * D + col) / kMxBlock] = (uint8_t)byte;
        }
        mx_quantize16(A1, q, byte);
        if (tb < M) {
          *reinterpret_cast<uint4*>(codes + tb * D + col) = q;
          if (!(t & 1)) scales[(tb * D + col) / kMxBlock] = (uint8_t)byte;
        }
      }
      if (!ok)  // a copy did not arrive within the wait limit: the tile's scores become NaN, and all that follow
        c0[0] = c0[1] = c0[2] = c0[3] = __uint_as_float(0x7FC00000u);
    } else {
      const __nv_bfloat16* xa = x + (ta < M ? ta : M - 1) * D + kbeg + 16 * t;
      const __nv_bfloat16* xb = x + (tb < M ? tb : M - 1) * D + kbeg + 16 * t;
#pragma unroll 2
      for (int k0 = 0; k0 < dpart; k0 += 64) {
        uint32_t A0[8], A1[8], W0[8], W1[8];
        load32(xa + k0, A0);
        load32(xb + k0, A1);
        load32(wa + k0, W0);
        load32(wb + k0, W1);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          mma_bf16(c0, A0[2 * st], A1[2 * st], A0[2 * st + 1], A1[2 * st + 1], W0[2 * st], W0[2 * st + 1]);
          mma_bf16(c1, A0[2 * st], A1[2 * st], A0[2 * st + 1], A1[2 * st + 1], W1[2 * st], W1[2 * st + 1]);
        }
      }
    }
    float* q = sq[group][quarter];
    q[g * 17 + 2 * t] = c0[0];
    q[g * 17 + 2 * t + 1] = c0[1];
    q[(g + 8) * 17 + 2 * t] = c0[2];
    q[(g + 8) * 17 + 2 * t + 1] = c0[3];
    q[g * 17 + 8 + 2 * t] = c1[0];
    q[g * 17 + 9 + 2 * t] = c1[1];
    q[(g + 8) * 17 + 8 + 2 * t] = c1[2];
    q[(g + 8) * 17 + 9 + 2 * t] = c1[3];
    __syncthreads();
    // the quarters' sum, in order: two tokens at a time, lane = (token, dimension)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = warp * 4 + 2 * h + (lane >> 4), j = lane & 15, i = (r & 15) * 17 + j;
      float v = sq[r >> 4][0][i];
#pragma unroll
      for (int w = 1; w < 4; ++w) v += sq[r >> 4][w][i];
      reinterpret_cast<float*>(sv)[r * 16 + j] = v;
    }
    __syncwarp();
    const float eps = 1.1920928955078125e-07f;  // torch.finfo(float32).eps: F.rms_norm's default
    float qv[4][16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t tok = tok0 + warp * 4 + r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = sv[(warp * 4 + r) * 4 + i];
        qv[r][4 * i] = v.x; qv[r][4 * i + 1] = v.y; qv[r][4 * i + 2] = v.z; qv[r][4 * i + 3] = v.w;
      }
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) ss = fmaf(qv[r][j], qv[r][j], ss);
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(ss * (1.0f / 16.0f) + eps));
#pragma unroll
      for (int j = 0; j < 16; ++j) qv[r][j] *= inv;
      if (tok < M) {
        if (lane < 16) q16[tok * 16 + lane] = reinterpret_cast<float*>(sv)[(warp * 4 + r) * 16 + lane] * inv;
        if (lane == 0) rnorm[tok] = inv;
      }
    }
    float* out = scores + (tok0 + warp * 4) * NB;
    const int live = (int)min((int64_t)4, M - (tok0 + warp * 4));
    for (int b = lane; b < NB; b += 32) {
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float kv = skeys[j * NB + b];
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[r] = fmaf(qv[r][j], kv, sc[r]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < live) out[(int64_t)r * NB + b] = sc[r] * 0.25f;  // / sqrt(16)
    }
    __syncthreads();  // the partial projections' place is free again
  }
  if (!ok)  // once more for the copies under way, before their place goes
    for (int k = 0; k < kFwStages; ++k) {
      mbar_wait(&bars[warp][stage], parity, nullptr, 0);
      if (++stage == kFwStages) {
        stage = 0;
        parity ^= 1;
      }
    }
}

// The same for fp32 and for widths that are not a multiple of 256: fp_router_scores' CUDA-core kernel in its
// order of sums (lane: columns 8 lane + 256 i, then a butterfly), so the same bits.  What held that kernel at
// 270 us (16384 x 4096 fp32) were W_q's loads, 16 rows of them one after the other for each step of x; here a
// step's W_q (256 columns) is in shared memory, copied one step ahead for the CTA's 32 tokens, and x is loaded
// one step ahead.  134 us then, of which the FMA units take 29 and shared memory 29: 206 registers leave one CTA
// of 8 warps to an SM (12.5 % of the warps, 47 % issue), too few to cover each other's latency.
constexpr int kAnyTokens = 4;  // of a warp

template <typename T>
struct Raw8 {  // 8 consecutive elements
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint4 a = w[0], b = w[1];
      v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    } else {
      const uint32_t r[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(r[i] << 16);
        v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
      }
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(kFwWarps * 32, 1)
router_fwd_any_kernel(const T* __restrict__ x, const T* __restrict__ wq, const T* __restrict__ k16, int64_t M, int D,
                      int NB, float* __restrict__ scores, float* __restrict__ q16, float* __restrict__ rnorm) {
  constexpr int kPieces = sizeof(T) / 2;                // 16-byte pieces of 8 elements
  constexpr int kStep = 16 * kPieces * 32;              // of one step of W_q
  extern __shared__ uint4 any_dyn[];                    // [2][16][piece][lane] W_q, then [16][NB] block keys
  float* skeys = reinterpret_cast<float*>(any_dyn + 2 * kStep);
  for (int i = threadIdx.x; i < NB * kIdx; i += blockDim.x) {
    const int j = i / NB, b = i - j * NB;
    skeys[i] = to_f32(k16[b * kIdx + j]);
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int steps = (D + 255) / 256;
  const auto copy_w = [&](int step) {
    if (step < steps) {
      for (int i = threadIdx.x; i < kStep; i += kFwWarps * 32) {
        const int l = (i / kPieces) & 31, j = i / (kPieces * 32), piece = i % kPieces;  // along a row of W_q
        const int c = step * 256 + l * 8;
        if (c < D)
          cp_async_16(smem_u32(any_dyn + (step & 1) * kStep + (j * kPieces + piece) * 32 + l),
                      reinterpret_cast<const uint4*>(wq + (int64_t)j * D + c) + piece);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kTile = kFwWarps * kAnyTokens;
  for (int64_t base = (int64_t)blockIdx.x * kTile; base < M; base += (int64_t)gridDim.x * kTile) {
    const int64_t tok0 = base + warp * kAnyTokens;
    const int live = (int)max((int64_t)0, min((int64_t)kAnyTokens, M - tok0));
    float acc[kAnyTokens][kIdx];
    Raw8<T> next[kAnyTokens];
#pragma unroll
    for (int r = 0; r < kAnyTokens; ++r)
#pragma unroll
      for (int j = 0; j < kIdx; ++j) acc[r][j] = 0.f;
    const auto load_x = [&](int step) {
      const int c = step * 256 + lane * 8;
#pragma unroll
      for (int r = 0; r < kAnyTokens; ++r)
        if (c < D) next[r].load(x + (tok0 + r < M ? tok0 + r : M - 1) * D + c);
    };
    __syncthreads();  // keys; W_q's first place is free
    copy_w(0);
    load_x(0);
    for (int step = 0; step < steps; ++step) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      copy_w(step + 1);
      float xv[kAnyTokens][8];
#pragma unroll
      for (int r = 0; r < kAnyTokens; ++r) next[r].unpack(xv[r]);
      if (step + 1 < steps) load_x(step + 1);
      if (step * 256 + lane * 8 < D) {
        const uint4* w = any_dyn + (step & 1) * kStep + lane;
#pragma unroll
        for (int j = 0; j < kIdx; ++j) {
          Raw8<T> raw;
#pragma unroll
          for (int i = 0; i < kPieces; ++i) raw.w[i] = w[(j * kPieces + i) * 32];
          float wv[8];
          raw.unpack(wv);
#pragma unroll
          for (int r = 0; r < kAnyTokens; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][j] = fmaf(xv[r][e], wv[e], acc[r][j]);
        }
      }
    }
    const float eps = 1.1920928955078125e-07f;  // torch.finfo(float32).eps: F.rms_norm's default
#pragma unroll
    for (int r = 0; r < kAnyTokens; ++r) {
#pragma unroll
      for (int j = 0; j < kIdx; ++j) acc[r][j] = warp_sum(acc[r][j]);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < kIdx; ++j) ss = fmaf(acc[r][j], acc[r][j], ss);
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(ss * (1.0f / 16.0f) + eps));
      float own = 0.f;
#pragma unroll
      for (int j = 0; j < kIdx; ++j) {
        acc[r][j] *= inv;
        if (lane == j) own = acc[r][j];
      }
      if (r < live) {
        if (lane < kIdx) q16[(tok0 + r) * kIdx + lane] = own;
        if (lane == 0) rnorm[tok0 + r] = inv;
      }
    }
    for (int b = lane; b < NB; b += 32) {
      float sc[kAnyTokens] = {};
#pragma unroll
      for (int j = 0; j < kIdx; ++j) {
        const float kv = skeys[j * NB + b];
#pragma unroll
        for (int r = 0; r < kAnyTokens; ++r) sc[r] = fmaf(acc[r][j], kv, sc[r]);
      }
#pragma unroll
      for (int r = 0; r < kAnyTokens; ++r)
        if (r < live) scores[(tok0 + r) * NB + b] = sc[r] * 0.25f;  // / sqrt(16)
    }
  }
}

template <typename T>
int launch_router_fwd_any(const void* x, const void* wq, const void* k16, int64_t M, int D, int NB, float* scores,
                          float* q16, float* rnorm, int sms, cudaStream_t st) {
  constexpr auto kern = router_fwd_any_kernel<T>;
  constexpr int ring = 2 * 16 * 256 * (int)sizeof(T);
  if (!allow_smem<kern>(ring + 64 * 1024)) return FP_ERR_CUDA;
  const int64_t tiles = (M + kFwWarps * kAnyTokens - 1) / (kFwWarps * kAnyTokens);
  kern<<<(int)std::min<int64_t>(tiles, 2 * sms), kFwWarps * 32, ring + NB * kIdx * 4, st>>>(
      (const T*)x, (const T*)wq, (const T*)k16, M, D, NB, scores, q16, rnorm);
  return launched();
}

template <bool kKeep>
int launch_router_fwd(const void* x, const void* wq, const void* k16, int64_t M, int D, int NB, float* scores,
                      float* q16, float* rnorm, void* codes, void* scales, int sms, cudaStream_t st) {
  constexpr auto kern = router_fwd_kernel<kKeep>;
  constexpr int ring = kKeep ? kFwRing : 0;
  const int smem = 1024 + ring + NB * kIdx * 4;  // at most 129 KB
  if (!allow_smem<kern>(1024 + ring + 64 * 1024)) return FP_ERR_CUDA;
  CUtensorMap map{};
  if (kKeep && !encode_map_2d(&map, x, D, M, (uint64_t)D * 2, 64, 16)) return FP_ERR_CUDA;
  const int grid = (int)std::min<int64_t>((M + kFwTokens - 1) / kFwTokens, 2 * sms);
  kern<<<grid, kFwWarps * 32, smem, st>>>(map, (const __nv_bfloat16*)x, (const __nv_bfloat16*)wq,
                                          (const __nv_bfloat16*)k16, M, D, NB, scores, q16, rnorm, (uint8_t*)codes,
                                          (uint8_t*)scales);
  return launched();
}

// ------------------------------------------------------------------ gradient of the scores
// Three launches.  (1) One pass over dS: dq of every token and partial sums of dK.  (2) One pass over x: dx and
// partial sums of dWq.  (3) The partial sums, in a fixed order.  The products are 16 wide on one side, so the
// passes are bound by memory once they run on tensor cores; a tile of 128 rows (tcgen05) would be filled to
// an eighth, mma.sync fits: the 16 router dimensions are its m (pass 1) and its k or two n-tiles (pass 2).
//
// Precision.  Pass 1 multiplies fp32 values as tf32 pieces, v = hi + lo (the rest is below 2^-22 of v):
// hi hi + hi lo + lo hi, fp32 accumulators.  Pass 2 with bf16 x holds dq as three bf16 pieces, which together are
// all of its 24 bits (two left errors of 2.5e-6 in dWq and moved one in 450 roundings of dx); x and Wq are
// exact.  fp32 x stays on the FMA units.
//
// Fragment coordinates below: lane = 4 g + t, g = 0..7, t = 0..3.

// 16 consecutive elements, 16-byte aligned.
__device__ __forceinline__ void load_row16(const float* p, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
    v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
  }
}
__device__ __forceinline__ void load_row16(const __nv_bfloat16* p, float (&v)[16]) {
  uint32_t w[8];
  load32(p, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// Four columns of one row of dS, zeros outside.  The loads are unconditional, from a place inside the tensor, so
// that a loop's loads can be issued together (behind a branch they went one by one: 22 us for dq at
// 16384 x 448).  kVec: NB % 4 == 0.
template <bool kVec>
__device__ __forceinline__ float4 ds4(const float* __restrict__ ds, int64_t t, int64_t M, int b, int NB) {
  const bool in = t < M;
  const float* row = ds + (in ? t : M - 1) * NB;
  float4 v;
  if constexpr (kVec) {
    v = __ldg(reinterpret_cast<const float4*>(row + min(b, NB - 4)));
    if (!in || b >= NB) v = make_float4(0.f, 0.f, 0.f, 0.f);
  } else {
    v.x = __ldg(row + min(b, NB - 1));
    v.y = __ldg(row + min(b + 1, NB - 1));
    v.z = __ldg(row + min(b + 2, NB - 1));
    v.w = __ldg(row + min(b + 3, NB - 1));
    if (!in || b >= NB) v.x = 0.f;
    if (!in || b + 1 >= NB) v.y = 0.f;
    if (!in || b + 2 >= NB) v.z = 0.f;
    if (!in || b + 3 >= NB) v.w = 0.f;
  }
  return v;
}

constexpr int kDqWarps = 8;
constexpr int kDqTokens = 8 * kDqWarps;  // tokens of a CTA's tile
constexpr int kDqMaxCtas = 296;  // two to each of the 148 SMs; also the partial sums of dK
constexpr int kDqPieces = 3;                  // bf16 pieces of a packed dq
constexpr int kDqTileBytes = kDqPieces * 512;  // 16 tokens of them

// Pass 1.  CTAs of two kinds, running side by side (one after the other in each CTA they took 31 us at 16384 x 448).
// dq (blockIdx.y = 0 where dq is wanted): 8 tokens to a warp, a^T[j, tok] = K^T[j, b] dS^T[b, tok], then dq.
// dK (the other rows of the grid, 256 blocks each): 32 blocks to a warp over the CTA's 64 tokens, dK^T[j, b] =
// n^T[j, tok] dS[tok, b], kept in registers over all of the CTA's tiles.  The order of b within a product and
// the columns of a tile are permuted so that a lane's elements are 16 contiguous bytes.
// dq: kPacked, per tile of 16 tokens the three bf16 pieces as pass 2's fragments ([tile][piece][lane] uint4);
// otherwise fp32 [M, 16].
template <typename T, bool kPacked, bool kVec>
__global__ void __launch_bounds__(kDqWarps * 32)
router_dq_kernel(const float* __restrict__ ds, const T* __restrict__ k16, const float* __restrict__ q16,
                 const float* __restrict__ rnorm, int64_t M, int NB, void* __restrict__ dq_out,
                 float* __restrict__ dk_part) {
  extern __shared__ float4 sk[];  // [ceil(NB / 16)][2][32]: K as the dq products' fragments
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int nk = (NB + 15) / 16;
  const bool for_dq = dq_out && blockIdx.y == 0;
  if (for_dq) {
    // the first tile's rows start towards L2 while K goes to shared memory, one row of K to a thread
    const int64_t row0 = (int64_t)blockIdx.x * kDqTokens + 8 * warp;
    const int64_t bytes = min((int64_t)8, M - row0) * NB * 4;
    for (int64_t o = 128 * lane; o < bytes; o += 4096)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(ds + row0 * NB) + o));
    for (int b = threadIdx.x; b < nk * 16; b += blockDim.x) {
      float v[kIdx];
#pragma unroll
      for (int j = 0; j < kIdx; ++j) v[j] = 0.f;
      if (b < NB) load_row16(k16 + b * kIdx, v);
      // row b is k-index t (even) or t + 4 (odd) of step s: t = b / 4 % 4, s = b / 2 % 2
      float* o = reinterpret_cast<float*>(sk) + (((b >> 4) * 2 + (b >> 1 & 1)) * 32 + (b >> 2 & 3)) * 4 + 2 * (b & 1);
#pragma unroll
      for (int j = 0; j < kIdx; ++j) o[16 * (j & 7) + (j >> 3)] = v[j];
    }
    __syncthreads();
  }
  // dK: the warp's blocks b0 + 0..31
  const int b0 = 32 * (kDqWarps * ((int)blockIdx.y - (dq_out ? 1 : 0)) + warp);
  float dk[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[k][e] = 0.f;

  for (int64_t base = (int64_t)blockIdx.x * kDqTokens; base < M; base += (int64_t)gridDim.x * kDqTokens) {
    const int64_t tok0 = base + 8 * warp;
    // (a tile of 16 tokens that ends past M is written whole: zeros behind the last token)
    if (for_dq && tok0 < (M + 15) / 16 * 16) {
      float a[4] = {};
      float n0[2], n1[2], r[2];  // of tokens 2 t and 2 t + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t tok = tok0 + 2 * t + e;
        n0[e] = n1[e] = r[e] = 0.f;
        if (tok < M) {
          n0[e] = __ldg(q16 + tok * kIdx + g);
          n1[e] = __ldg(q16 + tok * kIdx + g + 8);
          r[e] = __ldg(rnorm + tok);
        }
      }
      // The tensor cores round a sum towards zero: chains of 8 steps, joined by ordinary additions (one chain over
      // 1000 blocks left errors of 3e-6, this way 5e-7; one over a CTA's tokens 6e-6 in dK at 262144 tokens).
      for (int k0 = 0; k0 < nk; k0 += 8) {
        float c[4] = {}, cl[4] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = k0 + i < nk ? k0 + i : nk;  // step nk: columns past the end, zeros
          const float4 v = ds4<kVec>(ds, tok0 + g, M, 16 * k + 4 * t, NB);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float4 kv = sk[(min(k, nk - 1) * 2 + s) * 32 + lane];
            const float kf[4] = {kv.x, kv.y, kv.z, kv.w};
            uint32_t kh[4], kl[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (sizeof(T) == 4) tf32_split(kf[e], kh[e], kl[e]);
              else kh[e] = __float_as_uint(kf[e]);  // a bf16 value is a tf32 value
            }
            uint32_t h0, l0, h1, l1;
            tf32_split(s ? v.z : v.x, h0, l0);
            tf32_split(s ? v.w : v.y, h1, l1);
            mma_tf32(cl, kh, l0, l1);
            if constexpr (sizeof(T) == 4) mma_tf32(cl, kl, h0, h1);
            mma_tf32(c, kh, h0, h1);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += c[e] + cl[e];
      }
      // a: token 2 t (+1: odd element), j = g (elements 0, 1) and g + 8 (2, 3)
      float d[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t tok = tok0 + 2 * t + e;
        const bool in = tok < M;
        const float a0 = a[e] * 0.25f, a1 = a[2 + e] * 0.25f;
        float dot = a0 * n0[e] + a1 * n1[e];
        dot += __shfl_xor_sync(0xffffffffu, dot, 4);
        dot += __shfl_xor_sync(0xffffffffu, dot, 8);
        dot += __shfl_xor_sync(0xffffffffu, dot, 16);
        dot *= 1.0f / kIdx;
        d[0][e] = in ? r[e] * (a0 - n0[e] * dot) : 0.f;
        d[1][e] = in ? r[e] * (a1 - n1[e] * dot) : 0.f;
        if constexpr (!kPacked) {
          if (in) {
            float* o = reinterpret_cast<float*>(dq_out) + tok * kIdx + g;
            o[0] = d[0][e];
            o[8] = d[1][e];
          }
        }
      }
      if constexpr (kPacked) {
        uint2* o = reinterpret_cast<uint2*>(dq_out) + (tok0 / 16) * (64 * kDqPieces) + 2 * lane + (tok0 / 8 & 1);
#pragma unroll
        for (int k = 0; k < kDqPieces; ++k) {
          uint32_t w[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            w[j] = pack_bf16(d[j][0], d[j][1]);
            d[j][0] -= __uint_as_float(w[j] << 16);
            d[j][1] -= __uint_as_float(w[j] & 0xFFFF0000u);
          }
          o[64 * k] = make_uint2(w[0], w[1]);
        }
      }
    }
    if (!for_dq && b0 < NB) {
      const int64_t end = min(base + kDqTokens, M);
      float c[4][4] = {}, cl[4][4] = {};  // as for dq: chains of 8 steps, ordinary additions between tiles
#pragma unroll 4
      for (int64_t s0 = base; s0 < end; s0 += 8) {
        const int64_t ta = s0 + t, tb = s0 + t + 4;
        uint32_t nh[4], nl[4];
        // (past the last token dS is zero, and the row read in its place is a token's)
        const float* qa = q16 + min(ta, M - 1) * kIdx + g;
        const float* qb = q16 + min(tb, M - 1) * kIdx + g;
        const bool ia = ta < M, ib = tb < M;
        const float n4[4] = {ia ? __ldg(qa) : 0.f, ia ? __ldg(qa + 8) : 0.f, ib ? __ldg(qb) : 0.f,
                             ib ? __ldg(qb + 8) : 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) tf32_split(n4[e], nh[e], nl[e]);
        const float4 va = ds4<kVec>(ds, ta, M, b0 + 4 * g, NB), vb = ds4<kVec>(ds, tb, M, b0 + 4 * g, NB);
        const float fa[4] = {va.x, va.y, va.z, va.w}, fb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t h0, l0, h1, l1;
          tf32_split(fa[k], h0, l0);
          tf32_split(fb[k], h1, l1);
          mma_tf32(cl[k], nh, l0, l1);
          mma_tf32(cl[k], nl, h0, h1);
          mma_tf32(c[k], nh, h0, h1);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) dk[k][e] += c[k][e] + cl[k][e];
    }
  }
  if (!for_dq) {  // dk[k]: b = b0 + 8 t + k (+4: odd element), j = g (elements 0, 1) and g + 8 (2, 3)
    float* o = dk_part + (int64_t)blockIdx.x * NB * kIdx;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int b = b0 + 8 * t + 4 * (e & 1) + k;
        if (b < NB) o[b * kIdx + g + 8 * (e >> 1)] = dk[k][e] * 0.25f;
      }
  }
}

// Pass 2, bf16.  A warp owns 64 columns and steps through its CTA's tokens 16 at a time: the lane's four 16-byte
// pieces of x (tokens 2t, 2t+1, 2t+8, 2t+9, columns 8g..) become the dWq product's A operand by permuting
// halfwords of two tokens' words, without shared memory; dWq^T[d, j] stays in 32 registers over all tokens.
// dx[tok, d] = dq Wq takes dq's fragments transposed (movmatrix) and Wq's from registers, its columns permuted
// so that a lane stores 16 contiguous bytes.  Neither HBM (16384 x 4096: 57 us, 3.9 TB/s; from the copy 16384 x 8192:
// 127 us, 2.8 TB/s), issue (44 and 55 %) nor the tensor cores (48 and 41 %) is full: 16 warps to an SM wait for
// one another's chains; W_q's fragments in shared memory, 3 or 4 stages made no difference.  wd warps (1, 2, 4) lie along the columns, 8 / wd along tokens;
// the token groups' dWq are joined in shared memory, in order.
constexpr int kXWarps = 8;

// x (or its codes) comes by TMA, 64 columns x 16 tokens a tile, and dq with it, into a ring of kXStages tiles that a
// warp keeps for itself: one lane copies, every lane waits on the stage's mbarrier, no other barrier.  Rows
// and columns past the end arrive as zeros.
template <bool kCodes>
constexpr int kXStages = kCodes ? 4 : 3;  // two CTAs to an SM
template <bool kCodes>
constexpr int kXTileBytes = kCodes ? 1024 : 2048;
template <bool kCodes>
constexpr int kXSmem = kXWarps * kXStages<kCodes> * (kXTileBytes<kCodes> + kDqTileBytes + 8) + 1024;

template <bool kCodes>
__global__ void __launch_bounds__(kXWarps * 32, 2)
router_x_kernel(const __grid_constant__ CUtensorMap map, const uint8_t* __restrict__ scales,
                const uint4* __restrict__ dq, const __nv_bfloat16* __restrict__ wq, int64_t M, int D, int wd,
                __nv_bfloat16* __restrict__ dx, float* __restrict__ dw_part) {
  extern __shared__ uint8_t dyn[];
  constexpr int kStages = kXStages<kCodes>;
  // [warp][stage] tiles of x, [warp][stage] tiles of dq, [warp][stage] barriers; at the end red[token group][j][wd * 64]
  uint8_t* ring = dyn + (1024 - (smem_u32(dyn) & 1023)) % 1024;  // the swizzle counts from 1024-byte boundaries
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int dw = warp % wd, tw = warp / wd, ntw = kXWarps / wd;
  const int d0 = (blockIdx.x * wd + dw) * 64, dl = d0 + 8 * g;
  uint8_t* xs = ring + warp * kStages * kXTileBytes<kCodes>;
  uint8_t* qs = ring + kXWarps * kStages * kXTileBytes<kCodes> + warp * kStages * kDqTileBytes;
  uint64_t* bars =
      reinterpret_cast<uint64_t*>(ring + kXWarps * kStages * (kXTileBytes<kCodes> + kDqTileBytes)) + warp * kStages;
  if (lane == 0) {
    for (int k = 0; k < kStages; ++k) mbar_init(bars + k, 1);
    fence_mbar_init();
  }
  uint32_t wb[8][2];
  if (dx) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + 32 * (i >> 2) + 8 * (g >> 1) + 2 * (i & 3) + (g & 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 2 * t + 8 * h;
        const uint32_t a = d < D ? (uint32_t)__bfloat16_as_ushort(wq[(int64_t)j * D + d]) : 0u;
        const uint32_t b = d < D ? (uint32_t)__bfloat16_as_ushort(wq[(int64_t)(j + 1) * D + d]) : 0u;
        wb[i][h] = a | (b << 16);
      }
    }
  }
  float acc[4][2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  const int tiles = d0 < D ? (int)((M + 15) / 16) : 0;
  const int tile0 = blockIdx.y * ntw + tw, hop = gridDim.y * ntw;
  const auto fetch = [&](int tile, int stage) {  // lane 0
    if (tile >= tiles) return;
    mbar_arrive_expect_tx(bars + stage, dw_part ? kXTileBytes<kCodes> + kDqTileBytes : kDqTileBytes);
    if (dw_part) tma_load_2d(xs + stage * kXTileBytes<kCodes>, &map, bars + stage, d0, tile * 16);
    bulk_load(qs + stage * kDqTileBytes, dq + (int64_t)tile * (kDqTileBytes / 16), kDqTileBytes, bars + stage);
  };
  uint32_t byte[4] = {127u, 127u, 127u, 127u};
  int64_t at = ((int64_t)tile0 * 16 + 2 * t) * D + dl;  // element that the next scales belong to
  const auto fetch_scales = [&](int tile) {
    if constexpr (kCodes) {
      if (dw_part && dl < D && tile < tiles) {
        const bool whole = (int64_t)tile * 16 + 16 <= M;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = (k & 1) + 8 * (k >> 1);
          if (whole || (int64_t)tile * 16 + 2 * t + r < M) byte[k] = __ldg(scales + ((at + (int64_t)r * D) >> 5));
        }
      }
      at += (int64_t)16 * hop * D;
    }
  };
  __nv_bfloat16* po = dx + ((int64_t)tile0 * 16 + g) * D + d0 + 8 * t;
  const bool out0 = d0 + 8 * t < D, out1 = d0 + 32 + 8 * t < D;

  fetch_scales(tile0);
  griddep_wait();
  if (lane == 0)
    for (int k = 0; k < kStages; ++k) fetch(tile0 + k * hop, k);
  __syncwarp();  // the barriers' initialisation
  int stage = 0, tile = tile0;
  uint32_t parity = 0;
  for (; tile < tiles; tile += hop) {
    if (!__all_sync(0xffffffffu, mbar_wait(bars + stage, parity, nullptr, 0))) break;
    const uint4* q = reinterpret_cast<const uint4*>(qs + stage * kDqTileBytes) + lane;  // the pieces, largest first
    uint4 r[4];
    if (dw_part) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = 2 * t + (k & 1) + 8 * (k >> 1);
        if constexpr (kCodes) {  // 64-byte swizzle: 16-byte piece ^ (row / 2) % 4
          const uint2 c = *reinterpret_cast<const uint2*>(xs + stage * 1024 + row * 64 + (((g >> 1) ^ t) << 4) +
                                                          (g & 1) * 8);
          const float f = mx_scale((int)byte[k]);
          const float2 a = mx_unpack2((uint16_t)c.x), b = mx_unpack2((uint16_t)(c.x >> 16));
          const float2 e = mx_unpack2((uint16_t)c.y), z = mx_unpack2((uint16_t)(c.y >> 16));
          r[k] = make_uint4(pack_bf16(a.x * f, a.y * f), pack_bf16(b.x * f, b.y * f), pack_bf16(e.x * f, e.y * f),
                            pack_bf16(z.x * f, z.y * f));
        } else {  // 128-byte swizzle: 16-byte piece ^ row % 8
          r[k] = *reinterpret_cast<const uint4*>(xs + stage * 2048 + row * 128 + ((g ^ (row & 7)) << 4));
        }
      }
    }
    fetch_scales(tile + hop);
    if (dx) {
      uint32_t a[kDqPieces][4];
#pragma unroll
      for (int k = 0; k < kDqPieces; ++k) {
        const uint4 v = q[32 * k];
        a[k][0] = transpose8x8(v.x);
        a[k][1] = transpose8x8(v.z);
        a[k][2] = transpose8x8(v.y);
        a[k][3] = transpose8x8(v.w);
      }
      const bool in_a = (int64_t)tile * 16 + g < M, in_b = (int64_t)tile * 16 + 8 + g < M;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t oa[4], ob[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float c[4];
          mma_bf16_zero(c, a[2][0], a[2][1], a[2][2], a[2][3], wb[4 * h + i][0], wb[4 * h + i][1]);
          mma_bf16(c, a[1][0], a[1][1], a[1][2], a[1][3], wb[4 * h + i][0], wb[4 * h + i][1]);
          mma_bf16(c, a[0][0], a[0][1], a[0][2], a[0][3], wb[4 * h + i][0], wb[4 * h + i][1]);
          oa[i] = pack_bf16(c[0], c[1]);
          ob[i] = pack_bf16(c[2], c[3]);
        }
        if (h ? out1 : out0) {
          if (in_a) *reinterpret_cast<uint4*>(po + 32 * h) = make_uint4(oa[0], oa[1], oa[2], oa[3]);
          if (in_b) *reinterpret_cast<uint4*>(po + 32 * h + 8 * D) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
        }
      }
      po += (int64_t)16 * hop * D;
    }
    if (dw_part) {
      uint4 dq4[kDqPieces];  // (read again: held from above, they spill)
#pragma unroll
      for (int k = 0; k < kDqPieces; ++k) dq4[k] = q[32 * k];
      const uint32_t w0[4] = {r[0].x, r[0].y, r[0].z, r[0].w}, w1[4] = {r[1].x, r[1].y, r[1].z, r[1].w};
      const uint32_t w2[4] = {r[2].x, r[2].y, r[2].z, r[2].w}, w3[4] = {r[3].x, r[3].y, r[3].z, r[3].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = __byte_perm(w0[i], w1[i], 0x5410), a1 = __byte_perm(w0[i], w1[i], 0x7632);
        const uint32_t a2 = __byte_perm(w2[i], w3[i], 0x5410), a3 = __byte_perm(w2[i], w3[i], 0x7632);
        float c[2][4];  // of this tile alone: the tensor cores round towards zero, a chain over all tiles would add that up
        mma_bf16_zero(c[0], a0, a1, a2, a3, dq4[2].x, dq4[2].z);
        mma_bf16_zero(c[1], a0, a1, a2, a3, dq4[2].y, dq4[2].w);
#pragma unroll
        for (int k = 1; k >= 0; --k) {
          mma_bf16(c[0], a0, a1, a2, a3, dq4[k].x, dq4[k].z);
          mma_bf16(c[1], a0, a1, a2, a3, dq4[k].y, dq4[k].w);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += c[j][e];
      }
    }
    __syncwarp();  // the tile is in every lane's registers: its place takes the tile kStages on
    if (lane == 0) fetch(tile + kStages * hop, stage);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (tile < tiles) {  // a copy did not arrive within the wait limit: wait once more for all, leave NaN as the result
    for (int k = 0; k < kStages; ++k) {
      if (tile + k * hop < tiles) mbar_wait(bars + stage, parity, nullptr, 0);
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __uint_as_float(0x7FC00000u);
    for (; dx && tile < tiles; tile += hop) {
      const uint32_t n = 0x7FC07FC0u;
      for (int k = 0; k < 4; ++k) {
        const int64_t row = (int64_t)tile * 16 + g + 8 * (k & 1);
        if (row < M && (k < 2 ? out0 : out1))
          *reinterpret_cast<uint4*>(dx + row * D + d0 + 8 * t + (k < 2 ? 0 : 32)) = make_uint4(n, n, n, n);
      }
    }
  }
  if (!dw_part) return;
  // acc[i][j]: column 8 g + 2 i (elements 0, 1) and + 1 (2, 3), dimension 8 j + 2 t (+1: odd element)
  const int width = wd * 64;
  float* red = reinterpret_cast<float*>(ring);
  __syncthreads();  // every warp is through with its ring
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(tw * kIdx + 8 * j + 2 * t + (e & 1)) * width + dw * 64 + 8 * g + 2 * i + (e >> 1)] = acc[i][j][e];
  __syncthreads();
  float* part = dw_part + (int64_t)blockIdx.y * kIdx * D;
  const int d = threadIdx.x % width, c = blockIdx.x * width + d;
  for (int j = threadIdx.x / width; j < kIdx; j += kXWarps * 32 / width) {
    float s = 0.f;
    for (int k = 0; k < ntw; ++k) s += red[(k * kIdx + j) * width + d];
    if (c < D) part[(int64_t)j * D + c] = s;
  }
}

// Pass 2, fp32, on the FMA units (32 per element): a thread owns 4 columns (their Wq and dWq in registers), dq (and
// the copy's scales) of 32 tokens at a time in shared memory; tx threads (32, 64, 128) lie along the columns,
// 128 / tx along tokens.  x runs through a ring of kFAhead tokens that a thread keeps for itself (cp.async).
// 16384 x 4096 took 238 us with two loads in flight from registers, 160 us with the ring (3.1 TB/s; 67 % issue at 18 %
// of the warps, of the time 58 us are FMAs: 168 registers leave three CTAs of 4 warps); paired FMAs (fma.rn.f32x2) need fewer instructions, spill, and took 175 to 194 us.
constexpr int kFThreads = 128;
constexpr int kFTokens = 32;
constexpr int kFAhead = 8;
constexpr int kFScales = kFThreads * 4 / kMxBlock + 1;  // blocks that a CTA's columns of a token may touch

__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool kCodes>
__global__ void __launch_bounds__(kFThreads, 3)
router_x_f32_kernel(const float* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                    const float* __restrict__ dq, const float* __restrict__ wq, int64_t M, int D, int tx,
                    int64_t tokens_per_cta, float* __restrict__ dx, float* __restrict__ dw_part) {
  __shared__ float4 sq[kFTokens * 4];           // [token][16] dq
  __shared__ uint8_t ss[kCodes ? kFTokens * kFScales : 1];  // [token][block] scale bytes
  __shared__ float red[kFThreads * 4 * kIdx];   // during the pass its first half is the ring [kFAhead][thread] float4
  griddep_launch_dependents();
  const int lane = threadIdx.x % tx, ty = threadIdx.x / tx, nty = kFThreads / tx;
  const int db = blockIdx.x * tx * 4, d = db + lane * 4, width = tx * 4;
  const bool in = d < D;
  float w[kIdx][4], acc[kIdx][4];
#pragma unroll
  for (int j = 0; j < kIdx; ++j) {
    const float4 v = in && dx ? __ldg(reinterpret_cast<const float4*>(wq + (int64_t)j * D + d))
                              : make_float4(0.f, 0.f, 0.f, 0.f);
    w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  }
  const int64_t t1 = min((int64_t)(blockIdx.y + 1) * tokens_per_cta, M);
  const uint32_t ring = smem_u32(red) + threadIdx.x * 16;
  // the thread's n-th token from the CTA's first: ty + n nty
  const int64_t first = (int64_t)blockIdx.y * tokens_per_cta + ty;
  const auto fetch = [&](int64_t tok, int slot) {
    if (in && dw_part && tok < t1) {
      if constexpr (kCodes) cp_async4(ring + slot * kFThreads * 16, codes + tok * D + d);
      else cp_async_16(ring + slot * kFThreads * 16, x + tok * D + d);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < kFAhead - 1; ++k) fetch(first + (int64_t)k * nty, k);
  int slot = 0;
  griddep_wait();
  for (int64_t t0 = (int64_t)blockIdx.y * tokens_per_cta; t0 < t1; t0 += kFTokens) {
    const int n = (int)min((int64_t)kFTokens, t1 - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * 4; i += kFThreads)
      sq[i] = __ldg(reinterpret_cast<const float4*>(dq + t0 * kIdx) + i);
    if constexpr (kCodes) {
      if (dw_part)
        for (int i = threadIdx.x; i < n * kFScales; i += kFThreads) {
          const int64_t row = (t0 + i / kFScales) * D, b = (row + db) / kMxBlock + i % kFScales;
          if (b * kMxBlock < row + min(D, db + width)) ss[i] = __ldg(scales + b);
        }
    }
    __syncthreads();
    if (!in) continue;
#pragma unroll 2
    for (int k = ty; k < n; k += nty) {
      const int64_t i = (t0 + k) * D + d;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      cp_async_wait<kFAhead - 2>();
      const float4* mine = reinterpret_cast<const float4*>(red) + slot * kFThreads + threadIdx.x;
      fetch(t0 + k + (int64_t)(kFAhead - 1) * nty, slot == 0 ? kFAhead - 1 : slot - 1);
      slot = slot == kFAhead - 1 ? 0 : slot + 1;
      if (dw_part) {
        if constexpr (kCodes) {
          const uint32_t c = *reinterpret_cast<const uint32_t*>(mine);
          const float s = mx_scale((int)ss[k * kFScales + (int)(i / kMxBlock - (i - lane * 4) / kMxBlock)]);
          const float2 a = mx_unpack2((uint16_t)c), b = mx_unpack2((uint16_t)(c >> 16));
          v[0] = a.x * s; v[1] = a.y * s; v[2] = b.x * s; v[3] = b.y * s;
        } else {
          const float4 q = *mine;
          v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        }
      }
      float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const float4 q4 = sq[k * 4 + jj];
        const float q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[4 * jj + j][e] = fmaf(q[j], v[e], acc[4 * jj + j][e]);
            o[e] = fmaf(q[j], w[4 * jj + j][e], o[e]);
          }
      }
      if (dx) *reinterpret_cast<float4*>(dx + i) = make_float4(o[0], o[1], o[2], o[3]);
    }
  }
  cp_async_wait<0>();
  if (!dw_part) return;
  __syncthreads();  // the ring's place takes the sums
#pragma unroll
  for (int j = 0; j < kIdx; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[(ty * kIdx + j) * width + lane * 4 + e] = acc[j][e];
  __syncthreads();
  float* part = dw_part + (int64_t)blockIdx.y * kIdx * D;
  for (int c = threadIdx.x; c < width; c += kFThreads)
    for (int j = 0; j < kIdx; ++j) {
      float s = 0.f;
      for (int k = 0; k < nty; ++k) s += red[(k * kIdx + j) * width + c];
      if (db + c < D) part[(int64_t)j * D + db + c] = s;
    }
}

// Pass 3: out[i] = sum over the partials, 8 interleaved sums joined in order; dWq (n1 elements), then dK (n2).
template <typename T>
__global__ void __launch_bounds__(256)
sum_partials_kernel(const float* __restrict__ p1, int parts1, int64_t n1, T* __restrict__ o1,
                    const float* __restrict__ p2, int parts2, int64_t n2, T* __restrict__ o2) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t blocks1 = (n1 + 31) / 32;
  const bool first = blockIdx.x < blocks1;
  const float* p = first ? p1 : p2;
  const int64_t n = first ? n1 : n2, i = (first ? blockIdx.x : blockIdx.x - blocks1) * 32 + lane;
  const int parts = first ? parts1 : parts2;
  griddep_wait();
  float v = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int k = row; k < parts; k += 8) v += p[k * n + i];
  }
  s[row][lane] = v;
  __syncthreads();
  if (row == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += s[k][lane];
    (first ? o1 : o2)[i] = mx_from_f32<T>(v);
  }
}

// Launch shapes and workspace of the three passes: about two CTAs of pass 2 to an SM (three for fp32), and no
// more partial sums than that.
// Rows of codes that TMA cannot address (D % 16 != 0, bf16) go through pass 2 as bf16 in pieces: of 64 MB, which stay
// in L2 between the two kernels, or of a sixteenth of the rows, an eighth of the codes, where that is more.  Against
// all rows at once (2 bytes an element of workspace): 65536 x 1000 183 -> 160 us, 65536 x 4104 419 -> 477 us (with
// pieces of 32 MB 560 us).
constexpr int64_t kCopyBytes = 64 << 20;
struct BwdPlan {
  int dq_ctas, wide, col_ctas, parts, pieces;
  int64_t per_cta;     // pass 2: tiles of 16 tokens (bf16) or tokens (fp32)
  int64_t piece_rows;  // M unless the rows go in pieces
  size_t dq, dw, dk, copy, total;
};
BwdPlan bwd_plan(int dtype, int64_t M, int D, int NB, bool from_codes) {
  BwdPlan p{};
  p.dq_ctas = (int)std::min<int64_t>((M + kDqTokens - 1) / kDqTokens, kDqMaxCtas);
  const bool copied = from_codes && dtype == FP_DTYPE_BF16 && D % 16;
  p.piece_rows = M;
  if (copied) p.piece_rows = std::min(M, (std::max((kCopyBytes / 2 + D - 1) / D, (M + 15) / 16) + 15) / 16 * 16);
  p.pieces = (int)((M + p.piece_rows - 1) / p.piece_rows);
  int64_t units;
  if (dtype == FP_DTYPE_BF16) {
    p.wide = D <= 64 ? 1 : D <= 128 ? 2 : 4;
    p.col_ctas = (D + 64 * p.wide - 1) / (64 * p.wide);
    units = (p.piece_rows + 15) / 16;
    p.per_cta = std::max<int64_t>((units + std::max(296 / p.col_ctas, 1) - 1) / std::max(296 / p.col_ctas, 1),
                                  2 * kXWarps / p.wide);
  } else {
    p.wide = D <= 128 ? 32 : D <= 256 ? 64 : 128;
    p.col_ctas = (D + 4 * p.wide - 1) / (4 * p.wide);
    units = M;
    const int64_t want = std::max(444 / p.col_ctas, 1);
    p.per_cta = std::max<int64_t>((units + want - 1) / want, kFTokens);
  }
  p.parts = (int)((units + p.per_cta - 1) / p.per_cta);
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  p.dq = 0;
  p.dw = p.dq + up((size_t)((M + 15) / 16) * (dtype == FP_DTYPE_BF16 ? kDqTileBytes : 16 * kIdx * 4));
  p.dk = p.dw + up((size_t)p.parts * p.pieces * kIdx * D * 4);
  p.copy = p.dk + up((size_t)p.dq_ctas * kIdx * NB * 4);
  p.total = p.copy + (copied ? up((size_t)p.piece_rows * D * 2) : 0);
  return p;
}

template <typename T, bool kVec>
int launch_dq(const BwdPlan& p, const float* ds, const T* k16, const float* q16, const float* rnorm, int64_t M, int NB,
              void* dq, float* pk, cudaStream_t st) {
  constexpr auto kern = router_dq_kernel<T, sizeof(T) == 2, kVec>;
  const size_t smem = dq ? (size_t)((NB + 15) / 16) * 1024 : 0;  // at most 64 KB
  if (smem > 48 * 1024 && !allow_smem<kern>(64 * 1024)) return FP_ERR_CUDA;
  const int rows = (dq ? 1 : 0) + (pk ? (NB + 32 * kDqWarps - 1) / (32 * kDqWarps) : 0);
  if (rows == 0) return FP_OK;
  kern<<<dim3(p.dq_ctas, rows), kDqWarps * 32, smem, st>>>(ds, k16, q16, rnorm, M, NB, dq, pk);
  return launched();
}

template <typename T>
int router_bwd(const float* ds, const T* x, const uint8_t* codes, const uint8_t* scales, const T* wq, const T* k16,
               const float* q16, const float* rnorm, int64_t M, int D, int NB, T* dx, void* dwq, void* dk16,
               int grad_dtype, char* ws, cudaStream_t st) {
  const BwdPlan p = bwd_plan(sizeof(T) == 2 ? FP_DTYPE_BF16 : FP_DTYPE_F32, M, D, NB, codes != nullptr);
  void* dq = dx || dwq ? ws + p.dq : nullptr;
  float* pw = dwq ? reinterpret_cast<float*>(ws + p.dw) : nullptr;
  float* pk = dk16 ? reinterpret_cast<float*>(ws + p.dk) : nullptr;
  if (const int rc = NB % 4 == 0 ? launch_dq<T, true>(p, ds, k16, q16, rnorm, M, NB, dq, pk, st)
                                 : launch_dq<T, false>(p, ds, k16, q16, rnorm, M, NB, dq, pk, st))
    return rc;
  int parts = p.parts;
  if (dq) {
    const dim3 grid(p.col_ctas, p.parts);
    if constexpr (sizeof(T) == 2) {
      static_assert(kXSmem<true> >= kXWarps * 64 * kIdx * 4 + 1024, "the ring's place takes the sums");
      const bool copied = codes && D % 16;
      // without dWq nothing reads the rows, and one launch takes them all
      const int64_t step = copied && dwq ? p.piece_rows : M;
      const bool from_codes = codes && !copied;
      const auto kern = from_codes ? router_x_kernel<true> : router_x_kernel<false>;
      const int smem = from_codes ? kXSmem<true> : kXSmem<false>;
      if (!(from_codes ? allow_smem<router_x_kernel<true>>(smem) : allow_smem<router_x_kernel<false>>(smem)))
        return FP_ERR_CUDA;
      parts = 0;
      for (int64_t r0 = 0; r0 < M; r0 += step, parts += p.parts) {
        const int64_t n = std::min(step, M - r0);  // r0 is a multiple of 16 tokens, r0 D one of 128 elements
        const __nv_bfloat16* rows = x;
        if (copied && dwq) {
          rows = reinterpret_cast<const __nv_bfloat16*>(ws + p.copy);
          if (const int rc = fp_mxfp8_dequantize(codes + r0 * D, scales + r0 * D / kMxBlock, FP_DTYPE_BF16, n * D,
                                                 ws + p.copy, st))
            return rc;
        }
        CUtensorMap map{};
        if (dwq && !(from_codes ? encode_map_2d_u8(&map, codes, D, n, D, 64, 16)
                                : encode_map_2d(&map, rows, D, n, (uint64_t)D * 2, 64, 16)))
          return FP_ERR_CUDA;
        const uint4* dqt = reinterpret_cast<const uint4*>((const char*)dq + r0 / 16 * kDqTileBytes);
        if (launch_pdl(kern, grid, kXWarps * 32, smem, st, map, scales, dqt, wq, n, D, p.wide,
                       dx ? dx + r0 * D : nullptr, pw ? pw + (int64_t)parts * kIdx * D : nullptr) != cudaSuccess)
          return FP_ERR_CUDA;
      }
    } else if (launch_pdl(codes ? router_x_f32_kernel<true> : router_x_f32_kernel<false>, grid, kFThreads, 0, st, x,
                          codes, scales, (const float*)dq, wq, M, D, p.wide, p.per_cta, dx, pw) != cudaSuccess) {
      return FP_ERR_CUDA;
    }
  }
  if (dwq || dk16) {
    const int64_t n1 = dwq ? (int64_t)kIdx * D : 0, n2 = dk16 ? (int64_t)kIdx * NB : 0;
    const unsigned grid = (unsigned)((n1 + 31) / 32 + (n2 + 31) / 32);
    cudaError_t e;
    if (grad_dtype == FP_DTYPE_BF16)
      e = launch_pdl(sum_partials_kernel<__nv_bfloat16>, grid, 256, 0, st, pw, parts, n1, (__nv_bfloat16*)dwq, pk,
                     p.dq_ctas, n2, (__nv_bfloat16*)dk16);
    else
      e = launch_pdl(sum_partials_kernel<float>, grid, 256, 0, st, pw, parts, n1, (float*)dwq, pk, p.dq_ctas, n2,
                     (float*)dk16);
    if (e != cudaSuccess) return FP_ERR_CUDA;
  }
  return launched();
}

// ------------------------------------------------------------------ balance loss
// A warp takes kR rows at a time, each row's scores in its registers (kE to a lane), with all of the rows'
// loads issued before the first use.  What bounds the passes is the instructions of a row (about 230 forward
// with its list, 240 backward at 448 blocks) and, below some 10^4 rows, latency and the number of partial sums
// that the join has to read: CTAs in clusters of 8 add their column sums through distributed shared memory.
// 256 CTAs, not two to each of 148 SMs: 37 clusters of 8 are not resident at once, and the last ones ran alone
// (65521 x 448: forward 70 us with 296 CTAs, 51 us with 256; clusters of 4: 76 us with 288, 55 us with 256).
constexpr int kBalWarps = 16;
constexpr int kBalCluster = 8;
constexpr int kBalMaxCtas = 256;
constexpr int kGradWarps = 8;
// Temperatures: beyond these log2(e) / T or R / (T n) overflows or vanishes in 32 bits, and 0 * inf is NaN.
constexpr bool bal_temperature(float t) { return t >= 1e-30f && t <= 1e30f; }
// A list's longest form.  A cluster's slot count of one block has 32 bits: rows of one name only, 2^20 of them to
// a row, pass it with 2^31 entries to a cluster, 2^36 in all (256 GB).
constexpr int kBalMaxCapacity = 1 << 20;

template <int kE>
constexpr int kRowsOf = kE <= 4 ? 4 : kE == 8 ? 2 : 1;

// Column of a lane's i-th score: quads of columns where rows are 16-byte aligned (kVec), else single ones.
template <bool kVec>
__device__ __forceinline__ int bal_col(int lane, int i) {
  return kVec ? 4 * lane + 128 * (i >> 2) + (i & 3) : lane + 32 * i;
}
template <int kE, bool kVec>
__device__ __forceinline__ void bal_load(const float* __restrict__ row, int NB, int lane, float (&z)[kE]) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kE / 4; ++i) {
      const int b = 4 * lane + 128 * i;
      const float4 v = b < NB ? __ldg(reinterpret_cast<const float4*>(row + b))
                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      z[4 * i] = v.x; z[4 * i + 1] = v.y; z[4 * i + 2] = v.z; z[4 * i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i) z[i] = lane + 32 * i < NB ? __ldg(row + lane + 32 * i) : -INFINITY;
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Largest value over the warp; a NaN loses.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Scores (-inf past the row's end) to exp((z - max) / T) over the remote blocks, 0 for the base blocks; `sum` is
// the lane's part of their sum.  Returns whether the row is counted: a row whose remote scores are all -inf
// has no distribution and is not; a NaN makes the whole row NaN.  c = log2(e) / T.  The passes are issue bound
// at 448 blocks (24 instructions a score before, about 7 now), hence one fused multiply-add and the hardware
// exponential per score: 2^-22 of p, next to the rounding of z c (|z| c 2^-24).  The rounding of `d` is the same for
// a whole row and leaves p as it is, but it shifts the exponents by up to |d| 2^-24: from |d| = 2^20 on (a row of
// -1e30 as a mask, a temperature near 0) the difference to the largest score is taken first.
template <int kE, bool kVec>
__device__ __forceinline__ bool bal_exp(float (&z)[kE], int base, float c, int lane, float& sum) {
  constexpr int kHead = kVec ? 4 : 4 < kE ? 4 : kE;  // elements in a lane's first 128 columns
#pragma unroll
  for (int i = 0; i < kHead; ++i)
    if (bal_col<kVec>(lane, i) < base) z[i] = -INFINITY;
  if (base > 128) {
#pragma unroll
    for (int i = kHead; i < kE; ++i)
      if (bal_col<kVec>(lane, i) < base) z[i] = -INFINITY;
  }
  float top = z[0];
#pragma unroll
  for (int i = 1; i < kE; ++i) top = fmaxf(top, z[i]);
  top = warp_max(top);
  const float d = -top * c;
  sum = 0.f;
  if (fabsf(d) <= 0x1p20f) {
#pragma unroll
    for (int i = 0; i < kE; ++i) z[i] = exp2_fast(fmaf(z[i], c, d));
  } else {  // large scores, an infinity, a NaN, or nothing above -inf
    if (top == -INFINITY) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < kE; ++i) nan |= z[i] != z[i];
      if (!__any_sync(0xffffffffu, nan)) return false;
      top = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kE; ++i) z[i] = exp2_fast((z[i] - top) * c);
  }
#pragma unroll
  for (int i = 0; i < kE; ++i) sum += z[i];
  return true;
}

// Per cluster: column sums of p over its rows, the number of counted rows, and the blocks' slot counts.
// scores may be NULL (counts only); idx may be NULL (counts given).
//
// Counting: a row's list sets one byte per block in the warp's own shared memory; each lane adds the four columns
// of its words to byte counters in registers (spilled to the CTA's counts before they can pass 255) and clears
// them.  A list that names a block twice is noticed by its sum and counted with atomics.  With an atomic for
// every entry the counts alone took 89 us at 65521 rows of up to 112, this way 49 (296 CTAs both; now 35).
template <int kE, bool kVec>
__global__ void __cluster_dims__(kBalCluster, 1, 1) __launch_bounds__(kBalWarps * 32, kE <= 16 ? 2 : 1)
balance_partial_kernel(const float* __restrict__ scores, int64_t M, int NB, int base, float temperature,
                       const uint8_t* __restrict__ valid, const int32_t* __restrict__ idx,
                       const int32_t* __restrict__ cnt, int capacity, float* __restrict__ psum,
                       int32_t* __restrict__ rows, int32_t* __restrict__ hist) {
  constexpr int kR = kRowsOf<kE>;
  constexpr int kW = kE < 4 ? 1 : kE / 4;    // words of four byte counters in a lane
  constexpr int kL = kE <= 2 ? 2 : 4;        // list entries of a row that a lane loads ahead
  // [NB] column sums, [NB] slot counts, [kBalWarps][NB] the warps' sums, of which each warp uses its first NB
  // bytes as its flags before the sums are written
  extern __shared__ float sm[];
  int* sh = reinterpret_cast<int*>(sm + NB);
  float* sw = sm + 2 * NB;
  __shared__ int s_rows;
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < NB; i += blockDim.x) sh[i] = 0;
  if (threadIdx.x == 0) s_rows = 0;
  uint8_t* flags = reinterpret_cast<uint8_t*>(sw + warp * NB);
  uint32_t* flag4 = reinterpret_cast<uint32_t*>(flags);
#pragma unroll
  for (int i = 0; i < kW; ++i)
    if (4 * lane + 128 * i < NB) flag4[lane + 32 * i] = 0;
  __syncthreads();
  float acc[kE];
#pragma unroll
  for (int i = 0; i < kE; ++i) acc[i] = 0.f;
  uint32_t slots[kW] = {};
  int pending = 0, counted = 0;
  const float c = __fdiv_rn(1.4426950408889634f, temperature);
  const int64_t step = (int64_t)gridDim.x * kBalWarps;
  const bool lists = idx != nullptr;
  for (int64_t t0 = (int64_t)blockIdx.x * kBalWarps + warp;; t0 += step * kR) {
    const bool last = t0 >= M;
    if (pending > 255 - kR || last) {  // byte counters to the CTA's counts
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        for (int k = 0; k < 4; ++k) {
          const int n = (int)(slots[i] >> (8 * k) & 0xFF);
          if (n) atomicAdd(&sh[4 * lane + 128 * i + k], n);
        }
        slots[i] = 0;
      }
      pending = 0;
      if (last) break;
    }
    float z[kR][kE];
    bool on[kR];
    int n[kR], id[kR][kL];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int64_t t = t0 + r * step;
      on[r] = t < M;
      if (scores && on[r]) bal_load<kE, kVec>(scores + t * NB, NB, lane, z[r]);
      n[r] = 0;
      if (lists && on[r]) {
        n[r] = min(__ldg(cnt + t), capacity);
        const int32_t* list = idx + t * capacity + lane;
#pragma unroll
        for (int k = 0; k < kL; ++k) id[r][k] = lane + 32 * k < capacity ? __ldg(list + 32 * k) : -1;
      }
      if (valid && on[r]) on[r] = __ldg(valid + t) != 0;
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (!on[r]) continue;
      if (n[r] > 0) {
        const int32_t* list = idx + (t0 + r * step) * capacity;
        int named = 0;
#pragma unroll
        for (int k = 0; k < kL; ++k)
          if (lane + 32 * k < n[r] && (unsigned)id[r][k] < (unsigned)NB) {
            flags[id[r][k]] = 1;
            ++named;
          }
        for (int k = lane + 32 * kL; k < n[r]; k += 32) {
          const int b = __ldg(list + k);
          if ((unsigned)b < (unsigned)NB) {
            flags[b] = 1;
            ++named;
          }
        }
        __syncwarp();
        uint32_t f[kW];
#pragma unroll
        for (int i = 0; i < kW; ++i) {
          f[i] = 0;
          if (4 * lane + 128 * i < NB) {
            f[i] = flag4[lane + 32 * i];
            flag4[lane + 32 * i] = 0;
            named -= __popc(f[i]);
          }
        }
        __syncwarp();
        if (__reduce_add_sync(0xffffffffu, named) == 0) {
          ++pending;
#pragma unroll
          for (int i = 0; i < kW; ++i) slots[i] += f[i];
        } else {
          for (int k = lane; k < n[r]; k += 32) {
            const int b = __ldg(list + k);
            if ((unsigned)b < (unsigned)NB) atomicAdd(&sh[b], 1);
          }
        }
      }
      float sum;
      if (scores && bal_exp<kE, kVec>(z[r], base, c, lane, sum)) {
        ++counted;
        const float inv = rcp_fast(warp_sum(sum));
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[i] = fmaf(z[r][i], inv, acc[i]);
      }
    }
  }
  __syncwarp();  // the flags' place now takes the sums
#pragma unroll
  for (int i = 0; i < kE; ++i)
    if (bal_col<kVec>(lane, i) < NB) sw[warp * NB + bal_col<kVec>(lane, i)] = acc[i];
  if (lane == 0) atomicAdd(&s_rows, counted);
  __syncthreads();
  for (int b = threadIdx.x; b < NB; b += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kBalWarps; ++w) s += sw[w * NB + b];
    sm[b] = s;
  }
  cluster_sync();
  const int rank = (int)cluster_ctarank(), part = blockIdx.x / kBalCluster;
  for (int b = rank + kBalCluster * threadIdx.x; b < NB; b += kBalCluster * blockDim.x) {
    float s = 0.f;
    int c = 0;
#pragma unroll
    for (int k = 0; k < kBalCluster; ++k) {
      s += ld_cluster_f32(sm + b, k);
      c += __float_as_int(ld_cluster_f32(reinterpret_cast<const float*>(sh + b), k));
    }
    psum[(int64_t)part * NB + b] = s;
    hist[(int64_t)part * NB + b] = c;
  }
  if (threadIdx.x == 0) rows[blockIdx.x] = s_rows;
  cluster_sync();  // no CTA leaves while another reads its shared memory
}

// One CTA of 1024 threads, `width` (a power of two >= NB) columns by 1024 / width groups of the partials: joins
// them in their order, writes the counts, the loss and what the gradient needs: state[b] = f_b - 1/R (0 when
// nothing was routed) and state[NB] = R / (T n).
__global__ void __launch_bounds__(1024)
balance_join_kernel(const float* __restrict__ psum, const int32_t* __restrict__ rows,
                    const int32_t* __restrict__ hist, int ctas, int NB, int width, int base, float temperature,
                    const int64_t* __restrict__ counts_in, int64_t* __restrict__ counts, float* __restrict__ loss,
                    float* __restrict__ state) {
  __shared__ double s_p[1024];
  __shared__ long long s_c[1024];
  __shared__ double s_loss[32];
  __shared__ long long s_tot[32];
  __shared__ int s_rows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = tid & (width - 1), grp = tid / width, groups = 1024 / width, parts = ctas / kBalCluster;
  if (tid == 0) s_rows = 0;
  griddep_wait();
  __syncthreads();
  int64_t c = 0;
  double ps = 0.0;
  if (b < NB) {
#pragma unroll 8
    for (int i = grp; i < parts; i += groups) {
      if (!counts_in) c += hist[(int64_t)i * NB + b];
      ps += (double)psum[(int64_t)i * NB + b];
    }
  }
  if (tid < ctas) atomicAdd(&s_rows, rows[tid]);
  s_p[tid] = ps;
  s_c[tid] = c;
  __syncthreads();
  if (grp == 0) {
    for (int k = 1; k < groups; ++k) {
      ps += s_p[b + k * width];
      c += s_c[b + k * width];
    }
    if (b < NB) {
      if (counts_in) c = counts_in[b];
      if (counts) counts[b] = c;
    }
  } else {
    c = 0;
  }
  if (!loss) return;
  int64_t tot = c;
  for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
  if (lane == 0) s_tot[warp] = tot;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < 32; ++w) total += s_tot[w];
  const int R = NB - base, n = s_rows;
  const bool remote = grp == 0 && b >= base && b < NB;
  double part = remote && total > 0 ? (double)c / (double)total * ps : 0.0;
  for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if (lane == 0) s_loss[warp] = part;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < 32; ++w) s += s_loss[w];
    *loss = n > 0 ? (float)(s * R / (double)n) : 0.f;
    state[NB] = n > 0 ? (float)((double)R / ((double)temperature * (double)n)) : 0.f;
  }
  if (grp == 0 && b < NB)
    state[b] = total > 0 && remote ? (float)(fma((double)c, (double)R, -(double)total) / ((double)total * R)) : 0.f;
}

template <int kE, bool kVec>
__global__ void __launch_bounds__(kGradWarps * 32)
balance_grad_kernel(const float* __restrict__ scores, int64_t M, int NB, int base, float temperature,
                    const uint8_t* __restrict__ valid, const float* __restrict__ state,
                    const float* __restrict__ dloss, float* __restrict__ ds) {
  constexpr int kR = kRowsOf<kE>;
  constexpr int kHead = kVec ? 4 : 4 < kE ? 4 : kE;
  const int lane = threadIdx.x & 31;
  const float scale = state[NB] * *dloss;
  const float c = __fdiv_rn(1.4426950408889634f, temperature);
  float f[kE];
#pragma unroll
  for (int i = 0; i < kE; ++i) f[i] = bal_col<kVec>(lane, i) < NB ? state[bal_col<kVec>(lane, i)] : 0.f;
  const int64_t step = (int64_t)gridDim.x * kGradWarps;
  for (int64_t t0 = (int64_t)blockIdx.x * kGradWarps + (threadIdx.x >> 5); t0 < M; t0 += step * kR) {
    float p[kR][kE];
    bool on[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int64_t t = t0 + r * step;
      on[r] = t < M;
      if (on[r]) bal_load<kE, kVec>(scores + t * NB, NB, lane, p[r]);
      if (on[r] && valid) on[r] = __ldg(valid + t) != 0;
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int64_t t = t0 + r * step;
      if (t >= M) break;
      float sum;
      const bool counted = on[r] && bal_exp<kE, kVec>(p[r], base, c, lane, sum);
      if (counted) {
        float inner = 0.f;
#pragma unroll
        for (int i = 0; i < kE; ++i) inner = fmaf(p[r][i], f[i], inner);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
          inner += __shfl_xor_sync(0xffffffffu, inner, o);
        }
        const float inv = rcp_fast(sum), k = scale * inv, m = -inner * inv * k;
#pragma unroll
        for (int i = 0; i < kE; ++i) p[r][i] *= fmaf(f[i], k, m);
#pragma unroll
        for (int i = 0; i < kHead; ++i)
          if (bal_col<kVec>(lane, i) < base) p[r][i] = 0.f;  // also in a NaN row
        if (base > 128) {
#pragma unroll
          for (int i = kHead; i < kE; ++i)
            if (bal_col<kVec>(lane, i) < base) p[r][i] = 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) p[r][i] = 0.f;
      }
      float* o = ds + t * NB;
      if constexpr (kVec) {
#pragma unroll
        for (int i = 0; i < kE / 4; ++i)
          if (4 * lane + 128 * i < NB)
            *reinterpret_cast<float4*>(o + 4 * lane + 128 * i) =
                make_float4(p[r][4 * i], p[r][4 * i + 1], p[r][4 * i + 2], p[r][4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (lane + 32 * i < NB) o[lane + 32 * i] = p[r][i];
      }
    }
  }
}

int balance_ctas(int64_t M) {
  const int64_t want = (M + kBalWarps * 2 - 1) / (kBalWarps * 2);  // two rows to a warp
  const int64_t up = (want + kBalCluster - 1) / kBalCluster * kBalCluster;
  return (int)std::max<int64_t>(kBalCluster, std::min<int64_t>(up, kBalMaxCtas));
}

template <int kE, bool kVec>
int balance_fwd_go(const float* scores, int64_t M, int NB, int base, float temperature, const uint8_t* valid,
                   const int32_t* idx, const int32_t* cnt, int capacity, float* psum, int32_t* rows, int32_t* hist,
                   cudaStream_t st) {
  constexpr auto kern = balance_partial_kernel<kE, kVec>;
  const size_t smem = (size_t)(kBalWarps + 2) * NB * 4;  // at most 72 KB
  if (smem > 48 * 1024 && !allow_smem<kern>(72 * 1024)) return FP_ERR_CUDA;
  kern<<<balance_ctas(M), kBalWarps * 32, smem, st>>>(scores, M, NB, base, temperature, valid, idx, cnt, capacity,
                                                      psum, rows, hist);
  return launched();
}

template <int kE, bool kVec>
int balance_bwd_go(const float* scores, int64_t M, int NB, int base, float temperature, const uint8_t* valid,
                   const float* state, const float* dloss, float* ds, int sms, cudaStream_t st) {
  const int64_t rows = (int64_t)kGradWarps * kRowsOf<kE>;
  const int grid = (int)std::min<int64_t>((M + rows - 1) / rows, (int64_t)sms * 8);
  balance_grad_kernel<kE, kVec><<<grid, kGradWarps * 32, 0, st>>>(scores, M, NB, base, temperature, valid, state, dloss,
                                                                 ds);
  return launched();
}

}  // namespace
}  // namespace fp

using namespace fp;

// CALL with kE scores to a lane and kVec for the row width NB; rows are read in quads where they are 16-byte
// aligned and wide enough to fill half a warp's.
#define FP_BY_WIDTH(NB, ALIGNED, CALL)                                              \
  do {                                                                              \
    if ((ALIGNED) && (NB) % 4 == 0 && (NB) > 64) {                                  \
      constexpr bool kVec = true;                                                   \
      if ((NB) <= 128) { constexpr int kE = 4; CALL; }                              \
      else if ((NB) <= 256) { constexpr int kE = 8; CALL; }                         \
      else if ((NB) <= 512) { constexpr int kE = 16; CALL; }                        \
      else { constexpr int kE = 32; CALL; }                                         \
    } else {                                                                        \
      constexpr bool kVec = false;                                                  \
      if ((NB) <= 32) { constexpr int kE = 1; CALL; }                               \
      else if ((NB) <= 64) { constexpr int kE = 2; CALL; }                          \
      else if ((NB) <= 128) { constexpr int kE = 4; CALL; }                         \
      else if ((NB) <= 256) { constexpr int kE = 8; CALL; }                         \
      else if ((NB) <= 512) { constexpr int kE = 16; CALL; }                        \
      else { constexpr int kE = 32; CALL; }                                         \
    }                                                                               \
  } while (0)

extern "C" {

int fp_router_scores_train(const void* x, const void* q_proj, const void* block_keys, int dtype, int64_t M, int D,
                           int NB, float* scores, float* q16, float* rnorm, void* codes, void* scales, void* stream) {
  if (dtype != FP_DTYPE_F32 && dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (M < 0 || D <= 0 || NB <= 0) return FP_ERR_INVALID_ARG;
  if (D % 8 != 0 || D > kMaxWidth || NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if ((codes == nullptr) != (scales == nullptr)) return FP_ERR_INVALID_ARG;
  if (M == 0) return FP_OK;
  if (!x || !q_proj || !block_keys || !scores || !q16 || !rnorm) return FP_ERR_INVALID_ARG;
  if (!al16(x) || !al16(q_proj) || !al16(codes)) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == FP_DTYPE_BF16 && D % 256 == 0)
    return codes ? launch_router_fwd<true>(x, q_proj, block_keys, M, D, NB, scores, q16, rnorm, codes, scales, sms, st)
                 : launch_router_fwd<false>(x, q_proj, block_keys, M, D, NB, scores, q16, rnorm, codes, scales, sms, st);
  if (const int rc = dtype == FP_DTYPE_BF16
                         ? launch_router_fwd_any<__nv_bfloat16>(x, q_proj, block_keys, M, D, NB, scores, q16, rnorm, sms, st)
                         : launch_router_fwd_any<float>(x, q_proj, block_keys, M, D, NB, scores, q16, rnorm, sms, st))
    return rc;
  return codes ? fp_mxfp8_quantize(x, dtype, M * D, codes, scales, stream) : FP_OK;
}

size_t fp_router_scores_bwd_workspace_size(int dtype, int64_t M, int D, int NB, int from_codes) {
  return M > 0 && D > 0 && NB > 0 ? bwd_plan(dtype, M, D, NB, from_codes != 0).total : 256;
}

int fp_router_scores_bwd(const float* dscores, const void* x, const void* codes, const void* scales,
                         const void* q_proj, const void* block_keys, const float* q16, const float* rnorm, int dtype,
                         int64_t M, int D, int NB, void* dx, void* dq_proj, void* dblock_keys, int grad_dtype,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != FP_DTYPE_F32 && dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (grad_dtype != FP_DTYPE_F32 && grad_dtype != FP_DTYPE_BF16) return FP_ERR_UNSUPPORTED;
  if (M <= 0 || D <= 0 || NB <= 0) return FP_ERR_INVALID_ARG;
  if (D % 8 != 0 || D > kMaxWidth || NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if (!dscores || !q_proj || !block_keys || !q16 || !rnorm || !workspace) return FP_ERR_INVALID_ARG;
  if (dq_proj && !x && !codes) return FP_ERR_INVALID_ARG;
  if ((codes == nullptr) != (scales == nullptr)) return FP_ERR_INVALID_ARG;
  if (!al16(x) || !al16(codes) || !al16(q_proj) || !al16(block_keys) || !al16(dx) || !al16(dscores) || !al16(q16) ||
      !al16(workspace))
    return FP_ERR_INVALID_ARG;
  if (workspace_bytes < bwd_plan(dtype, M, D, NB, codes != nullptr).total) return FP_ERR_WORKSPACE;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  if (dtype == FP_DTYPE_BF16)
    return router_bwd(dscores, (const __nv_bfloat16*)x, (const uint8_t*)codes, (const uint8_t*)scales,
                      (const __nv_bfloat16*)q_proj, (const __nv_bfloat16*)block_keys, q16, rnorm, M, D, NB,
                      (__nv_bfloat16*)dx, dq_proj, dblock_keys, grad_dtype, ws, st);
  return router_bwd(dscores, (const float*)x, (const uint8_t*)codes, (const uint8_t*)scales, (const float*)q_proj,
                    (const float*)block_keys, q16, rnorm, M, D, NB, (float*)dx, dq_proj, dblock_keys, grad_dtype, ws,
                    st);
}

size_t fp_balance_workspace_size(int64_t M, int NB) {
  return M >= 0 && NB > 0 ? (size_t)balance_ctas(M) * ((size_t)NB + 4) + 256 : 256;
}

int fp_balance_loss_fwd(const float* scores, int64_t M, int NB, int base_blocks, float temperature,
                        const uint8_t* valid, const int32_t* remote_indices, const int32_t* remote_counts,
                        int capacity, const int64_t* counts_in, int64_t* counts, float* loss, float* state,
                        void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || NB <= 0 || base_blocks < 0 || capacity < 0) return FP_ERR_INVALID_ARG;
  if (NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if ((remote_indices == nullptr) != (remote_counts == nullptr)) return FP_ERR_INVALID_ARG;
  if ((loss == nullptr) != (state == nullptr)) return FP_ERR_INVALID_ARG;
  if (capacity > kBalMaxCapacity) return FP_ERR_UNSUPPORTED;
  if (loss && ((M > 0 && !scores) || base_blocks >= NB || !bal_temperature(temperature))) return FP_ERR_INVALID_ARG;
  if (!loss && !counts) return FP_ERR_INVALID_ARG;
  if (M > 0 && !remote_indices && !counts_in) return FP_ERR_INVALID_ARG;
  if (!workspace || !al16(workspace)) return FP_ERR_INVALID_ARG;
  if (workspace_bytes < fp_balance_workspace_size(M, NB)) return FP_ERR_WORKSPACE;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const int ctas = balance_ctas(M), parts = ctas / kBalCluster;
  float* psum = (float*)workspace;
  int32_t* hist = (int32_t*)(psum + (size_t)parts * NB);
  int32_t* rows = hist + (size_t)parts * NB;
  const int32_t* idx = counts_in ? nullptr : remote_indices;
  const float* s = loss ? scores : nullptr;
  int rc = FP_OK;
  FP_BY_WIDTH(NB, al16(scores), (rc = balance_fwd_go<kE, kVec>(s, M, NB, base_blocks, temperature, valid, idx, remote_counts,
                                                              capacity, psum, rows, hist, st)));
  if (rc) return rc;
  int width = 32;
  while (width < NB) width *= 2;
  if (launch_pdl(balance_join_kernel, dim3(1), dim3(1024), 0, st, psum, rows, hist, ctas, NB, width, base_blocks,
                 temperature, counts_in, counts, loss, state) != cudaSuccess)
    return FP_ERR_CUDA;
  return launched();
}

int fp_balance_loss_bwd(const float* scores, int64_t M, int NB, int base_blocks, float temperature,
                        const uint8_t* valid, const float* state, const float* dloss, float* dscores, void* stream) {
  if (M < 0 || NB <= 0 || base_blocks < 0 || base_blocks >= NB || !bal_temperature(temperature))
    return FP_ERR_INVALID_ARG;
  if (NB > 1024 || M > (int64_t)INT32_MAX / 8) return FP_ERR_UNSUPPORTED;
  if (M == 0) return FP_OK;
  if (!scores || !state || !dloss || !dscores) return FP_ERR_INVALID_ARG;
  int sms;
  if (const int rc = device_info(sms)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = FP_OK;
  FP_BY_WIDTH(NB, al16(scores) && al16(dscores), (rc = balance_bwd_go<kE, kVec>(scores, M, NB, base_blocks, temperature, valid,
                                                                               state, dloss, dscores, sms, st)));
  return rc;
}

}  // extern "C"
