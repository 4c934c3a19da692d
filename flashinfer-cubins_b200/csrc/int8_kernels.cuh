// The 8-bit-integer operators: products of INT8 codes with an FP32 scale for each token and each
// output channel, the per-token quantiser that makes such codes, and the norms around a block.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "sm100_ptx.cuh"

namespace nvfp4 {

// ---------------------------------------------------------------------------
// Element types
// ---------------------------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------------------
// Codes and scales of a row
// ---------------------------------------------------------------------------

// A row's magnitudes are compared as integers: the bits of |x| order like |x|, and an infinity
// or NaN is larger than every finite value, so one maximum finds both.
__device__ __forceinline__ uint32_t magnitude_bits(float v) {
  return __float_as_uint(v) & 0x7FFFFFFFu;
}

// What a row is divided by: its largest magnitude over 127, rounded once. A row that holds an
// infinity or a NaN gets that as its scale (and codes of zero), so that products of it are NaN.
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
  return __fdiv_rn(__uint_as_float(amax_bits), 127.0f);
}

// The code of v: the integer nearest to v / scale, ties to even, within +-127 (beyond them only
// where the scale itself is so small that it was rounded).
__device__ __forceinline__ int row_code(float v, float scale) {
  const float q = rintf(__fdiv_rn(v, scale));
  return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// Whether the row has codes at all: not if it is zero (or its scale is), infinite or NaN.
__device__ __forceinline__ bool row_has_codes(uint32_t amax_bits, float scale) {
  return amax_bits < 0x7F800000u && scale > 0.0f;
}

template <int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) all = max(all, shared[w]);
  __syncthreads();
  return all;
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) all += shared[w];
  __syncthreads();
  return all;
}

constexpr int kRowThreads = 256;

// Row r of the codes = row source[r] (or r) of x. A source row outside [0, tokens) leaves the
// row's codes and its scale as they were.
template <typename In>
__global__ void __launch_bounds__(kRowThreads)
int8_quantize_kernel(const In* __restrict__ x, long long ldx, const int* __restrict__ source,
                     int rows, int tokens, int k, int8_t* __restrict__ q, long long ldq,
                     float* __restrict__ scales) {
  __shared__ uint32_t shared[kRowThreads / 32];
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int t = source != nullptr ? source[r] : r;
    if (t < 0 || t >= tokens) continue;
    const In* in = x + t * ldx;
    uint32_t amax = 0;
    for (int c = threadIdx.x; c < k; c += kRowThreads) {
      amax = max(amax, magnitude_bits(to_float(in[c])));
    }
    amax = block_max<kRowThreads>(amax, shared);
    const float scale = row_scale(amax);
    const bool live = row_has_codes(amax, scale);
    for (int c = threadIdx.x; c < k; c += kRowThreads) {
      q[r * ldq + c] = static_cast<int8_t>(live ? row_code(to_float(in[c]), scale) : 0);
    }
    if (threadIdx.x == 0) scales[r] = scale;
  }
}

// ---------------------------------------------------------------------------
// The norms around a block
// ---------------------------------------------------------------------------

struct NormParams {
  const void* x;         // [tokens][hidden], the block's output (or, alone, what is normed)
  const void* residual;  // [tokens][hidden] or null
  const float* post_weight;
  const float* gate;  // [gates][hidden]; each row serves tokens_per_gate tokens
  const float* next_weight;
  void* r;       // new residual, in the residual's type; null without one
  void* y;       // normed rows: codes, or values of type y_kind; null without next_weight
  float* scales; // with codes
  long long ldx, ldres, ldr, ldy;
  int tokens, hidden, tokens_per_gate;
  float residual_scale;
  double eps;
  int x_kind, residual_kind, y_kind;  // NVFP4_IN_*; y_kind -1: codes
};

__device__ __forceinline__ float load_kind(const void* p, long long i, int kind) {
  if (kind == 0) return static_cast<const float*>(p)[i];
  if (kind == 1) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_kind(void* p, long long i, int kind, float v) {
  if (kind == 0) {
    static_cast<float*>(p)[i] = v;
  } else if (kind == 1) {
    static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
  } else {
    static_cast<__half*>(p)[i] = from_float<__half>(v);
  }
}

// 1 / sqrt(mean + eps) of a row, rounded to FP32 once. The sum is taken in 64 bits: its value
// then does not depend, at FP32's precision, on how a row is split over threads, and codes that
// lie next to a border come out the same for every split.
__device__ __forceinline__ float row_rstd(double sum, int hidden, double eps) {
  return static_cast<float>(1.0 / sqrt(sum / hidden + eps));
}

__global__ void __launch_bounds__(kRowThreads) residual_norm_kernel(const NormParams p) {
  extern __shared__ float row[];
  __shared__ double sums[kRowThreads / 32];
  __shared__ uint32_t maxima[kRowThreads / 32];
  for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    double sum = 0.0;
    for (int c = threadIdx.x; c < p.hidden; c += kRowThreads) {
      const float v = load_kind(p.x, t * p.ldx + c, p.x_kind);
      row[c] = v;
      sum += static_cast<double>(v) * v;
    }
    if (p.post_weight != nullptr) sum = block_sum<kRowThreads>(sum, sums);
    const float post = p.post_weight != nullptr ? row_rstd(sum, p.hidden, p.eps) : 1.0f;
    sum = 0.0;
    for (int c = threadIdx.x; c < p.hidden; c += kRowThreads) {
      float v = row[c];
      if (p.post_weight != nullptr) v = __fmul_rn(__fmul_rn(v, post), p.post_weight[c]);
      if (p.gate != nullptr) {
        v = __fmul_rn(v, p.gate[static_cast<long long>(t / p.tokens_per_gate) * p.hidden + c]);
      }
      if (p.residual != nullptr) {
        v = __fadd_rn(__fmul_rn(load_kind(p.residual, t * p.ldres + c, p.residual_kind),
                                p.residual_scale), v);
        store_kind(p.r, t * p.ldr + c, p.residual_kind, v);
      }
      row[c] = v;
      sum += static_cast<double>(v) * v;
    }
    if (p.next_weight == nullptr) continue;
    sum = block_sum<kRowThreads>(sum, sums);
    const float next = row_rstd(sum, p.hidden, p.eps);
    uint32_t amax = 0;
    for (int c = threadIdx.x; c < p.hidden; c += kRowThreads) {
      const float v = __fmul_rn(__fmul_rn(row[c], next), p.next_weight[c]);
      if (p.y_kind >= 0) {
        store_kind(p.y, t * p.ldy + c, p.y_kind, v);
      } else {
        row[c] = v;
        amax = max(amax, magnitude_bits(v));
      }
    }
    if (p.y_kind >= 0) continue;
    amax = block_max<kRowThreads>(amax, maxima);
    const float scale = row_scale(amax);
    const bool live = row_has_codes(amax, scale);
    for (int c = threadIdx.x; c < p.hidden; c += kRowThreads) {
      static_cast<int8_t*>(p.y)[t * p.ldy + c] =
          static_cast<int8_t>(live ? row_code(row[c], scale) : 0);
    }
    if (threadIdx.x == 0) p.scales[t] = scale;
  }
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

// x * sigmoid(x).
__device__ __forceinline__ float silu(float x) { return x * __fdividef(1.0f, 1.0f + __expf(-x)); }

// Routing of pairs to unpadded groups: offsets[e] = number of pairs of the experts before e
// (offsets[experts]: of all), and a cursor per expert that starts there.
__global__ void expert_offsets_kernel(const int* __restrict__ counts, int experts,
                                      int* __restrict__ offsets) {
  __shared__ int scan[1024];
  const int e = threadIdx.x;
  scan[e] = e < experts ? counts[e] : 0;
  __syncthreads();
  for (int d = 1; d < 1024; d *= 2) {
    const int before = e >= d ? scan[e - d] : 0;
    __syncthreads();
    scan[e] += before;
    __syncthreads();
  }
  if (e < experts) offsets[e + 1] = scan[e];
  if (e == 0) offsets[0] = 0;
}

}  // namespace nvfp4
