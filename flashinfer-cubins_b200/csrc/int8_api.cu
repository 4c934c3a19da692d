// Host side of the 8-bit-integer operators of include/nvfp4_b200.h: argument checks and
// launches. Nothing here keeps state between calls, allocates, throws or synchronises.

#include "../../include/nvfp4_b200.h"

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "int8_kernels.cuh"
#include "nvfp4_host.h"

using namespace nvfp4;

namespace {

template <typename... Args>
int fail(int code, const char* format, Args... args) {
  char text[384];
  snprintf(text, sizeof(text), format, args...);
  return host_fail(code, text);
}

int fail(int code, const char* text) { return host_fail(code, text); }

#define CUDA_TRY(expr)                                             \
  do {                                                             \
    cudaError_t err__ = (expr);                                    \
    if (err__ != cudaSuccess) return host_fail_cuda(err__, #expr); \
  } while (0)

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int kind_bytes(int kind) { return kind == NVFP4_IN_F32 ? 4 : 2; }

bool is_in_kind(int kind) {
  return kind == NVFP4_IN_F32 || kind == NVFP4_IN_BF16 || kind == NVFP4_IN_F16;
}

// Sums of k products of two codes of -128..127 stay below 2^31 up to here.
constexpr int kMaxDepth = 131071;
constexpr int kMaxExperts = 1024;
constexpr int kMaxHidden = 32768;

int check_product(const Int8GemmParams& p, int width) {
  if (p.rows < 0 || p.n < 1 || p.k < 1 || p.k > kMaxDepth || p.experts < 1 ||
      p.experts > kMaxExperts || width > (1 << 30)) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE,
                "unsupported product: %d rows, n=%d, k=%d (at most %d), %d experts (at most %d)",
                p.rows, p.n, p.k, kMaxDepth, p.experts, kMaxExperts);
  }
  if (p.rows == 0) return 0;
  if (p.a == nullptr || p.b == nullptr || p.a_scales == nullptr || p.b_scales == nullptr ||
      p.d == nullptr) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  }
  if (p.out_kind != NVFP4_OUT_F16 && p.out_kind != NVFP4_OUT_F32 && p.out_kind != NVFP4_OUT_BF16) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "unknown output kind %d", p.out_kind);
  }
  if (p.lda < p.k || p.ldb < p.k || p.ldd < p.n || p.expert_stride < 0) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "rows overlap: lda=%lld ldb=%lld ldd=%lld", p.lda, p.ldb,
                p.ldd);
  }
  if (!aligned(p.a, 16) || !aligned(p.b, 16) || p.lda % 16 != 0 || p.ldb % 16 != 0 ||
      p.expert_stride % 16 != 0 || !aligned(p.a_scales, 4) || !aligned(p.b_scales, 4) ||
      !aligned(p.bias, 4) || !aligned(p.offsets, 4) ||
      !aligned(p.d, p.out_kind == NVFP4_OUT_F32 ? 4 : 2)) {
    return fail(NVFP4_E_MISALIGNED, "codes must start and lie 16-byte aligned");
  }
  return 0;
}

int launch_product(const Int8GemmParams& p, int gated, void* stream) {
  const int width = gated ? 2 * p.n : p.n;
  if (p.n > (1 << 29)) return fail(NVFP4_E_UNSUPPORTED_SHAPE, "n=%d is too large", p.n);
  if (int rc = check_product(p, width)) return rc;
  if (p.rows == 0) return 0;
  const int tiles = (p.rows + kTile - 1) / kTile + p.experts - 1;
  const dim3 grid((p.n + kTile - 1) / kTile, tiles);
  if (tiles > 65535) return fail(NVFP4_E_UNSUPPORTED_SHAPE, "too many rows: %d", p.rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (gated) {
    int8_gemm_kernel<true><<<grid, 256, 0, s>>>(p);
  } else {
    int8_gemm_kernel<false><<<grid, 256, 0, s>>>(p);
  }
  CUDA_TRY(cudaGetLastError());
  return 0;
}

template <typename In>
void launch_quantize(int blocks, cudaStream_t s, const void* x, long long ldx, const int* source,
                     int rows, int tokens, int k, void* q, long long ldq, float* scales) {
  int8_quantize_kernel<In><<<blocks, kRowThreads, 0, s>>>(
      static_cast<const In*>(x), ldx, source, rows, tokens, k, static_cast<int8_t*>(q), ldq, scales);
}

}  // namespace

extern "C" {

int nvfp4_int8_gemm(const void* a, long long lda, const void* b, long long ldb,
                    const float* a_scales, const float* b_scales, const float* bias, void* d,
                    long long ldd, int m, int n, int k, int out_kind, int gated, void* stream) {
  Int8GemmParams p{};
  p.a = static_cast<const int8_t*>(a);
  p.b = static_cast<const int8_t*>(b);
  p.a_scales = a_scales;
  p.b_scales = b_scales;
  p.bias = bias;
  p.d = d;
  p.lda = lda;
  p.ldb = ldb;
  p.ldd = ldd;
  p.rows = m;
  p.n = n;
  p.k = k;
  p.experts = 1;
  p.out_kind = out_kind;
  return launch_product(p, gated, stream);
}

int nvfp4_int8_group_gemm(const void* a, long long lda, const void* b, long long ldb,
                          long long expert_stride, const float* a_scales, const float* b_scales,
                          const int* offsets, void* d, long long ldd, int experts, int rows, int n,
                          int k, int out_kind, int gated, void* stream) {
  if (offsets == nullptr && rows > 0) return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  Int8GemmParams p{};
  p.a = static_cast<const int8_t*>(a);
  p.b = static_cast<const int8_t*>(b);
  p.a_scales = a_scales;
  p.b_scales = b_scales;
  p.offsets = offsets;
  p.d = d;
  p.lda = lda;
  p.ldb = ldb;
  p.expert_stride = expert_stride;
  p.ldd = ldd;
  p.rows = rows;
  p.n = n;
  p.k = k;
  p.experts = experts;
  p.out_kind = out_kind;
  return launch_product(p, gated, stream);
}

int nvfp4_int8_quantize(const void* x, int x_kind, long long ldx, const int* source_rows, int rows,
                        int tokens, int k, void* q, long long ldq, float* scales, void* stream) {
  if (!is_in_kind(x_kind)) return fail(NVFP4_E_INVALID_ARGUMENT, "unknown input kind %d", x_kind);
  if (rows < 0 || tokens < 0 || k < 1) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "unsupported tensor: %d rows of %d, k=%d", rows, tokens, k);
  }
  if (rows == 0) return 0;
  if (source_rows == nullptr && rows != tokens) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "%d rows of %d tokens without source rows", rows, tokens);
  }
  if (q == nullptr || scales == nullptr || (x == nullptr && tokens > 0)) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  }
  if (ldq < k || (ldx < k && tokens > 1)) return fail(NVFP4_E_INVALID_ARGUMENT, "rows overlap");
  if (!aligned(x, kind_bytes(x_kind)) || !aligned(scales, 4) || !aligned(source_rows, 4)) {
    return fail(NVFP4_E_MISALIGNED, "misaligned operand address");
  }
  const int blocks = std::min(rows, 8 * host_sm_count());
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_kind == NVFP4_IN_F32) {
    launch_quantize<float>(blocks, s, x, ldx, source_rows, rows, tokens, k, q, ldq, scales);
  } else if (x_kind == NVFP4_IN_BF16) {
    launch_quantize<__nv_bfloat16>(blocks, s, x, ldx, source_rows, rows, tokens, k, q, ldq, scales);
  } else {
    launch_quantize<__half>(blocks, s, x, ldx, source_rows, rows, tokens, k, q, ldq, scales);
  }
  CUDA_TRY(cudaGetLastError());
  return 0;
}

int nvfp4_residual_norm(const void* x, int x_kind, long long ldx, const void* residual,
                        int residual_kind, long long ldres, const float* post_weight,
                        const float* gate, int gates, float residual_scale,
                        const float* next_weight, double eps, void* r, long long ldr, void* y,
                        int y_kind, long long ldy, float* scales, int tokens, int hidden,
                        void* stream) {
  if (!is_in_kind(x_kind) || (residual != nullptr && !is_in_kind(residual_kind)) ||
      (next_weight != nullptr && y_kind != NVFP4_NORM_CODES && !is_in_kind(y_kind))) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "unknown type: x %d, residual %d, y %d", x_kind,
                residual_kind, y_kind);
  }
  if (tokens < 0 || hidden < 1 || hidden > kMaxHidden) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "unsupported rows: %d of %d (at most %d wide)", tokens,
                hidden, kMaxHidden);
  }
  if (!(eps > 0.0) || !(eps < 1e30)) return fail(NVFP4_E_INVALID_ARGUMENT, "eps must be positive");
  if (gate != nullptr && (gates < 1 || tokens % gates != 0)) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "%d tokens do not share %d gates evenly", tokens, gates);
  }
  if (residual == nullptr &&
      (post_weight != nullptr || gate != nullptr || next_weight == nullptr || residual_scale != 1.0f)) {
    return fail(NVFP4_E_INVALID_ARGUMENT,
                "without a residual there is only the norm of x: no post weight, gate or scale");
  }
  if (tokens == 0) return 0;
  if (x == nullptr || (residual != nullptr && r == nullptr) ||
      (next_weight != nullptr && (y == nullptr || (y_kind == NVFP4_NORM_CODES && scales == nullptr)))) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  }
  if (tokens > 1 && (ldx < hidden || (residual != nullptr && (ldres < hidden || ldr < hidden)) ||
                     (next_weight != nullptr && ldy < hidden))) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "rows overlap");
  }
  const uintptr_t residual_bytes = residual != nullptr ? kind_bytes(residual_kind) : 1;
  if (!aligned(x, kind_bytes(x_kind)) || !aligned(residual, residual_bytes) ||
      !aligned(r, residual_bytes) || !aligned(post_weight, 4) || !aligned(gate, 4) ||
      !aligned(next_weight, 4) || !aligned(scales, 4) ||
      (next_weight != nullptr && y_kind != NVFP4_NORM_CODES && !aligned(y, kind_bytes(y_kind)))) {
    return fail(NVFP4_E_MISALIGNED, "misaligned operand address");
  }
  NormParams p{};
  p.x = x;
  p.residual = residual;
  p.post_weight = post_weight;
  p.gate = gate;
  p.next_weight = next_weight;
  p.r = r;
  p.y = y;
  p.scales = scales;
  p.ldx = ldx;
  p.ldres = ldres;
  p.ldr = ldr;
  p.ldy = ldy;
  p.tokens = tokens;
  p.hidden = hidden;
  p.tokens_per_gate = gate != nullptr ? tokens / gates : 1;
  p.residual_scale = residual_scale;
  p.eps = eps;
  p.x_kind = x_kind;
  p.residual_kind = residual_kind;
  p.y_kind = y_kind;
  const size_t bytes = static_cast<size_t>(hidden) * sizeof(float);
  CUDA_TRY(cudaFuncSetAttribute(residual_norm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kMaxHidden * static_cast<int>(sizeof(float))));
  const int blocks = std::min(tokens, 8 * host_sm_count());
  residual_norm_kernel<<<blocks, kRowThreads, bytes, static_cast<cudaStream_t>(stream)>>>(p);
  CUDA_TRY(cudaGetLastError());
  return 0;
}

int nvfp4_moe_offsets(const int* counts, int experts, int* offsets, void* stream) {
  if (counts == nullptr || offsets == nullptr) return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  if (experts < 1 || experts > kMaxExperts) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "%d experts (at most %d)", experts, kMaxExperts);
  }
  expert_offsets_kernel<<<1, kMaxExperts, 0, static_cast<cudaStream_t>(stream)>>>(counts, experts,
                                                                                  offsets);
  CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // extern "C"
