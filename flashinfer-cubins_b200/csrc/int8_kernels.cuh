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

// Two products or sums an instruction, each rounded on its own: a row's values, and with them its
// codes, are those of the separate operations. (A packed sum behind a packed product was fused in
// spite of its rounding mode: where one follows the other the product is taken unpacked.)
__device__ __forceinline__ float2 product2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t"
      ".reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t"
      "}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float2 sum2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t"
      ".reg .b64 x, y;\n\t"
      "mov.b64 x, {%2, %3};\n\t"
      "mov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t"
      "}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
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

// The code of v: the integer nearest to the correctly rounded v / scale, ties to even, within
// +-127 (beyond them only where the scale is subnormal and was rounded coarsely).
__device__ __forceinline__ int row_code(float v, float scale) {
  const float q = rintf(__fdiv_rn(v, scale));
  return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// How a row's codes are made.
struct RowCodes {
  float scale, inverse;
  bool live;     // false: zero row (or scale), infinite or NaN: codes are zero
  bool divide;   // the scale is subnormal: divide every value
};

__device__ __forceinline__ RowCodes row_codes(uint32_t amax_bits) {
  RowCodes r;
  r.scale = row_scale(amax_bits);
  r.live = amax_bits < 0x7F800000u && r.scale > 0.0f;
  r.divide = r.scale < 1.17549435e-38f;
  r.inverse = __frcp_rn(r.scale);
  return r;
}

// Codes of values. A product with the reciprocal decides: it is within 1.5 steps of 2^-17 of the
// quotient (|q| <= 127), so where it lies more than 2^-15 from the middle between two integers the
// quotient, rounded, lies on the same side. Adding 1.5 * 2^23 rounds it to an integer (ties to even)
// whose low byte is the code. Values nearer to a middle (one in 2^14) are divided. Dividing all of
// them cost 94 us for 8192 x 7168 BF16 values, this 32.
constexpr float kRoundBias = 12582912.0f;

__device__ __forceinline__ bool near_middle(float off) { return off >= 0.5f - 0x1p-15f; }

__device__ __forceinline__ uint2 eight_codes(const float (&v)[8], const RowCodes& row) {
  if (!row.live) return make_uint2(0u, 0u);
  const float2 inverse = make_float2(row.inverse, row.inverse), round = make_float2(kRoundBias, kRoundBias);
  uint32_t b[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 x = make_float2(v[i], v[i + 1]);
    const float2 t = __ffma2_rn(x, inverse, round);                          // round + n
    const float2 n = __ffma2_rn(t, make_float2(-1.0f, -1.0f), round);        // -n
    const float2 d = __ffma2_rn(x, inverse, n);
    off = fmaxf(fmaxf(off, fabsf(d.x)), fabsf(d.y));
    b[i] = __float_as_uint(t.x);
    b[i + 1] = __float_as_uint(t.y);
  }
  if (row.divide || near_middle(off)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = static_cast<uint32_t>(row_code(v[i], row.scale));
  }
  return make_uint2(
      __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

__device__ __forceinline__ int one_code(float v, const RowCodes& row) {
  if (!row.live) return 0;
  const float t = fmaf(v, row.inverse, kRoundBias);
  const float off = fabsf(fmaf(v, row.inverse, kRoundBias - t));
  if (row.divide || near_middle(off)) return row_code(v, row.scale);
  return static_cast<int>(__float_as_uint(t));
}

// ---------------------------------------------------------------------------
// Rows in registers
// ---------------------------------------------------------------------------
//
// A row belongs to one warp (WARP: eight rows to a CTA, no barrier) or to one CTA, whose threads
// hold N pieces of P neighbouring elements each, read once, every load issued before the first is
// used. P = 8 where all rows start on a multiple of eight elements and are a multiple of eight long:
// 16-byte loads of 16-bit elements, 32-byte ones of 32-bit elements (two 16-byte loads a lane, 32
// bytes apart, took the L1 cache twice the cycles). P = 1 for any other start, pitch and length:
// there the CTA has its full THREADS, so that a thread's elements lie constant distances apart and
// an access needs no address of its own (8192 x 5121 norms: 319 us with computed addresses).

__device__ __forceinline__ void load_32_bytes(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}

__device__ __forceinline__ void store_32_bytes(void* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p)
               : "memory");
}

// P elements as they lie in memory.
template <bool WIDE, int P>
struct Raw {
  static constexpr int kWords = WIDE ? P : (P + 1) / 2;
  uint32_t w[kWords];
};

// Elements c .. c + P - 1 of a row of `width`; zero if they lie beyond it.
template <bool WIDE, int P>
__device__ __forceinline__ Raw<WIDE, P> load_raw(const void* row, int c, int width) {
  Raw<WIDE, P> r{};
  if (c < width) {
    if constexpr (P == 1) {
      if constexpr (WIDE) {
        r.w[0] = static_cast<const uint32_t*>(row)[c];
      } else {
        r.w[0] = static_cast<const uint16_t*>(row)[c];
      }
    } else if constexpr (WIDE) {
      load_32_bytes(static_cast<const float*>(row) + c, r.w);
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c);
      r.w[0] = q.x;
      r.w[1] = q.y;
      r.w[2] = q.z;
      r.w[3] = q.w;
    }
  }
  return r;
}

// The values; `half`: 16-bit elements are FP16, else BF16.
template <bool WIDE, int P>
__device__ __forceinline__ void unpack(const Raw<WIDE, P>& r, bool half, float (&v)[P]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = __uint_as_float(r.w[i]);
  } else if (half) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      v[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(r.w[i / 2] >> (16 * (i % 2)))));
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      v[i] = __uint_as_float(i % 2 != 0 ? r.w[i / 2] & 0xFFFF0000u : r.w[i / 2] << 16);
    }
  }
}

// FP32 values of a vector over the row (weights, gates), zero beyond it.
template <int P>
__device__ __forceinline__ void load_weights(const float* row, int c, int width, float (&v)[P]) {
  unpack<true, P>(load_raw<true, P>(row, c, width), false, v);
}

// Stores values of kind NVFP4_IN_*.
template <int P>
__device__ __forceinline__ void store_values(void* row, int c, int kind, const float (&v)[P]) {
  if (kind == 0) {
    float* p = static_cast<float*>(row) + c;
    if constexpr (P == 8) {
      store_32_bytes(p, v);
    } else {
      p[0] = v[0];
    }
    return;
  }
  uint16_t* p = static_cast<uint16_t*>(row) + c;
  if constexpr (P == 8) {
    uint32_t w[4];
    if (kind == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if (kind == 1) {
    *reinterpret_cast<__nv_bfloat16*>(p) = from_float<__nv_bfloat16>(v[0]);
  } else {
    *reinterpret_cast<__half*>(p) = from_float<__half>(v[0]);
  }
}

// Codes of P values.
template <int P>
__device__ __forceinline__ void store_codes(int8_t* row, int c, const float (&v)[P], const RowCodes& codes) {
  if constexpr (P == 8) {
    *reinterpret_cast<uint2*>(row + c) = eight_codes(v, codes);
  } else {
    row[c] = static_cast<int8_t>(one_code(v[0], codes));
  }
}

// Registers of a thread. What bounds the row kernels is how many rows are under way on an SM (half of
// the issue slots idle with three), so they get fewer than the compiler would take: the norms in pieces
// of eight 48 (8192 x 5120: 70 us, with 64 registers 78, with 40 and spills 73), the quantiser 40 (8192 x
// 7168: 31.8 us, with 52 registers 32.4), rows taken one element at a time 40 (4096 x 3001 to codes: 43
// us, with 64 registers 53; codes of 8192 x 7169 76, with 64 registers 90). CTAs of 1,024 threads need 64, and
// the norms' threads of 16 single elements do no better with fewer.
constexpr int row_registers(bool norm, int p, int n, int threads, bool warp) {
  const int elements = p * n;
  if (elements == 8) return p == 1 ? 40 : threads == 1024 ? 64 : 48;
  if (warp) return 48;  // of the quantiser alone
  if (!norm && threads == 512) return 40;
  if (p == 8 && threads == 512) return n == 2 ? 48 : 64;
  return 64;
}

// Over the row's threads; `shared` (one word for each warp) serves one reduction of a kernel.
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xFFFFFFFFu, v);
  if constexpr (WARP) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xFFFFFFFFu, lane < static_cast<int>(blockDim.x >> 5) ? shared[lane] : 0u);
}

template <bool WARP>
__device__ __forceinline__ double row_sum(double v, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if constexpr (WARP) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < static_cast<int>(blockDim.x >> 5) ? shared[lane] : 0.0;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

constexpr int kWarpRows = 8;  // rows of a CTA where each belongs to a warp

template <bool WARP>
__device__ __forceinline__ int row_of_thread() {
  return WARP ? static_cast<int>(blockIdx.x) * kWarpRows + static_cast<int>(threadIdx.x >> 5)
              : static_cast<int>(blockIdx.x);
}

struct QuantizeParams {
  const void* x;
  const int* source;  // or null
  int8_t* q;
  float* scales;
  long long ldx, ldq;
  int rows, tokens, k;
  int x_kind;
};

// Row r of the codes = row source[r] (or r) of x. A source row outside [0, tokens) leaves the
// row's codes and its scale as they were. Plain loads: the kernel may be resident while the one before
// writes what it reads.
template <bool WIDE, int P, int N, int THREADS, bool WARP>
__global__ void __maxnreg__(row_registers(false, P, N, THREADS, WARP)) int8_quantize_kernel(const QuantizeParams p) {
  __shared__ uint32_t maxima[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int r = row_of_thread<WARP>();
  if (r >= p.rows) return;
  const int t = p.source != nullptr ? p.source[r] : r;
  if (t < 0 || t >= p.tokens) return;
  const int step = P * (WARP ? 32 : P == 1 ? THREADS : blockDim.x);
  const int first = P * (WARP ? threadIdx.x & 31 : threadIdx.x);
  const void* in = static_cast<const uint8_t*>(p.x) + t * p.ldx * (WIDE ? 4 : 2);
  Raw<WIDE, P> raw[N];
#pragma unroll
  for (int j = 0; j < N; ++j) raw[j] = load_raw<WIDE, P>(in, first + step * j, p.k);
  // 16-bit magnitudes order like their bits, too: the largest of the negative ones is the largest
  // unsigned pattern, that of the positive ones the largest signed one.
  uint32_t amax = 0, positive = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < P; ++i) amax = max(amax, raw[j].w[i] & 0x7FFFFFFFu);
    } else if constexpr (P == 8) {
      amax = __vimax3_u16x2(__vimax3_u16x2(amax, raw[j].w[0], raw[j].w[1]), raw[j].w[2], raw[j].w[3]);
      positive = __vimax3_s16x2(__vimax3_s16x2(positive, raw[j].w[0], raw[j].w[1]), raw[j].w[2], raw[j].w[3]);
    } else {
      amax = max(amax, raw[j].w[0] & 0x7FFFu);
    }
  }
  const bool half = p.x_kind == 2;
  if constexpr (!WIDE) {
    if constexpr (P == 8) amax = __vmaxu2(amax & 0x7FFF7FFFu, positive);
    const uint32_t both = max(amax & 0xFFFFu, amax >> 16);
    amax = half ? magnitude_bits(__half2float(__ushort_as_half(static_cast<unsigned short>(both))))
                : both << 16;
  }
  amax = row_max<WARP>(amax, maxima);
  const RowCodes row = row_codes(amax);
  int8_t* out = p.q + r * p.ldq;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = first + step * j;
    if (c < p.k) {
      float v[P];
      unpack<WIDE, P>(raw[j], half, v);
      store_codes<P>(out, c, v, row);
    }
  }
  if (first == 0) p.scales[r] = row.scale;
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
  double eps, inverse_hidden;
  int x_kind, residual_kind, y_kind;  // NVFP4_IN_*; y_kind -1: codes
};

__device__ __forceinline__ const void* row_at(const void* p, long long element, int kind) {
  return static_cast<const uint8_t*>(p) + element * (kind == 0 ? 4 : 2);
}

__device__ __forceinline__ void* row_at(void* p, long long element, int kind) {
  return static_cast<uint8_t*>(p) + element * (kind == 0 ? 4 : 2);
}

// 1 / sqrt(mean + eps) of a row, rounded to FP32 once. The sum is taken in 64 bits: its value
// then does not depend, at FP32's precision, on how a row is split over threads, and codes that
// lie next to a border come out the same for every split. Two steps of Newton's iteration for
// m^(-1/2) in 64 bits, r += r (1 - m r^2) / 2, square the error of FP32's estimate twice (2^-21 to
// below 2^-52); the 64-bit square root and quotient are left to means FP32 cannot hold.
__device__ __forceinline__ float row_rstd(double sum, double inverse_hidden, double eps) {
  const double m = fma(sum, inverse_hidden, eps);
  if (!(m > 1e-30 && m < 1e30)) return static_cast<float>(1.0 / sqrt(m));
  double r = rsqrtf(static_cast<float>(m));
#pragma unroll
  for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-m * r, r, 1.0), r);
  return static_cast<float>(r);
}

// Sums of squares in four chains: a chain of 32 dependent 64-bit additions took longer than the
// loads.
struct SquareSum {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  template <int P>
  __device__ __forceinline__ void add(const float (&v)[P], int piece) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const double d = v[i];
      double& chain = s[(piece * P + i) % 4];
      chain = fma(d, d, chain);
    }
  }
  __device__ __forceinline__ double total() const { return (s[0] + s[1]) + (s[2] + s[3]); }
};

template <int P>
__device__ __forceinline__ void scale_by(float (&v)[P], float s) {
#pragma unroll
  for (int i = 0; i + 1 < P; i += 2) {
    const float2 f = product2(make_float2(v[i], v[i + 1]), make_float2(s, s));
    v[i] = f.x;
    v[i + 1] = f.y;
  }
  if constexpr (P == 1) v[0] = __fmul_rn(v[0], s);
}

template <int P>
__device__ __forceinline__ void multiply(float (&v)[P], const float (&w)[P]) {
#pragma unroll
  for (int i = 0; i + 1 < P; i += 2) {
    const float2 f = product2(make_float2(v[i], v[i + 1]), make_float2(w[i], w[i + 1]));
    v[i] = f.x;
    v[i + 1] = f.y;
  }
  if constexpr (P == 1) v[0] = __fmul_rn(v[0], w[0]);
}

template <int P>
__device__ __forceinline__ void add(float (&v)[P], const float (&w)[P]) {
#pragma unroll
  for (int i = 0; i + 1 < P; i += 2) {
    const float2 f = sum2(make_float2(v[i], v[i + 1]), make_float2(w[i], w[i + 1]));
    v[i] = f.x;
    v[i + 1] = f.y;
  }
  if constexpr (P == 1) v[0] = __fadd_rn(v[0], w[0]);
}

template <bool X_WIDE, bool R_WIDE, int P, int N, int THREADS, bool WARP>
__global__ void __maxnreg__(row_registers(true, P, N, THREADS, WARP)) residual_norm_kernel(const NormParams p) {
  __shared__ double post_sums[32], next_sums[32];
  __shared__ uint32_t maxima[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = row_of_thread<WARP>();
  if (t >= p.tokens) return;
  const int hidden = p.hidden;
  const int step = P * (WARP ? 32 : P == 1 ? THREADS : blockDim.x);
  const int first = P * (WARP ? threadIdx.x & 31 : threadIdx.x);
  Raw<X_WIDE, P> raw_x[N];
  Raw<R_WIDE, P> raw_r[N];
  const void* x_row = row_at(p.x, t * p.ldx, p.x_kind);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    raw_x[j] = load_raw<X_WIDE, P>(x_row, first + step * j, hidden);
  }
  if (p.residual != nullptr) {
    const void* res_row = row_at(p.residual, t * p.ldres, p.residual_kind);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      raw_r[j] = load_raw<R_WIDE, P>(res_row, first + step * j, hidden);
    }
  }
  float v[N][P];
#pragma unroll
  for (int j = 0; j < N; ++j) unpack<X_WIDE, P>(raw_x[j], p.x_kind == 2, v[j]);
  if (p.post_weight != nullptr) {
    SquareSum sum;
#pragma unroll
    for (int j = 0; j < N; ++j) sum.add(v[j], j);
    const float rstd = row_rstd(row_sum<WARP>(sum.total(), post_sums), p.inverse_hidden, p.eps);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float w[P];
      load_weights<P>(p.post_weight, first + step * j, hidden, w);
      scale_by(v[j], rstd);
      multiply(v[j], w);
    }
  }
  if (p.gate != nullptr) {
    const float* gate = p.gate + static_cast<long long>(t / p.tokens_per_gate) * hidden;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float g[P];
      load_weights<P>(gate, first + step * j, hidden, g);
      multiply(v[j], g);
    }
  }
  if (p.residual != nullptr) {
    void* r_row = row_at(p.r, t * p.ldr, p.residual_kind);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = first + step * j;
      float res[P];
      unpack<R_WIDE, P>(raw_r[j], p.residual_kind == 2, res);
#pragma unroll
      for (int i = 0; i < P; ++i) res[i] = __fmul_rn(res[i], p.residual_scale);
      add(v[j], res);
      if (c < hidden) store_values<P>(r_row, c, p.residual_kind, v[j]);
    }
  }
  if (p.next_weight == nullptr) return;
  SquareSum sum;
#pragma unroll
  for (int j = 0; j < N; ++j) sum.add(v[j], j);
  const float rstd = row_rstd(row_sum<WARP>(sum.total(), next_sums), p.inverse_hidden, p.eps);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float w[P];
    load_weights<P>(p.next_weight, first + step * j, hidden, w);
    scale_by(v[j], rstd);
    multiply(v[j], w);
  }
  if (p.y_kind >= 0) {
    void* y_row = row_at(p.y, t * p.ldy, p.y_kind);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = first + step * j;
      if (c < hidden) store_values<P>(y_row, c, p.y_kind, v[j]);
    }
    return;
  }
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int i = 0; i < P; ++i) amax = max(amax, magnitude_bits(v[j][i]));
  }
  const RowCodes row = row_codes(row_max<WARP>(amax, maxima));
  int8_t* y_row = static_cast<int8_t*>(p.y) + t * p.ldy;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = first + step * j;
    if (c < hidden) store_codes<P>(y_row, c, v[j], row);
  }
  if (first == 0) p.scales[t] = row.scale;
}

// ---------------------------------------------------------------------------
// Rows too long for registers
// ---------------------------------------------------------------------------

__device__ __forceinline__ float load_kind(const void* p, long long i, int kind) {
  if (kind == 0) return static_cast<const float*>(p)[i];
  if (kind == 1) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}

// A CTA to a row, which is read twice (the second time mostly from the caches).
__global__ void __launch_bounds__(1024) int8_quantize_long_kernel(const QuantizeParams p) {
  __shared__ uint32_t maxima[32];
  const int r = blockIdx.x;
  const int t = p.source != nullptr ? p.source[r] : r;
  if (t < 0 || t >= p.tokens) return;
  uint32_t amax = 0;
#pragma unroll 8
  for (int c = threadIdx.x; c < p.k; c += 1024) {
    amax = max(amax, magnitude_bits(load_kind(p.x, t * p.ldx + c, p.x_kind)));
  }
  const RowCodes row = row_codes(row_max<false>(amax, maxima));
#pragma unroll 8
  for (int c = threadIdx.x; c < p.k; c += 1024) {
    p.q[r * p.ldq + c] = static_cast<int8_t>(one_code(load_kind(p.x, t * p.ldx + c, p.x_kind), row));
  }
  if (threadIdx.x == 0) p.scales[r] = row.scale;
}

// ---------------------------------------------------------------------------
// Products and routing
// ---------------------------------------------------------------------------

// x * sigmoid(x) with the approximate exponential and reciprocal (2^-22 and 2^-23 relative). Where x is
// well below zero the rounding of x log2(e) and of its constant counts for more: the exponential turns
// them into up to 1.25 |x| 2^-24 of the value, 4.5e-6 at x = -60. That is far below a rounding to 16 bits
// and seen by FP32 results alone. No slow path where exp(-x) overflows, its reciprocal is 0 there (from
// x = -87.3 on, where the value is below 1e-36).
__device__ __forceinline__ float silu(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return x * r;
}

// Routing of pairs to unpadded groups: offsets[e] = number of pairs of the experts before e
// (offsets[experts]: of all).
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
