// Host side of the 8-bit-integer operators of include/nvfp4_b200.h: argument checks and
// launches. Nothing here allocates, throws or (but for the status call) synchronises; what is kept
// between calls are properties of devices.

#include "../../include/nvfp4_b200.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include <cuda_runtime.h>

#include "int8_gemm_kernel.cuh"
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
constexpr int kMaxHidden = 32768;
// 1 / sqrt(eps) is 3.2e38, below FP32's largest number: a row's factor is finite, and a zero row zero.
constexpr double kMinEps = 1e-77;
// Rows of any operand, and elements of a row of the quantiser: a count and a tile, a CTA's rows or a
// step of its threads together stay within 32 bits.
constexpr int kMaxRows = 1 << 30;

// One product, dense (offsets null, one expert) or grouped.
struct Product {
  const void* a;
  const void* b;
  const float* a_scales;
  const float* b_scales;
  const float* bias;
  const int* offsets;
  void* d;
  long long lda, ldb, expert_stride, ldd;
  int rows, n, k, experts, out_kind;
  bool gated;
};

int check_product(const Product& p) {
  if (p.rows < 0 || p.rows > kMaxRows || p.n < 1 || p.n > (p.gated ? kMaxRows / 2 : kMaxRows) ||
      p.k < 1 || p.k > kMaxDepth || p.experts < 1 || p.experts > kInt8MaxExperts) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE,
                "unsupported product: %d rows, n=%d, k=%d (at most %d), %d experts (at most %d)",
                p.rows, p.n, p.k, kMaxDepth, p.experts, kInt8MaxExperts);
  }
  if (p.rows == 0) return 0;
  if (p.a == nullptr || p.b == nullptr || p.a_scales == nullptr || p.b_scales == nullptr ||
      p.d == nullptr) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  }
  if (p.out_kind != NVFP4_OUT_F16 && p.out_kind != NVFP4_OUT_F32 && p.out_kind != NVFP4_OUT_BF16) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "unknown output kind %d", p.out_kind);
  }
  const long long width = p.gated ? 2ll * p.n : p.n;
  if (p.lda < p.k || p.ldb < p.k || p.ldd < p.n ||
      (p.experts > 1 && p.expert_stride < (width - 1) * p.ldb + p.k)) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "rows overlap: lda=%lld ldb=%lld ldd=%lld, experts %lld apart",
                p.lda, p.ldb, p.ldd, p.expert_stride);
  }
  if (!aligned(p.a, 16) || !aligned(p.b, 16) || p.lda % 16 != 0 || p.ldb % 16 != 0 ||
      (p.experts > 1 && p.expert_stride % 16 != 0) || !aligned(p.a_scales, 4) ||
      !aligned(p.b_scales, 4) || !aligned(p.bias, 4) || !aligned(p.offsets, 4) ||
      !aligned(p.d, p.out_kind == NVFP4_OUT_F32 ? 4 : 2)) {
    return fail(NVFP4_E_MISALIGNED, "codes must start and lie 16-byte aligned");
  }
  return 0;
}

using TileKernel = void (*)(Int8TileParams);

TileKernel tile_kernel(int ctas, int sub, bool gated) {
  if (ctas == 1) return gated ? int8_tile_kernel<1, 2, true> : int8_tile_kernel<1, 2, false>;
  if (sub == 1) return gated ? int8_tile_kernel<2, 1, true> : int8_tile_kernel<2, 1, false>;
  return gated ? int8_tile_kernel<2, 2, true> : int8_tile_kernel<2, 2, false>;
}

// Codes (128-byte swizzle), or with `output` 16-bit elements as they lie.
int encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims,
           const cuuint64_t* strides, const cuuint32_t* box, bool output = false) {
  EncodeTiled encoder = nullptr;
  if (int rc = host_encoder(&encoder)) return rc;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult res = encoder(
      map, output ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, rank,
      const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
      output ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
      output ? CU_TENSOR_MAP_L2_PROMOTION_NONE : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) {
    return fail(static_cast<int>(res), "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(res));
  }
  return 0;
}

// How a product is cut: CTAs that share a tile's MMAs, tokens of a tile, pieces of 128 k in a stage,
// and parts of k.
struct Tiling {
  int ctas, tile_tokens, sub, split;
};

// Clusters of `split` CTAs, one to an SM, that the current device holds at once: clusters do not reach
// over its groups of SMs, which are not all of one size (B200: 74 of two, 33 of four, 15 of eight). A
// property of the device, asked for once.
int cluster_slots(int split, int sms) {
  static std::atomic<int> known[64][4];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return sms / split * 3 / 4;
  std::atomic<int>& slot = known[device][split == 2 ? 1 : split == 4 ? 2 : 3];
  int count = slot.load(std::memory_order_relaxed);
  if (count > 0) return count;
  const void* kernel = reinterpret_cast<const void*>(tile_kernel(1, 2, false));
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = static_cast<unsigned int>(split);
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned int>(split));
  config.blockDim = dim3(int8_threads(32));
  config.dynamicSmemBytes = kInt8SharedLimit;
  config.attrs = attribute;
  config.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kInt8SharedLimit) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&count, kernel, &config) != cudaSuccess || count < 1) {
    cudaGetLastError();
    return sms / split * 3 / 4;
  }
  slot.store(count, std::memory_order_relaxed);
  return count;
}

// Microseconds of a tiling by the measured costs of its parts (1.9 GHz):
//   a step of 128 k   the largest of its loads (140 GB/s an SM), its MMAs (2 columns a clock; 4 x 32 k)
//                     and the loops that issue them (0.135 us; with one piece a stage 0.22 us)
//   a tile            its steps or, where those are shorter, its epilogue: 0.6 us and 0.3 (gated
//                     0.33) for every 32 tokens; the first tile's steps or the last one's epilogue
//                     stand alone
//   a pair            0.5 us for its cluster; a split 0.5 us, 0.6 for every 32 tokens and 0.1 for
//                     each part for the exchange of partial sums
//   everything        not less than the operands' bytes at 6 TB/s; and a tenth of the loads at 12 TB/s,
//                     which decides between tilings that are otherwise alike
// Groups differ in size: 0.6 of a tile each is counted for their last ones.
// What the choice is worth (device time, rows x n x k): 256 x 4096 x 7168 takes 13.4 us in pairs on 64
// tokens and 21.9 on 256, where 32 of 148 SMs work; 16 x 7168 x 2048 6.3 us with all of k in one CTA and
// 7.3 split in two; 32 x 4096 x 8192 9.6 split in four and 23 whole; 277 x 256 x 5136 8.0 split in four,
// 12.8 whole and 14.3 in eight, whose clusters find no room together; 16 experts of 8192 rows, gated 1536
// x 4096, 92 in pairs on 256 tokens, 98 on 192 and 270 on 32; 2 experts of 3303 rows, 352 x 4384, 11.7
// on 96 and 16.4 on 256.
double tiling_us(const Product& q, const Tiling& t, int sms, double* tiles) {
  const int groups = std::min(q.experts, q.rows);
  const int per_group = (q.rows + groups - 1) / groups;
  const double m_tiles = q.experts == 1 ? (q.rows + t.tile_tokens - 1) / t.tile_tokens
                                        : std::max<double>(groups, static_cast<double>(q.rows) / t.tile_tokens +
                                                                       0.6 * groups);
  const int columns = std::min<long long>(t.tile_tokens, ((q.experts == 1 ? 1ll : 2ll) * per_group + 31) / 32 * 32);
  const int channels = (q.gated ? 64 : 128) * t.ctas;
  *tiles = m_tiles * ((q.n + channels - 1) / channels);
  const double loads = (128.0 + static_cast<double>(columns) / t.ctas) * 128.0 / 140e3;
  const double mmas = columns * 2.0 / 1900.0;
  const int chunks = columns / 32;
  const double epilogue = 0.6 + (q.gated ? 0.33 : 0.3) * chunks;
  const int k_tiles = (q.k + 127) / 128;
  const double steps = (k_tiles + t.split - 1) / t.split *
                       std::max(std::max(loads, mmas), t.sub == 2 ? 0.135 : 0.22);
  const double rounds = t.split > 1 ? 1.0 : std::ceil(*tiles / (sms / t.ctas));
  const double work = rounds * std::max(steps, epilogue) + std::min(steps, epilogue) +
                      (t.ctas == 2 ? 0.5 : 0.0) + (t.split > 1 ? 0.5 + 0.6 * chunks + 0.1 * t.split : 0.0);
  const double width = q.gated ? 2.0 * q.n : q.n;
  const double bytes = groups * width * q.k + static_cast<double>(q.rows) * (q.k + 2.0 * q.n);
  const double loaded = *tiles * k_tiles * (128.0 * t.ctas + columns) * 128.0;
  return std::max(work, bytes / 6e6) + 0.1 * loaded / 12e6;
}

Tiling choose_tiling(const Product& q, int sms) {
  const int groups = std::min(q.experts, q.rows);
  const int per_group = (q.rows + groups - 1) / groups;
  // Of groups a tile up to twice the average: what is larger takes several.
  const int widest = static_cast<int>(
      std::min<long long>(256, ((q.experts == 1 ? 1ll : 2ll) * per_group + 31) / 32 * 32));
  Tiling best{};
  double best_us = 0.0;
  for (int ctas = per_group > 32 ? 2 : 1; ctas >= 1; --ctas) {
    for (int tokens = widest; tokens >= 32 * ctas; tokens -= 32) {
      for (int split = 1; split <= (ctas == 1 ? 8 : 1); split *= 2) {
        const Tiling t{ctas, tokens, ctas == 1 || tokens <= 128 ? 2 : 1, split};
        double tiles = 0.0;
        const double us = tiling_us(q, t, sms, &tiles);
        // A split tile is a cluster's only one: all of them run at once.
        if (split > 1 && (split * 2 > (q.k + 127) / 128 || tiles > cluster_slots(split, sms))) break;
        if (best.ctas == 0 || us < best_us * 0.98) {
          best = t;
          best_us = us;
        }
      }
    }
  }
  return best;
}

int launch_product(const Product& q, void* stream) {
  if (int rc = check_product(q)) return rc;
  if (q.rows == 0) return 0;
  const int sms = host_sm_count();
  const Tiling tiling = choose_tiling(q, sms);
  const int ctas = tiling.ctas, tile_tokens = tiling.tile_tokens, split = tiling.split;
  const int channels = (q.gated ? 64 : 128) * ctas;
  const long long n_tiles = (q.n + channels - 1) / channels;
  // No routing makes more token tiles than this.
  const long long m_tiles = q.experts == 1 ? (q.rows + tile_tokens - 1) / tile_tokens
                                           : q.rows / tile_tokens + std::min(q.experts, q.rows);
  const long long tiles = m_tiles * n_tiles;
  if (tiles > (1ll << 31) - 1 - 1024) {  // and with a step of the walk behind them
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "too many tiles: %d rows, n=%d, %d experts", q.rows, q.n, q.experts);
  }

  Int8TileParams p{};
  const cuuint64_t half = static_cast<cuuint64_t>(q.n) * q.ldb;
  const cuuint64_t expert = q.experts > 1 ? static_cast<cuuint64_t>(q.expert_stride) : 2 * half;
  p.whole = q.gated && q.n % 16 == 0;
  if (p.whole) {
    const cuuint64_t dims[5] = {static_cast<cuuint64_t>(q.k), 16, 2, static_cast<cuuint64_t>(q.n) / 16,
                                static_cast<cuuint64_t>(q.experts)};
    const cuuint64_t strides[4] = {static_cast<cuuint64_t>(q.ldb), half,
                                   16 * static_cast<cuuint64_t>(q.ldb), expert};
    const cuuint32_t box[5] = {128, 16, 2, 4, 1};
    if (int rc = encode(&p.map_b, q.b, 5, dims, strides, box)) return rc;
  } else {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(q.k), static_cast<cuuint64_t>(q.n),
                                q.gated ? 2u : 1u, static_cast<cuuint64_t>(q.experts)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(q.ldb), half, expert};
    const cuuint32_t box[4] = {128, q.gated ? 16u : 128u, q.gated ? 2u : 1u, 1};
    if (int rc = encode(&p.map_b, q.b, 4, dims, strides, box)) return rc;
  }
  const cuuint64_t a_dims[2] = {static_cast<cuuint64_t>(q.k), static_cast<cuuint64_t>(q.rows)};
  const cuuint64_t a_strides[1] = {static_cast<cuuint64_t>(q.lda)};
  const cuuint32_t a_box[2] = {128, static_cast<cuuint32_t>(tile_tokens / ctas)};
  if (int rc = encode(&p.map_a, q.a, 2, a_dims, a_strides, a_box)) return rc;
  // Only a tile of fewer MMA columns than the others reads through the second map: the last one of a
  // dense product, any group's last one of a grouped product (of one expert, too).
  const int last = q.rows % tile_tokens;
  if (q.offsets != nullptr || (last != 0 && (last + 31) / 32 * 32 != tile_tokens)) {
    const cuuint32_t part_box[2] = {128, static_cast<cuuint32_t>(32 / ctas)};
    if (int rc = encode(&p.map_a_part, q.a, 2, a_dims, a_strides, part_box)) return rc;
  } else {
    p.map_a_part = p.map_a;
  }
  // 16-bit results leave through shared memory where the MMAs do not hide a store of 64 bytes a warp and
  // CTAs take several tiles: 8192 x 8192 x 64 takes 32.3 us against 38.6 with direct stores, k = 256 33.9
  // against 39.6, gated 4096 x 8192 x 256 45.3 against 47.5; k = 1024 56.8 against 57.7; k = 2048 92.8
  // against 91.1. A CTA's only tile gains nothing: 300 x 4096 x 256 4.9 us against 4.7. The copies
  // write 16 bytes at a time, so rows of D must start, follow and end on multiples of eight.
  const long long walkers = sms / ctas;
  const bool may_stage = q.out_kind != NVFP4_OUT_F32 && q.k <= 1024 && split == 1 && tiles > walkers &&
                         q.n % 8 == 0 && q.ldd % 8 == 0 && aligned(q.d, 16);
  const Int8Ring ring = int8_ring(ctas, tile_tokens, tiling.sub, q.k, q.experts, may_stage);
  p.staged = ring.staged;
  if (p.staged) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(q.n), static_cast<cuuint64_t>(q.rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(q.ldd) * 2};
    const cuuint32_t box[2] = {q.gated ? 16u : 32u, 32};
    if (int rc = encode(&p.map_d, q.d, 2, dims, strides, box, true)) return rc;
  }
  p.a_scales = q.a_scales;
  p.b_scales = q.b_scales;
  p.bias = q.bias;
  p.offsets = q.offsets;
  p.d = q.d;
  p.ldd = q.ldd;
  p.rows = q.rows;
  p.n = q.n;
  p.k = q.k;
  p.experts = q.experts;
  p.out_kind = q.out_kind;
  p.tile_tokens = tile_tokens;
  p.split = split;
  p.tmem_columns = 32;
  while (p.tmem_columns < (split > 1 ? 1 : 2) * tile_tokens) p.tmem_columns *= 2;
  p.stages = ring.stages;

  const TileKernel kernel = tile_kernel(ctas, tiling.sub, q.gated);
  CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                cudaFuncAttributeMaxDynamicSharedMemorySize, kInt8SharedLimit));
  const int group = split > 1 ? split : ctas;
  // A split tile is a cluster's only one; otherwise a CTA (or pair) on every SM walks the tiles.
  const long long groups = split > 1 ? tiles : std::min(tiles, walkers);
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = static_cast<unsigned int>(group);
  attribute[1].val.clusterDim.y = 1;
  attribute[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned int>(groups * group));
  config.blockDim = dim3(int8_threads(tile_tokens));
  config.dynamicSmemBytes = static_cast<size_t>(ring.bytes);
  config.stream = static_cast<cudaStream_t>(stream);
  config.attrs = attribute;
  config.numAttrs = group > 1 ? 2 : 1;
  void* args[1] = {&p};
  CUDA_TRY(cudaLaunchKernelExC(&config, reinterpret_cast<const void*>(kernel), args));
  return 0;
}

// Launches a row kernel with programmatic stream serialization: its blocks may take their places while
// the kernel before it ends (they wait on the device before they touch memory), and it lets the next
// one do so.
template <class Params>
void launch_rows(void (*kernel)(Params), int blocks, int threads, cudaStream_t stream, Params p) {
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned int>(blocks));
  config.blockDim = dim3(static_cast<unsigned int>(threads));
  config.stream = stream;
  config.attrs = attribute;
  config.numAttrs = 1;
  void* args[1] = {&p};
  // An error is the launch's own and reported by the caller's cudaGetLastError().
  (void)cudaLaunchKernelExC(&config, reinterpret_cast<const void*>(kernel), args);
}

// How rows of `width` elements lie over threads. A warp to a row up to `warp_width` elements, where there
// are rows enough; else a CTA. The quantiser in pieces of eight takes warps up to 1,024 elements (8192 x
// 1000: 5.9 us, with CTAs 9.1); the others only up to 256, since a lane with 32 elements and their
// 64-bit sums takes longer than a CTA's barriers (norms of 2900 x 370: 8.7 us, with warps 19; 8192 x 1000
// 15.5 and 17.7; 8192 x 101 7.7 and with CTAs 24; codes of 4000 x 945 6.2, with warps 8.1). In pieces of eight: few threads with much work where there are many
// rows (`elements` a thread: fewer, and the fixed cost of a row's reductions shows), many threads
// where there are too few to fill the SMs (a row's latency is what counts then). One at a time: 8
// elements a thread, or what 1,024 threads need.
struct RowGrid {
  int elements, threads, blocks;
  bool warp;
};

constexpr int kMaxRegisterRow = 32768;

RowGrid row_grid(int rows, int width, int p, int elements, int warp_width) {
  RowGrid g{};
  g.warp = width <= warp_width && rows > host_sm_count();
  if (g.warp) {
    g.elements = width <= 256 ? 8 : 32;
    g.threads = 32 * kWarpRows;
    g.blocks = (rows + kWarpRows - 1) / kWarpRows;
    return g;
  }
  g.elements = p == 8 && rows > 2 * host_sm_count() ? elements : 8;
  while ((width + g.elements - 1) / g.elements > 1024) g.elements *= 2;
  // One CTA of 1,024 threads on an SM is one row under way: two of 512 with twice the work.
  if (p == 8 && rows > 2 * host_sm_count() && g.elements == 16 && width > 8192) g.elements = 32;
  g.threads = ((width + g.elements - 1) / g.elements + 31) / 32 * 32;
  if (p == 1) {  // the shapes that there are kernels for
    if (g.elements > 8) {
      g.threads = 1024;
    } else if (g.threads > 768) {
      g.elements = 16;
      g.threads = 512;
    } else {
      g.threads = g.threads > 512 ? 768 : (g.threads + 127) / 128 * 128;
    }
  }
  g.blocks = rows;
  return g;
}

template <bool WIDE, int P>
void launch_quantize(const RowGrid& g, cudaStream_t s, const QuantizeParams& p) {
  constexpr int kWarps = 32 * kWarpRows;
  void (*kernel)(QuantizeParams);
  if (g.warp) {
    kernel = int8_quantize_kernel<WIDE, P, 8 / P, kWarps, true>;
    if constexpr (P == 8) {
      if (g.elements == 32) kernel = int8_quantize_kernel<WIDE, 8, 4, kWarps, true>;
    }
  } else if constexpr (P == 1) {
    kernel = g.threads == 128   ? int8_quantize_kernel<WIDE, 1, 8, 128, false>
             : g.threads == 256 ? int8_quantize_kernel<WIDE, 1, 8, 256, false>
             : g.threads == 384 ? int8_quantize_kernel<WIDE, 1, 8, 384, false>
             : g.threads == 768 ? int8_quantize_kernel<WIDE, 1, 8, 768, false>
             : g.elements == 8  ? int8_quantize_kernel<WIDE, 1, 8, 512, false>
             : g.threads == 512 ? int8_quantize_kernel<WIDE, 1, 16, 512, false>
             : g.elements == 16 ? int8_quantize_kernel<WIDE, 1, 16, 1024, false>
                                : int8_quantize_kernel<WIDE, 1, 32, 1024, false>;
  } else {
    kernel = g.elements == 8    ? int8_quantize_kernel<WIDE, 8, 1, 1024, false>
             : g.elements == 16 ? int8_quantize_kernel<WIDE, 8, 2, 1024, false>
             : g.threads <= 512 ? int8_quantize_kernel<WIDE, 8, 4, 512, false>
                                : int8_quantize_kernel<WIDE, 8, 4, 1024, false>;
  }
  launch_rows(kernel, g.blocks, g.threads, s, p);
}

template <bool X_WIDE, bool R_WIDE, int P>
void launch_norm(const RowGrid& g, cudaStream_t s, const NormParams& p) {
  constexpr int kWarps = 32 * kWarpRows;
  void (*kernel)(NormParams);
  if (g.warp) {
    kernel = residual_norm_kernel<X_WIDE, R_WIDE, P, 8 / P, kWarps, true>;
  } else if constexpr (P == 1) {
    kernel = g.threads == 128   ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 8, 128, false>
             : g.threads == 256 ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 8, 256, false>
             : g.threads == 384 ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 8, 384, false>
             : g.threads == 768 ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 8, 768, false>
             : g.elements == 8  ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 8, 512, false>
             : g.threads == 512 ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 16, 512, false>
             : g.elements == 16 ? residual_norm_kernel<X_WIDE, R_WIDE, 1, 16, 1024, false>
                                : residual_norm_kernel<X_WIDE, R_WIDE, 1, 32, 1024, false>;
  } else {
    kernel = g.elements == 8    ? residual_norm_kernel<X_WIDE, R_WIDE, 8, 1, 1024, false>
             : g.elements == 32 ? (g.threads <= 512 ? residual_norm_kernel<X_WIDE, R_WIDE, 8, 4, 512, false>
                                                    : residual_norm_kernel<X_WIDE, R_WIDE, 8, 4, 1024, false>)
             : g.threads <= 512 ? residual_norm_kernel<X_WIDE, R_WIDE, 8, 2, 512, false>
                                : residual_norm_kernel<X_WIDE, R_WIDE, 8, 2, 1024, false>;
  }
  launch_rows(kernel, g.blocks, g.threads, s, p);
}

template <int P>
void launch_norm(const RowGrid& g, cudaStream_t s, const NormParams& p) {
  const bool wide_r = p.residual != nullptr && p.residual_kind == NVFP4_IN_F32;
  if (p.x_kind == NVFP4_IN_F32) {
    if (wide_r) launch_norm<true, true, P>(g, s, p); else launch_norm<true, false, P>(g, s, p);
  } else {
    if (wide_r) launch_norm<false, true, P>(g, s, p); else launch_norm<false, false, P>(g, s, p);
  }
}

// Whether rows of `bytes`-sized elements, `pitch` elements apart, all start on a multiple of eight
// elements.
bool rows_in_eights(const void* p, long long pitch, int bytes, int rows) {
  return aligned(p, 8 * bytes) && (rows <= 1 || pitch % 8 == 0);
}

}  // namespace

extern "C" {

int nvfp4_int8_gemm(const void* a, long long lda, const void* b, long long ldb,
                    const float* a_scales, const float* b_scales, const float* bias, void* d,
                    long long ldd, int m, int n, int k, int out_kind, int gated, void* stream) {
  const Product q{a, b, a_scales, b_scales, bias, nullptr, d, lda, ldb, 0, ldd,
                  m, n, k, 1, out_kind, gated != 0};
  return launch_product(q, stream);
}

int nvfp4_int8_group_gemm(const void* a, long long lda, const void* b, long long ldb,
                          long long expert_stride, const float* a_scales, const float* b_scales,
                          const int* offsets, void* d, long long ldd, int experts, int rows, int n,
                          int k, int out_kind, int gated, void* stream) {
  if (offsets == nullptr && rows > 0) return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  const Product q{a, b, a_scales, b_scales, nullptr, offsets, d, lda, ldb, expert_stride, ldd,
                  rows, n, k, experts, out_kind, gated != 0};
  return launch_product(q, stream);
}

int nvfp4_int8_status(void* stream, int* status) {
  if (status == nullptr) return fail(NVFP4_E_INVALID_ARGUMENT, "null argument");
  *status = 0;
  void* word = nullptr;
  CUDA_TRY(cudaGetSymbolAddress(&word, g_int8_status));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int value = 0;
  CUDA_TRY(cudaMemcpyAsync(&value, word, sizeof(int), cudaMemcpyDeviceToHost, s));
  CUDA_TRY(cudaStreamSynchronize(s));
  *status = value;
  if (value == 0) return 0;
  CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), s));
  CUDA_TRY(cudaStreamSynchronize(s));
  return fail(NVFP4_E_DEVICE_TIMEOUT, "an INT8 product abandoned a bounded wait (code %d)", value);
}

int nvfp4_int8_quantize(const void* x, int x_kind, long long ldx, const int* source_rows, int rows,
                        int tokens, int k, void* q, long long ldq, float* scales, void* stream) {
  if (!is_in_kind(x_kind)) return fail(NVFP4_E_INVALID_ARGUMENT, "unknown input kind %d", x_kind);
  if (rows < 0 || rows > kMaxRows || tokens < 0 || tokens > kMaxRows || k < 1 || k > kMaxRows) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "unsupported tensor: %d rows of %d, k=%d (at most %d each)", rows,
                tokens, k, kMaxRows);
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
  const QuantizeParams p{x, source_rows, static_cast<int8_t*>(q), scales, ldx, ldq,
                         rows, tokens, k, x_kind};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (k > kMaxRegisterRow) {
    int8_quantize_long_kernel<<<rows, 1024, 0, s>>>(p);
  } else if (k % 8 == 0 && rows_in_eights(x, ldx, kind_bytes(x_kind), tokens) &&
             rows_in_eights(q, ldq, 1, rows)) {
    const RowGrid g = row_grid(rows, k, 8, 32, 1024);
    if (x_kind == NVFP4_IN_F32) launch_quantize<true, 8>(g, s, p); else launch_quantize<false, 8>(g, s, p);
  } else {
    const RowGrid g = row_grid(rows, k, 1, 32, 256);
    if (x_kind == NVFP4_IN_F32) launch_quantize<true, 1>(g, s, p); else launch_quantize<false, 1>(g, s, p);
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
  if (tokens < 0 || tokens > kMaxRows || hidden < 1 || hidden > kMaxHidden) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "unsupported rows: %d of %d (at most %d wide)", tokens,
                hidden, kMaxHidden);
  }
  if (!(eps >= kMinEps) || !(eps < 1e30)) {
    return fail(NVFP4_E_INVALID_ARGUMENT, "eps must be at least %g and below 1e30", kMinEps);
  }
  if (gate == nullptr && gates != 0) return fail(NVFP4_E_INVALID_ARGUMENT, "%d gates without a gate", gates);
  if (gate != nullptr && (gates < 1 || tokens % gates != 0)) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "%d tokens do not share %d gates evenly", tokens, gates);
  }
  if (tokens == 0) return 0;  // the addresses of empty tensors are null: the residual's says nothing here
  if (residual == nullptr &&
      (post_weight != nullptr || gate != nullptr || next_weight == nullptr || residual_scale != 1.0f)) {
    return fail(NVFP4_E_INVALID_ARGUMENT,
                "without a residual there is only the norm of x: no post weight, gate or scale");
  }
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
  p.inverse_hidden = 1.0 / hidden;
  p.x_kind = x_kind;
  p.residual_kind = residual_kind;
  p.y_kind = y_kind;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int y_bytes = y_kind == NVFP4_NORM_CODES ? 1 : kind_bytes(y_kind);
  const int r_bytes = static_cast<int>(residual_bytes);
  if (hidden % 8 == 0 && rows_in_eights(x, ldx, kind_bytes(x_kind), tokens) &&
      rows_in_eights(residual, ldres, r_bytes, tokens) &&
      rows_in_eights(r, ldr, r_bytes, tokens) && rows_in_eights(post_weight, 0, 4, 1) &&
      rows_in_eights(gate, hidden, 4, gates) &&
      (next_weight == nullptr || (rows_in_eights(next_weight, 0, 4, 1) && rows_in_eights(y, ldy, y_bytes, tokens)))) {
    launch_norm<8>(row_grid(tokens, hidden, 8, 16, 256), s, p);
  } else {
    launch_norm<1>(row_grid(tokens, hidden, 1, 16, 256), s, p);
  }
  CUDA_TRY(cudaGetLastError());
  return 0;
}

int nvfp4_moe_offsets(const int* counts, int experts, int* offsets, void* stream) {
  if (counts == nullptr || offsets == nullptr) return fail(NVFP4_E_INVALID_ARGUMENT, "null operand");
  if (experts < 1 || experts > kInt8MaxExperts) {
    return fail(NVFP4_E_UNSUPPORTED_SHAPE, "%d experts (at most %d)", experts, kInt8MaxExperts);
  }
  expert_offsets_kernel<<<1, kInt8MaxExperts, 0, static_cast<cudaStream_t>(stream)>>>(counts, experts,
                                                                                  offsets);
  CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // extern "C"
