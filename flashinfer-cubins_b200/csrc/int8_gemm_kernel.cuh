// Products of INT8 codes on the tensor cores, dense or over ragged groups of rows:
//   D[m][c] = out((float(sum_k A[m][k] B[c][k]) * a_scales[m]) * b_scales[c] + bias[c])
// and with a gate silu of that for gate channels times that for up channels.
//
// The tile lies on its side: channels (rows of B, the weights) are the MMA's 128 rows, tokens
// (rows of A) its columns. A few tokens then cost a narrow MMA instead of an empty tile, the
// weights stream through the wide operand, and in the epilogue a warp holds 32 neighbouring
// channels of one token at a time, which are neighbours in D: every store instruction of a warp
// is one run of 64 or 128 bytes, for any n, ldd and alignment. Products of a small depth, whose time
// is that of their results, stage 32 tokens of a warp's channels and store them by one copy.
//
// Warps of a CTA: 0 loads (one thread issues cp.async.bulk.tensor into a ring of
// stages of SUB pieces of 128 k), 1 issues tcgen05.mma.kind::i8 (32 k each) into one of two accumulators in
// tensor memory, the others take the other accumulator out, scale and store it. CTAS = 2: a pair of CTAs
// on neighbouring SMs works on 256 channel rows with tcgen05.mma.cta_group::2; each loads its own
// 128 rows of B and half of the tile's tokens.
//
// GATED: of a CTA's 128 rows every 32 are 16 gate channels and the same 16 up channels (the tensor
// map has gate and up as a dimension of its own, so one copy brings both). A warp of the epilogue
// then holds both of 16 channels, lanes 16 apart, and exchanges two tokens' values in one shuffle.
//
// SPLIT (cluster of `split` CTAs, one tile each cluster): each CTA takes a part of k, the partial
// sums meet in shared memory, and each CTA finishes a share of the tokens. The sums are integers:
// no order of them changes a bit.
#pragma once

#include <cuda.h>

#include "int8_kernels.cuh"
#include "int8_ring.h"

namespace nvfp4 {

// Token tiles that are walked together, channel tile by channel tile, for the L2 cache: 8192^3 takes 348,
// 340 and 333 us with bands of 4, 8 and 16, 32 experts of 4096 rows, gated 2048 x 7168, 183, 184 and 187.
constexpr int kInt8Band = 8;

struct Int8TileParams {
  // Weights: [experts][1][n][k], box 128 rows of 128 bytes. Gated: [experts][n / 16][2][16][k], box
  // 4 x 2 x 16 rows, or where n is no multiple of 16 [experts][2][n][k], box 2 x 16 rows.
  CUtensorMap map_b;
  CUtensorMap map_a;       // [rows][k], box of a whole tile's tokens (a pair: of half of them)
  CUtensorMap map_a_part;  // the same with a box of 32 (a pair: 16) rows
  CUtensorMap map_d;       // staged: 16-bit [rows][n], box 32 rows of a warp's 32 (gated: 16) channels
  const float* a_scales;
  const float* b_scales;
  const float* bias;
  const int* offsets;
  void* d;
  long long ldd;
  int rows, n, k, experts;
  int out_kind;
  int tile_tokens;  // a multiple of 32, at most 256
  int tmem_columns;
  int stages;
  int split;
  int whole;   // gated: one copy brings a stage's weights
  int staged;  // D leaves through shared memory
};

// Set to a role's code when it abandons a wait; read and cleared by nvfp4_int8_status.
__device__ int g_int8_status;
constexpr int kInt8ProducerTimeout = 1, kInt8MmaInputTimeout = 2, kInt8MmaAccumTimeout = 3,
              kInt8EpilogueTimeout = 4;

__device__ __forceinline__ void int8_give_up(volatile int* abort_flag, int code) {
  *abort_flag = 1;
  atomicCAS(&g_int8_status, 0, code);
}

// D[tmem] (+)= A[smem] B[smem]^T, signed bytes, 32-bit integer sums, K = 32.
template <int CTAS>
__device__ __forceinline__ void tc_mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b,
                                          uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 1) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Instruction descriptor of kind::i8: 32-bit integer D (2 in bits 4-5), signed A and B (1 in bits
// 7-9 and 10-12), K-major both, N and M in units of 8 and 16.
__host__ __device__ constexpr uint32_t i8_instr_desc(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Tiled copies into this CTA's shared memory; `bar` is this CTA's barrier, or with a pair the
// leader's (a shared::cluster address).
template <int CTAS>
__device__ __forceinline__ void tma_rows(uint32_t dst, const void* map, uint32_t bar, int k, int row) {
  if constexpr (CTAS == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(row)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(row)
        : "memory");
  }
}

template <int CTAS>
__device__ __forceinline__ void tma_weights(uint32_t dst, const void* map, uint32_t bar, int k,
                                            int channel, int expert) {
  if constexpr (CTAS == 1) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(channel), "r"(0), "r"(expert)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(channel), "r"(0), "r"(expert)
        : "memory");
  }
}

template <int CTAS>
__device__ __forceinline__ void tma_gated_weights(uint32_t dst, const void* map, uint32_t bar, int k,
                                                  int channel_group, int expert) {
  if constexpr (CTAS == 1) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(0), "r"(channel_group), "r"(expert)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(k), "r"(0), "r"(channel_group), "r"(expert)
        : "memory");
  }
}

template <int CTAS>
__device__ __forceinline__ void int8_commit(uint32_t bar) {
  if constexpr (CTAS == 1) {
    tc_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  }
}

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Stores a box from shared memory as part of the thread's current bulk group; what lies beyond the
// tensor is not written.
__device__ __forceinline__ void tma_store_rows(const void* map, uint32_t src, int channel, int row) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(channel), "r"(row)
               : "memory");
}

// 32 tokens of a warp's channels through its 2 KB of shared memory, a 16-bit value at a time: the
// addresses are constants apart, where a store to D needs one of its own.
template <typename T, int COLUMNS>
__device__ __forceinline__ void stage_columns(uint32_t to, uint32_t step, const float (&v)[COLUMNS]) {
#pragma unroll
  for (int i = 0; i < COLUMNS; ++i) {
    const T value = from_float<T>(v[i]);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(to + i * step),
                 "h"(*reinterpret_cast<const unsigned short*>(&value))
                 : "memory");
  }
}

struct Int8Tile {
  int expert;
  int m0;      // first token (row of A)
  int tokens;  // tokens of the tile, at most tile_tokens
  int columns; // tokens rounded up to the MMA's granularity of 32
  int n_tile;
};

// Stores `v` (token column values of this lane's channel) for tokens m, m + 1, ... while they are
// below `count`.
template <typename T, int COLUMNS>
__device__ __forceinline__ void store_columns(T* d, long long step, const float (&v)[COLUMNS], int count) {
  if (count >= COLUMNS) {
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) {
      *d = from_float<T>(v[i]);
      d += step;
    }
  } else {
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) {
      if (i < count) *d = from_float<T>(v[i]);
      d += step;
    }
  }
}

template <int CTAS, int SUB, bool GATED>
__global__ void __launch_bounds__(64 + 128 * kInt8MaxParts, 1)
int8_tile_kernel(const __grid_constant__ Int8TileParams p) {
  extern __shared__ uint8_t dyn_smem[];
  __shared__ alignas(8) uint64_t bar_full[kInt8MaxStages];
  __shared__ alignas(8) uint64_t bar_empty[kInt8MaxStages];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(16) float scale_stage[4 * kInt8MaxParts][64];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(dyn_smem) + 1023u) & ~1023u;
  const uint32_t rank = (CTAS == 2 || p.split > 1) ? cluster_cta_rank() : 0u;
  const bool leader = CTAS == 1 || rank == 0;
  const int tile_tokens = p.tile_tokens;
  const int stages = p.stages;
  const int parts = (static_cast<int>(blockDim.x) - 64) / 128;  // warps that share a quarter
  constexpr int channels = GATED ? 64 : 128;  // output channels of a CTA
  constexpr uint32_t weight_bytes = 128u * 128u;  // of a piece of 128 k
  const uint32_t token_bytes = static_cast<uint32_t>(tile_tokens / CTAS) * 128u;
  const uint32_t stage_bytes = SUB * (weight_bytes + token_bytes);
  // Behind the stages: the epilogue warps' staging, if any; for every expert the token tiles of those
  // before it, and its first row.
  const uint32_t staging = smem_base + stages * stage_bytes;
  int* tiles_before = reinterpret_cast<int*>(dyn_smem + (staging - smem_u32(dyn_smem)) +
                                             (p.staged ? 4 * parts * kInt8StagedBytes : 0u));
  int* first_row = tiles_before + p.experts + 1;
  const uint32_t tmem_cols = p.tmem_columns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1);
      mbar_init(smem_u32(&bar_acc_empty[i]), 4 * parts * CTAS);
    }
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {  // the maps are launch parameters: nothing to wait for
    prefetch_tensormap(&p.map_b);
    prefetch_tensormap(&p.map_a);
    prefetch_tensormap(&p.map_a_part);
  }
  if (warp == 1) {
    if constexpr (CTAS == 1) {
      tmem_alloc(smem_u32(&tmem_base_slot), tmem_cols);
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(&tmem_base_slot)),
                   "r"(tmem_cols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  // What the kernel before writes is read behind this, by plain loads: the read-only path (__ldg) is for
  // memory that nothing writes while the kernel is resident, and this one may be resident early.
  grid_dependency_wait();
  grid_launch_dependents();
  if (warp == 0) {
    // First rows: the offsets cut to [0, rows], and where they decrease their running maximum, so
    // that no value of theirs makes groups overlap or reach outside. Then a prefix over the
    // experts' token tiles.
    int before = 0, last_row = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + lane;
      int row = e < p.experts ? (p.offsets != nullptr ? p.offsets[e] : 0) : 0;
      int next = e < p.experts ? (p.offsets != nullptr ? p.offsets[e + 1] : p.rows) : 0;
      row = min(max(row, last_row), p.rows);
      next = min(max(next, row), p.rows);
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int other = __shfl_up_sync(0xFFFFFFFFu, next, d);
        if (lane >= d) next = max(next, other);
      }
      const int previous = __shfl_up_sync(0xFFFFFFFFu, next, 1);
      row = lane == 0 ? row : previous;
      int tiles = e < p.experts ? (next - row + tile_tokens - 1) / tile_tokens : 0;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int other = __shfl_up_sync(0xFFFFFFFFu, tiles, d);
        if (lane >= d) tiles += other;
      }
      if (e == 0) first_row[0] = row;
      if (e < p.experts) {
        first_row[e + 1] = next;
        tiles_before[e + 1] = before + tiles;
      }
      before += __shfl_sync(0xFFFFFFFFu, tiles, 31);
      last_row = __shfl_sync(0xFFFFFFFFu, next, 31);
    }
    if (lane == 0) tiles_before[0] = 0;
  }
  tc_fence_before_sync();
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();  // the peer's barriers and tensor memory exist
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_slot;
  volatile int* abort_ptr = &abort_flag;

  const int m_tiles = tiles_before[p.experts];
  const int n_tiles = (p.n + channels * CTAS - 1) / (channels * CTAS);
  // 32 bits hold every tile's number (the host checks): the divisions below are done by every warp for
  // every tile, and 64-bit ones cost 8192 x 8192 x 64 0.9 us.
  const uint32_t tiles = static_cast<uint32_t>(m_tiles) * static_cast<uint32_t>(n_tiles);
  const int group = p.split > 1 ? p.split : CTAS;  // CTAs that share a tile
  const uint32_t first_tile = blockIdx.x / group;
  const uint32_t step = gridDim.x / group;
  const int k_tiles = (p.k + 127) / 128;
  const int kt0 = p.split > 1 ? static_cast<int>(rank) * k_tiles / p.split : 0;
  const int kt1 = p.split > 1 ? (static_cast<int>(rank) + 1) * k_tiles / p.split : k_tiles;

  bool partials_written = false;  // a split tile's epilogue has passed the cluster's first barrier

  auto decode = [&](uint32_t t) {
    Int8Tile tile;
    const uint32_t band_tiles = kInt8Band * static_cast<uint32_t>(n_tiles);
    const uint32_t band = t / band_tiles;
    const uint32_t in_band = t - band * band_tiles;
    const uint32_t height = min(kInt8Band, m_tiles - static_cast<int>(band) * kInt8Band);
    const uint32_t across = in_band / height;
    const int m_tile = static_cast<int>(band * kInt8Band + in_band - across * height);
    tile.n_tile = static_cast<int>(across);
    // The last expert whose first tile is not behind m_tile, and that has tiles.
    int lo = 0, hi = p.experts;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tiles_before[mid] <= m_tile) lo = mid; else hi = mid;
    }
    tile.expert = lo;
    tile.m0 = first_row[lo] + (m_tile - tiles_before[lo]) * tile_tokens;
    tile.tokens = min(tile_tokens, first_row[lo + 1] - tile.m0);
    tile.columns = (tile.tokens + 31) & ~31;
    return tile;
  };

  // Where a tile begins in k (it goes round): a single CTA's channel tiles begin in different places, so
  // that the SMs do not all read the same columns of rows a power of two apart (one token: 8192 x 8192
  // 16.1 us from the start of k, 15.0 so; 16384 x 8192 25.3 and 23.4). Pairs work on more tokens and are
  // not bound by memory; the loops are shorter without it.
  constexpr bool kRound = CTAS == 1;
  auto first_piece = [&](const Int8Tile& tile) {
    if constexpr (!kRound) return kt0;
    const uint32_t steps = static_cast<uint32_t>(kt1 - kt0 + SUB - 1) / SUB;
    return kt0 + static_cast<int>(static_cast<uint32_t>(tile.n_tile) * 5u % steps) * SUB;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    // One thread runs the whole loop, here and in the MMA warp: electing it anew at every step cost
    // 70 clocks of a step's 430.
    if (elect_one()) {
      const uint32_t full0 = CTAS == 1 ? smem_u32(&bar_full[0])
                                       : cluster_map_shared(smem_u32(&bar_full[0]), 0);
      const uint32_t empty0 = smem_u32(&bar_empty[0]);
      int stage = 0;
      uint32_t phase = 1;
      uint32_t w_dst = smem_base;
      bool ok = true;
      for (uint32_t t = first_tile; ok && t < tiles; t += step) {
        const Int8Tile tile = decode(t);
        const int channel0 = (tile.n_tile * CTAS + static_cast<int>(CTAS == 2 ? rank : 0)) * channels;
        const int share = tile.columns / CTAS;  // tokens this CTA loads
        const int token0 = tile.m0 + static_cast<int>(CTAS == 2 ? rank : 0) * share;
        const uint32_t bytes = CTAS * (weight_bytes + static_cast<uint32_t>(share) * 128u);
        int kt = first_piece(tile);
        for (int i0 = kt0; i0 < kt1; i0 += SUB) {
          if (!mbar_wait(empty0 + 8 * stage, phase, abort_ptr)) {
            int8_give_up(abort_ptr, kInt8ProducerTimeout);
            ok = false;
            break;
          }
          const uint32_t bar = full0 + 8 * stage;
          const uint32_t bar_here = smem_u32(&bar_full[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
          const int parts = SUB == 1 ? 1 : min(SUB, kt1 - kt);
          if (leader) mbar_expect_tx(bar_here, parts * bytes);
          uint32_t w = w_dst, r = w_dst + SUB * weight_bytes;
#pragma unroll
          for (int i = 0; i < SUB; ++i) {
            if (i >= parts) break;
            const int k = (kt + i) * 128;
            if (GATED && p.whole) {
              tma_gated_weights<CTAS>(w, &p.map_b, bar, k, channel0 / 16, tile.expert);
            } else if constexpr (GATED) {
#pragma unroll
              for (int j = 0; j < channels; j += 16) {
                tma_weights<CTAS>(w + 256 * j, &p.map_b, bar, k, channel0 + j, tile.expert);
              }
            } else {
              tma_weights<CTAS>(w, &p.map_b, bar, k, channel0, tile.expert);
            }
            if (tile.columns == tile_tokens) {
              tma_rows<CTAS>(r, &p.map_a, bar, k, token0);
            } else {
              for (int c = 0; c < share; c += 32 / CTAS) {
                tma_rows<CTAS>(r + c * 128, &p.map_a_part, bar, k, token0 + c);
              }
            }
            w += weight_bytes;
            r += token_bytes;
          }
          kt += SUB;
          if (kRound && kt >= kt1) kt = kt0;
          w_dst = stage == 0 ? smem_base : w_dst + stage_bytes;
        }
      }
    }
    __syncwarp();
    if (*abort_ptr != 0) {
      // Copies may still be on their way into this CTA's memory: let them land.
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (leader && elect_one()) {
      constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t lo0 = ((smem_base >> 4) & 0x3FFFu) | (1u << 16);
      const uint32_t full0 = smem_u32(&bar_full[0]);
      const uint32_t empty0 = smem_u32(&bar_empty[0]);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t acc = 0, acc_phase = 1;
      uint32_t lo_w = lo0;
      bool ok = true;
      for (uint32_t t = first_tile; ok && t < tiles; t += step) {
        const Int8Tile tile = decode(t);
        const uint32_t idesc = i8_instr_desc(128 * CTAS, static_cast<uint32_t>(tile.columns));
        if (!mbar_wait(smem_u32(&bar_acc_empty[acc]), acc_phase, abort_ptr)) {
          int8_give_up(abort_ptr, kInt8MmaAccumTimeout);
          break;
        }
        tc_fence_after_sync();
        const uint32_t d = tmem_base + acc * tile_tokens;
        uint32_t accumulate = 0;
        int kt = first_piece(tile);
        for (int i0 = kt0; i0 < kt1; i0 += SUB) {
          if (!mbar_wait(full0 + 8 * stage, phase, abort_ptr)) {
            int8_give_up(abort_ptr, kInt8MmaInputTimeout);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t empty = empty0 + 8 * stage;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
          uint32_t w = lo_w, r = lo_w + SUB * (weight_bytes >> 4);
#pragma unroll
          for (int i = 0; i < SUB; ++i) {
            // k of the last piece beyond the depth is zero in both operands and not multiplied.
            const int left = min(p.k, kt1 * 128) - (kt + i) * 128;
            if (left > 96) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                tc_mma_i8<CTAS>(d, pack_desc(w + 2 * j, kHi), pack_desc(r + 2 * j, kHi), idesc,
                                j > 0 ? 1u : accumulate);
              }
            } else {
              for (int j = 0; j * 32 < left; ++j) {
                tc_mma_i8<CTAS>(d, pack_desc(w + 2 * j, kHi), pack_desc(r + 2 * j, kHi), idesc,
                                j > 0 ? 1u : accumulate);
              }
            }
            accumulate = 1;
            w += weight_bytes >> 4;
            r += token_bytes >> 4;
          }
          kt += SUB;
          if (kRound && kt >= kt1) kt = kt0;
          int8_commit<CTAS>(empty);
          lo_w = stage == 0 ? lo0 : lo_w + (stage_bytes >> 4);
        }
        if (!ok) break;
        int8_commit<CTAS>(smem_u32(&bar_acc_full[acc]));
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    const int part = (warp - 2) / 4;  // this warp's chunks of 32 tokens: part, part + parts, ...
    float* sa_stage = scale_stage[warp - 2];
    const uint32_t leader_acc_empty0 = CTAS == 1 ? smem_u32(&bar_acc_empty[0])
                                                 : cluster_map_shared(smem_u32(&bar_acc_empty[0]), 0);
    // A tile as this lane sees it: its row of B is a channel of D and has a scale and a bias; its
    // tokens are all of the tile's, or with a split this CTA's share, and the warp's two chunks of them
    // have a scale each lane.
    struct Share {
      Int8Tile tile;
      int channel, c_begin, c_end;
      float sb, bias, sa[2];
    };
    auto share_of = [&](uint32_t t) {
      Share s;
      s.tile = decode(t);
      const int channel0 = (s.tile.n_tile * CTAS + static_cast<int>(CTAS == 2 ? rank : 0)) * channels;
      s.channel = GATED ? channel0 + quarter * 16 + (lane & 15) : channel0 + quarter * 32 + lane;
      const bool live = s.channel < p.n;
      const int width = GATED ? 2 * p.n : p.n;
      const int row = GATED && lane >= 16 ? p.n + s.channel : s.channel;
      s.sb = live ? p.b_scales[static_cast<long long>(s.tile.expert) * width + row] : 0.0f;
      s.bias = live && p.bias != nullptr ? p.bias[row] : 0.0f;
      s.c_begin = p.split > 1 ? s.tile.columns * static_cast<int>(rank) / p.split : 0;
      s.c_end = min(p.split > 1 ? s.tile.columns * (static_cast<int>(rank) + 1) / p.split : s.tile.columns,
                    s.tile.tokens);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = s.c_begin + 32 * (part + i * parts) + lane;
        s.sa[i] = c < s.c_end ? p.a_scales[s.tile.m0 + c] : 0.0f;
      }
      return s;
    };
    uint32_t acc = 0, acc_phase = 0;
    Share next{};
    if (first_tile < tiles) next = share_of(first_tile);
    for (uint32_t t = first_tile; t < tiles; t += step) {
      const Int8Tile tile = next.tile;
      const int channel = next.channel, c_begin = next.c_begin, c_end = next.c_end;
      const bool live = channel < p.n;
      const float sb = next.sb, bias = next.bias;
      sa_stage[lane] = next.sa[0];
      sa_stage[32 + lane] = next.sa[1];
      // The next tile's scales are on their way while this tile's MMAs run and its results leave: with
      // each tile fetching its own 8192 x 8192 x 256 took 38.6 us, so 34.7.
      if (t + step < tiles) next = share_of(t + step);
      __syncwarp();
      if (!mbar_wait(smem_u32(&bar_acc_full[acc]), acc_phase, abort_ptr)) {
        int8_give_up(abort_ptr, kInt8EpilogueTimeout);
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * tile_tokens;
      if (p.split > 1) {
        // Partial sums to shared memory (the stages are free: every MMA that read them is done),
        // [token][channel row]; after the cluster's barrier each CTA adds up its share of tokens.
        for (int c = 32 * part; c < tile.columns; c += 32 * parts) {
          uint32_t r[32];
          tmem_load_32(taddr + c, r);
          tmem_load_wait();
          const uint32_t to = smem_base + static_cast<uint32_t>(c * 128 + quarter * 32 + lane) * 4u;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + i * 512), "r"(r[i]) : "memory");
          }
        }
        cluster_sync_all();
        partials_written = true;
      }
      const float* sa_next = sa_stage;
      for (int c = c_begin + 32 * part; c < c_end; c += 32 * parts, sa_next += 32) {
        const int count = min(c_end - c, 32);
        uint32_t r[32];
        if (p.split > 1) {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
          // Eight tokens at a time from all parts, the loads of four parts under way together (3 x 96 x
          // 6832 split in eight: one part after the other 9.5 us, this 6.4).
#pragma unroll
          for (int i0 = 0; i0 < 32; i0 += 8) {
            if (i0 >= count) break;
#pragma unroll 4
            for (int s = 0; s < p.split; ++s) {
              const uint32_t from = cluster_map_shared(
                  smem_base + static_cast<uint32_t>((c + i0) * 128 + quarter * 32 + lane) * 4u, s);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (i0 + i < count) r[i0 + i] += static_cast<uint32_t>(ld_cluster_s32(from + i * 512));
              }
            }
          }
        } else {
          tmem_load_32(taddr + c, r);
          tmem_load_wait();
        }
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 sa = *reinterpret_cast<const float4*>(sa_next + i);
          const float2 sb2 = make_float2(sb, sb);
          const float2 x = make_float2(static_cast<float>(static_cast<int>(r[i])),
                                       static_cast<float>(static_cast<int>(r[i + 1])));
          const float2 z = make_float2(static_cast<float>(static_cast<int>(r[i + 2])),
                                       static_cast<float>(static_cast<int>(r[i + 3])));
          const float2 low = product2(product2(x, make_float2(sa.x, sa.y)), sb2);
          const float2 high = product2(product2(z, make_float2(sa.z, sa.w)), sb2);
          v[i] = low.x;
          v[i + 1] = low.y;
          v[i + 2] = high.x;
          v[i + 3] = high.y;
        }
        if (p.bias != nullptr) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __fadd_rn(v[i], bias);
        }
        if constexpr (GATED) {
          // Of tokens 2i and 2i + 1 the gate lanes finish the first, the up lanes the second, by one
          // silu: with one for each side 4096 x 8192 x 256 takes 54.6 us, this 45.0.
          float y[16];
          const bool up_lane = lane >= 16;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float mine = up_lane ? v[2 * i + 1] : v[2 * i];
            const float other = __shfl_xor_sync(0xFFFFFFFFu, up_lane ? v[2 * i] : v[2 * i + 1], 16);
            y[i] = silu(up_lane ? other : mine) * (up_lane ? mine : other);
          }
          const int parity = up_lane ? 1 : 0;
          if (p.staged && count == 32) {
            // A token's 16 channels are 32 bytes of the box.
            const uint32_t box = staging + static_cast<uint32_t>(warp - 2) * kInt8StagedBytes;
            const uint32_t to = box + static_cast<uint32_t>(parity * 32 + (lane & 15) * 2);
            if (lane == 0) bulk_wait_group_read_all();
            __syncwarp();
            if (p.out_kind == 0) {
              stage_columns<__half>(to, 64, y);
            } else {
              stage_columns<__nv_bfloat16>(to, 64, y);
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && channel < p.n) {
              tma_store_rows(&p.map_d, box, channel, tile.m0 + c);
              bulk_commit_group();
            }
            continue;
          }
          const long long first = (tile.m0 + c + parity) * p.ldd + channel;
          const int mine = live ? (count - parity + 1) / 2 : 0;
          if (p.out_kind == 0) {
            store_columns(static_cast<__half*>(p.d) + first, 2 * p.ldd, y, mine);
          } else if (p.out_kind == 1) {
            store_columns(static_cast<float*>(p.d) + first, 2 * p.ldd, y, mine);
          } else {
            store_columns(static_cast<__nv_bfloat16*>(p.d) + first, 2 * p.ldd, y, mine);
          }
        } else {
          if (p.staged && count == 32) {
            const uint32_t box = staging + static_cast<uint32_t>(warp - 2) * kInt8StagedBytes;
            const uint32_t to = box + static_cast<uint32_t>(lane * 2);
            if (lane == 0) bulk_wait_group_read_all();
            __syncwarp();
            if (p.out_kind == 0) {
              stage_columns<__half>(to, 64, v);
            } else {
              stage_columns<__nv_bfloat16>(to, 64, v);
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0 && channel < p.n) {
              tma_store_rows(&p.map_d, box, channel, tile.m0 + c);
              bulk_commit_group();
            }
            continue;
          }
          const long long first = (tile.m0 + c) * p.ldd + channel;
          const int mine = live ? count : 0;
          if (p.out_kind == 0) {
            store_columns(static_cast<__half*>(p.d) + first, p.ldd, v, mine);
          } else if (p.out_kind == 1) {
            store_columns(static_cast<float*>(p.d) + first, p.ldd, v, mine);
          } else {
            store_columns(static_cast<__nv_bfloat16*>(p.d) + first, p.ldd, v, mine);
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();  // also: every lane has read this tile's scales
      if (lane == 0) {
        if constexpr (CTAS == 1) {
          mbar_arrive(leader_acc_empty0 + 8 * acc);
        } else {
          mbar_arrive_peer(leader_acc_empty0 + 8 * acc);
        }
      }
      acc ^= 1u;
      if (acc == 0) acc_phase ^= 1u;
    }
    // The staging outlives the last stores' reads of it.
    if (p.staged && lane == 0) bulk_wait_group_read_all();
  }

  tc_fence_before_sync();
  __syncwarp();
  if (p.split > 1) {
    // Two phases of the cluster's barrier, in every thread: the partial sums are written; they are
    // read. An epilogue warp with a tile has passed the first above.
    if (!partials_written) cluster_sync_all();
    cluster_sync_all();
  }
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();  // neither CTA frees tensor memory while the pair is in use
  if (warp == 1) {
    tc_fence_after_sync();
    __syncwarp();
    if constexpr (CTAS == 1) {
      tmem_dealloc(tmem_base, tmem_cols);
    } else {
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "r"(tmem_cols)
                   : "memory");
    }
  }
}

}  // namespace nvfp4
