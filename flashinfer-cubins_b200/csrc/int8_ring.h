// Shared memory of the INT8 products' kernel: a ring of stages that the loads fill ahead of the MMAs, the
// epilogue's staging and the experts' tables. Host arithmetic, without CUDA.
#pragma once

namespace nvfp4 {

// Epilogue warps: four (one for each quarter of tensor memory's lanes) for every 32 tokens of a tile,
// up to sixteen. A tile of 256 tokens then leaves in two rounds of 32 tokens a warp; with four warps
// the epilogue took longer than the MMAs of 4096 k (gated 1000 x 14336 x 4096: 153 us, now 82), and
// warps without work only poll.
constexpr int kInt8MaxParts = 4;
constexpr int int8_parts(int tile_tokens) {
  return tile_tokens / 32 < kInt8MaxParts ? tile_tokens / 32 : kInt8MaxParts;
}
constexpr int int8_threads(int tile_tokens) { return 64 + 128 * int8_parts(tile_tokens); }
constexpr int kInt8MaxStages = 12;
constexpr int kInt8MaxExperts = 1024;
// 32 tokens of a warp's channels as 16-bit results, on their way to a copy.
constexpr unsigned int kInt8StagedBytes = 2048;

// What a block can have of shared memory, less the kernels' static share (barriers and the epilogue's
// scales, 4.4 KB) and the slack that aligns the stages to 1,024 bytes.
constexpr int kInt8SharedLimit = 232448 - 5 * 1024;

struct Int8Ring {
  int stages, bytes;  // bytes: of dynamic shared memory, the slack included
  bool staged;        // results leave through shared memory
};

// The ring of a tile of `tile_tokens` on `ctas` CTAs with `sub` pieces of 128 k in a stage. `may_stage`:
// staging the results is possible and pays where a ring remains.
//
// Staging takes up to 32 KB. A single CTA's tile of 256 tokens keeps two stages of 256 k without it and
// one with it, where loads and MMAs take turns: 5053 x 6512 x 857 53.7 us with one stage, 38.2 with two and
// direct stores; 7242 x 944 x 835 gated 30.3 and 22.8. A tile whose k is one stage loses nothing by it:
// 6036 x 1496 x 229 10.8 us staged, 11.6 with direct stores; 2402 x 7400 x 61 13.5 and 15.7.
constexpr Int8Ring int8_ring(int ctas, int tile_tokens, int sub, int k, int experts, bool may_stage) {
  const int stage = sub * 128 * (128 + tile_tokens / ctas);
  const int tables = 8 * (experts + 1);
  const int staging = 4 * int8_parts(tile_tokens) * static_cast<int>(kInt8StagedBytes);
  const int room = kInt8SharedLimit - 1024 - tables;
  const int left = (room - staging) / stage;
  const bool staged = may_stage && (left >= 2 || (left == 1 && k <= sub * 128));
  const int fit = staged ? left : room / stage;
  const int stages = fit < kInt8MaxStages ? fit : kInt8MaxStages;
  return {stages, 1024 + stages * stage + tables + (staged ? staging : 0), staged};
}

}  // namespace nvfp4
