// How a product of the dense operators is cut into launches: which kernel, tiles, stages and the split of the k axis.
// Host arithmetic only, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "dense_types.h"

namespace fdmoe {

constexpr int kStreamSmemTwo = 112 * 1024;    // dynamic shared memory of a CTA when two share an SM (228 KB, 1 KB each reserved)
constexpr int kStreamSmemOne = 226 * 1024;
constexpr int kStreamSlack = 1024;            // for the alignment of the stages

struct StreamPlan {
  int tile_tokens, token_tiles, row_tiles, split, stages, smem, tmem_cols, per_sm;
};

inline int RoundUp(int v, int m) { return (v + m - 1) / m * m; }

// `rows` weight rows (gated: of each projection), `tokens` >= 1, `kblocks` stages of k in all.
inline StreamPlan MakeStreamPlan(int rows, int tokens, int kblocks, bool gated, bool mx4, int sms) {
  StreamPlan s;
  const int parts = gated ? 2 : 1;
  s.token_tiles = (tokens + FDMOE_STREAM_TOKENS - 1) / FDMOE_STREAM_TOKENS;
  s.tile_tokens = s.token_tiles > 1 ? FDMOE_STREAM_TOKENS : RoundUp(tokens, 16);
  s.row_tiles = (rows + FDMOE_STREAM_ROWS - 1) / FDMOE_STREAM_ROWS;
  const int stage = parts * 16384 + s.tile_tokens * 128 + (mx4 ? (parts + 1) * 1024 : 0);
  const int sums = std::min(tokens, s.tile_tokens) * parts * 512;  // partial sums, in the stages' place
  // Two CTAs per SM hide each other's beginning and end, if three stages each are left.
  s.per_sm = (kStreamSmemTwo - kStreamSlack) / stage >= 3 && sums <= kStreamSmemTwo - kStreamSlack ? 2 : 1;
  const int room = (s.per_sm == 2 ? kStreamSmemTwo : kStreamSmemOne) - kStreamSlack;
  // Time in units of one k block on a full GPU: a CTA's k blocks and its beginning and end, times the waves.
  double best = 0;
  s.split = 1;
  for (int n = 1; n <= FDMOE_STREAM_SPLIT && n <= kblocks; ++n) {
    const int64_t ctas = (int64_t)s.row_tiles * s.token_tiles * n, slots = (int64_t)sms * s.per_sm;
    const double t = (double)((ctas + slots - 1) / slots) * ((kblocks + n - 1) / n + 6);
    if (n == 1 || t < best) best = t, s.split = n;
  }
  s.stages = std::min(std::min(room / stage, (int)FDMOE_STREAM_STAGES), (kblocks + s.split - 1) / s.split);
  const int scales = mx4 ? (parts + 1) * 8 : 0;  // TMEM columns per stage
  const int cols_max = s.per_sm == 2 ? 256 : 512;
  if (scales) s.stages = std::min(s.stages, (cols_max - parts * s.tile_tokens) / scales);
  const int cols = parts * s.tile_tokens + s.stages * scales;
  s.tmem_cols = 32;
  while (s.tmem_cols < cols) s.tmem_cols *= 2;
  s.smem = std::max(s.stages * stage, sums) + kStreamSlack;
  return s;
}

// Whether the streaming kernel takes a product instead of the pair kernel.
inline bool UseStream(int tokens) { return tokens <= FDMOE_STREAM_TOKENS; }

inline size_t AlignBytes(size_t v) { return (v + 255) / 256 * 256; }

// 512-byte blocks of scales per 128 rows: an even number, as many as the stages of 256 columns take.
inline int64_t ScaleChunks(int64_t cols) { return (cols + FDMOE_MX4_STAGE_K - 1) / FDMOE_MX4_STAGE_K * 2; }
inline size_t ScaleBytes(int64_t batch, int64_t rows, int64_t cols) {
  return (size_t)(batch * ((rows + 127) / 128) * ScaleChunks(cols) * 512);
}

}  // namespace fdmoe
