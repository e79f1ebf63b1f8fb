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

// What the device runs at once: clusters of n CTAs of the streaming kernel with one or two CTAs per SM, and of the
// pair kernel with n pairs.  A GPC's SMs hold whole clusters only, so these are fewer than the SMs would give.
struct DeviceSlots {
  int stream_one[FDMOE_STREAM_SPLIT + 1], stream_two[FDMOE_STREAM_SPLIT + 1], pair[FDMOE_PAIR_SPLIT + 1];
};

// `rows` weight rows (gated: of each projection), `tokens` >= 1, `kblocks` stages of k in all.
inline StreamPlan MakeStreamPlan(int rows, int tokens, int kblocks, bool gated, bool mx4, const DeviceSlots& dev) {
  StreamPlan s;
  const int parts = gated ? 2 : 1;
  s.token_tiles = (tokens + FDMOE_STREAM_TOKENS - 1) / FDMOE_STREAM_TOKENS;
  s.tile_tokens = s.token_tiles > 1 ? FDMOE_STREAM_TOKENS : RoundUp(tokens, 16);
  s.row_tiles = (rows + FDMOE_STREAM_ROWS - 1) / FDMOE_STREAM_ROWS;
  const int stage = parts * 16384 + s.tile_tokens * 128 + (mx4 ? (parts + 1) * 1024 : 0);
  // Partial sums, in the stages' place: groups of four tokens, the same number for every CTA of the cluster.
  const int sums = (RoundUp(std::min(tokens, s.tile_tokens), 4) + 4 * (FDMOE_STREAM_SPLIT - 1)) * parts * 512;
  // Two CTAs per SM hide each other's beginning and end, if three stages each are left.
  s.per_sm = (kStreamSmemTwo - kStreamSlack) / stage >= 3 && sums <= kStreamSmemTwo - kStreamSlack ? 2 : 1;
  const int room = (s.per_sm == 2 ? kStreamSmemTwo : kStreamSmemOne) - kStreamSlack;
  // Time in cycles: a k block takes as long as its MMAs' issue or, with `active` CTAs reading weights at once, its share
  // of the memory's 3500 bytes per cycle; a wave has a beginning and an end.
  const double weights = parts * (mx4 ? 16384 + 1024 : 16384), issue = mx4 ? 400 + 250 * parts : 300 + 150 * parts;
  double best = 0;
  s.split = 1;
  for (int n = 1; n <= FDMOE_STREAM_SPLIT && n <= kblocks; ++n) {
    const int64_t slots = std::max(1, s.per_sm == 2 ? dev.stream_two[n] : dev.stream_one[n]);
    double t = 0;
    int64_t clusters = (int64_t)s.row_tiles * s.token_tiles;
    for (int wave = 0; clusters > 0 && wave < 64; ++wave, clusters -= slots) {
      const double active = (double)std::min(clusters, slots) * n;
      t += (double)((kblocks + n - 1) / n) * std::max(issue, active * weights / 3500) + 5000;
    }
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

struct PairPlan {
  int tile_n, split, tiles_m, tiles_n, clusters;
};

// `cols`: of the result; `kblocks` stages of k.  Time in cycles: the waves of tiles, each its k blocks' MMAs, and once
// per launch (per cluster where pairs share a tile) its beginning and end.
inline PairPlan MakePairPlan(int64_t rows, int64_t cols, int kblocks, bool gated, bool mx4, const DeviceSlots& dev) {
  PairPlan best = {};
  double best_time = 0;
  for (int tile_n = 256; tile_n >= (mx4 ? 256 : 128); tile_n -= gated ? 128 : 64)  // whole groups of 64 result columns
    for (int split = 1; split <= FDMOE_PAIR_SPLIT && split <= kblocks; split *= 2) {
      PairPlan p;
      p.tile_n = tile_n;
      p.split = split;
      p.tiles_m = (int)((rows + FDMOE_PAIR_TILE - 1) / FDMOE_PAIR_TILE);
      const int tile_cols = gated ? tile_n / 2 : tile_n;
      p.tiles_n = (int)((cols + tile_cols - 1) / tile_cols);
      const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, slots = std::max(1, dev.pair[split]);
      const double waves = (double)((tiles + slots - 1) / slots);
      const double block = tile_n == 256 ? 512 : tile_n == 192 ? 435 : 360;
      const double k = (double)((kblocks + split - 1) / split) * block;
      const double t = split == 1 ? waves * k + 3000 : waves * (k + 6000);
      p.clusters = (int)(split == 1 ? std::min(tiles, slots) : tiles);
      if (best_time == 0 || t < best_time) best = p, best_time = t;
    }
  return best;
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
