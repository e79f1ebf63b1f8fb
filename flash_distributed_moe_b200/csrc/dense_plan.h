// How a product of the dense operators is cut into launches: which kernel, tiles, stages and the split of the k axis.
// Host arithmetic only, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "dense_types.h"

namespace fdmoe {

// Dynamic shared memory of a CTA when two share an SM (228 KB, 1 KB each reserved), and of one alone.
constexpr int kStreamSmemTwo = 112 * 1024;
constexpr int kStreamSmemOne = 226 * 1024;
constexpr int kStreamSlack = 1024;            // for the alignment of the stages

struct StreamPlan {
  int tile_tokens, token_tiles, row_tiles, split, stages, smem, tmem_cols, per_sm;
  double cycles;  // estimated
};

inline int RoundUp(int v, int m) { return (v + m - 1) / m * m; }

// What the device runs at once: clusters of n CTAs of the streaming kernel with one or two CTAs per SM, and of the
// pair kernel with n pairs.  A GPC's SMs hold whole clusters only, so these are fewer than the SMs would give.
struct DeviceSlots {
  int stream_one[FDMOE_STREAM_SPLIT + 1], stream_two[FDMOE_STREAM_SPLIT + 1], pair[FDMOE_PAIR_SPLIT + 1];
};

// `rows` weight rows (gated: of each projection), `tokens` >= 1, `kblocks` stages of k in all.
//
// Time in cycles.  A k block takes as long as its MMAs' issue, or as the weights of `active` CTAs do at the rate at which
// their stages in flight are filled, at most the memory's 3400 bytes per cycle; another wave of CTAs costs far more than
// its k blocks.  The constants are those with which the choice is on average 0.7 % and at most 6 % slower than the best
// of all splits with one and two CTAs per SM, over 124 products (1 to 128 tokens; 512 x 1024 to 8192 x 8192; cold
// weights).  In us, with 2, 3, 4, 6 and 8 CTAs per tile: 64 tokens, gated, 4096 rows, k 1024 8.5, 8.5, 8.4, 11.0 and 11.0;
// with 4 bits, 2048 rows, k 2048 6.8, 6.5, 6.1, 6.7 and 7.9; 1 token, 2048 rows, k 6144 12.7, 10.0, 8.7, 8.0 and 7.9.
inline StreamPlan MakeStreamPlan(int rows, int tokens, int kblocks, bool gated, bool mx4, const DeviceSlots& dev) {
  StreamPlan best = {};
  double best_time = 0;
  const int parts = gated ? 2 : 1;
  for (int per_sm = 2; per_sm >= 1; --per_sm) {
    StreamPlan s = {};
    s.per_sm = per_sm;
    const int most_tokens = mx4 ? FDMOE_STREAM_TOKENS_MX4 : FDMOE_STREAM_TOKENS;
    s.token_tiles = (tokens + most_tokens - 1) / most_tokens;
    s.tile_tokens = s.token_tiles > 1 ? most_tokens : RoundUp(tokens, 16);
    s.row_tiles = (rows + FDMOE_STREAM_ROWS - 1) / FDMOE_STREAM_ROWS;
    const int stage = parts * 16384 + s.tile_tokens * 128 + (mx4 ? (parts + 1) * 1024 : 0);
    const int room = (per_sm == 2 ? kStreamSmemTwo : kStreamSmemOne) - kStreamSlack;
    // Partial sums, in the stages' place: groups of four tokens, the same number for every CTA of the cluster.
    const int sums = (RoundUp(std::min(tokens, s.tile_tokens), 4) + 4 * (FDMOE_STREAM_SPLIT - 1)) * parts * 512;
    const int scales = mx4 ? (parts + 1) * 8 : 0;  // TMEM columns per stage
    int most = std::min(room / stage, (int)FDMOE_STREAM_STAGES);
    if (scales) most = std::min(most, ((per_sm == 2 ? 256 : 512) - parts * s.tile_tokens) / scales);
    if (per_sm == 2 && (most < 2 || parts * s.tile_tokens > 256)) continue;
    const double weights = parts * (mx4 ? 16384 + 1024 : 16384), issue = mx4 ? 650 + 40 * parts : 560 + 160 * parts;
    for (int n = 1; n <= FDMOE_STREAM_SPLIT && n <= kblocks; ++n) {
      const int64_t slots = per_sm == 2 ? dev.stream_two[n] : dev.stream_one[n];
      if (slots < 1 || (n > 1 && sums > room)) continue;  // the device cannot hold such a cluster, or a CTA the sums
      const int blocks = (kblocks + n - 1) / n;
      double t = per_sm == 1 ? 250 : 0;  // the launches before and after it cannot overlap with it
      // the partial sums' way through the cluster's shared memory at 14 bytes per cycle, and the epilogue
      t += (n > 1 ? 1000 + 250 * n : 0) + s.tile_tokens * parts * (42.0 * (n - 1) + 20.0) / n;
      int64_t clusters = (int64_t)s.row_tiles * s.token_tiles;
      for (int wave = 0; clusters > 0 && wave < 64; ++wave, clusters -= slots) {
        const double active = (double)std::min(clusters, slots) * n;
        const double rate = std::min(3400.0, active * most * weights / 4200);
        t += blocks * std::max(issue, active * weights / rate) + 16000;
      }
      if (best_time != 0 && t >= best_time) continue;
      best_time = t;
      best = s;
      best.cycles = t;
      best.split = n;
      best.stages = std::min(most, blocks);
      const int cols = parts * s.tile_tokens + best.stages * scales;
      best.tmem_cols = 32;
      while (best.tmem_cols < cols) best.tmem_cols *= 2;
      // The whole share, used or not: then CTAs that fit on an SM together find their columns there too.  One that had to
      // wait for columns could wait for a CTA whose cluster waits for columns that this one's cluster holds elsewhere.
      best.smem = per_sm == 2 ? kStreamSmemTwo : kStreamSmemOne;
    }
  }
  return best;
}

struct PairPlan {
  int tile_n, split, tiles_m, tiles_n, clusters;
  double cycles;  // estimated
};

inline double BlockCycles(int tile_n) { return tile_n == 256 ? 520 : tile_n == 192 ? 455 : 365; }

// `cols`: of the result; `kblocks` stages of k.  Time in cycles: the waves of tiles, each its k blocks, and once per
// launch, or per cluster where pairs share a tile, its beginning and end; sharing also takes the partial sums' way
// through the cluster's shared memory, at 14 bytes a cycle.  A k block is planned with 520, 455 and 365 cycles at widths
// of 256, 192 and 128.  Its MMAs are 512, 384 and 256; at about 128 bytes a cycle its operands take 512, 448 and 384 to
// be written to and read from shared memory, a rough figure: 365 to 400 were measured at a width of 128.
// In us, for width / pairs per tile: 4096 x 2048 x 6144 (rows, columns, k) 69 with 256/1, 80 with 192/1, 95 with
// 128/1, 90 with 256/2; 777 x 1000 x 5488 36, 32, 28 and 24, 19 with 128/2, 36 with 128/4.
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
      const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, slots = dev.pair[split];
      if (slots < 1) continue;  // the device cannot hold such a cluster
      const double waves = (double)((tiles + slots - 1) / slots);
      const double k = (double)((kblocks + split - 1) / split) * BlockCycles(tile_n);
      const double exchange = (double)tile_n * 512 * (split - 1) / split / 14;
      const double t = split == 1 ? waves * k + 3000 : waves * (k + 3500 + exchange);
      p.clusters = (int)(split == 1 ? std::min(tiles, slots) : tiles);
      p.cycles = t;
      if (best_time == 0 || t < best_time) best = p, best_time = t;
    }
  return best;
}

// Several products in one launch of the pair kernel: their tiles, the longest first, fill the pairs evenly, where
// launches of their own would each end with a wave that is partly empty.
struct ManyShape {
  int64_t rows, cols;
  int kblocks;
};
struct ManyPlan {
  bool use;              // better than a launch for each
  int pairs;
  int order[FDMOE_PAIR_PRODUCTS];   // the products by the length of their tiles
  int tile_n[FDMOE_PAIR_PRODUCTS];  // of each product
  uint8_t count[FDMOE_PAIR_PRODUCTS][FDMOE_PAIR_MOST];  // tiles of order[i] for each pair
};

inline ManyPlan MakeManyPlan(const ManyShape* shape, int n, const DeviceSlots& dev) {
  ManyPlan m = {};
  m.pairs = std::min(dev.pair[1], (int)FDMOE_PAIR_MOST);
  if (n < 2 || m.pairs < 1) return m;
  double apart = 0;  // launches of their own
  for (int i = 0; i < n; ++i) {
    const PairPlan p = MakePairPlan(shape[i].rows, shape[i].cols, shape[i].kblocks, false, false, dev);
    apart += p.cycles + 4000;
  }
  auto tiles = [&](int i, int tile_n) {
    return (double)((shape[i].rows + FDMOE_PAIR_TILE - 1) / FDMOE_PAIR_TILE) * ((shape[i].cols + tile_n - 1) / tile_n);
  };
  auto length = [&](int i, int tile_n) { return shape[i].kblocks * BlockCycles(tile_n) + 600; };
  // Widths: every choice, by the even share and the longest tile.
  const int widths[3] = {256, 192, 128};
  int choices = 1;
  for (int i = 0; i < n; ++i) choices *= 3;
  double best = 0;
  for (int c = 0; c < choices; ++c) {
    double total = 0, most = 0, least = 0;
    for (int i = 0, d = c; i < n; ++i, d /= 3) {
      const double l = length(i, widths[d % 3]);
      total += l * tiles(i, widths[d % 3]);
      most = std::max(most, l);
      least = least == 0 ? l : std::min(least, l);
    }
    const double t = std::max(total / m.pairs + least / 2, most);
    if (c == 0 || t < best) {
      best = t;
      for (int i = 0, d = c; i < n; ++i, d /= 3) m.tile_n[i] = widths[d % 3];
    }
  }
  for (int i = 0; i < n; ++i) m.order[i] = i;
  std::sort(m.order, m.order + n, [&](int x, int y) { return length(x, m.tile_n[x]) > length(y, m.tile_n[y]); });
  // Deal out: raise a level under which every pair is filled with whole tiles, until all tiles have a place.
  double load[FDMOE_PAIR_MOST] = {};
  int held[FDMOE_PAIR_MOST] = {};
  for (int i = 0; i < n; ++i) {
    const int x = m.order[i];
    const double l = length(x, m.tile_n[x]), want = tiles(x, m.tile_n[x]);
    if (want > (double)m.pairs * (FDMOE_PAIR_LIST - 3)) return m;
    double low = 0, high = want * l;
    for (int p = 0; p < m.pairs; ++p) high = std::max(high, load[p] + (want / m.pairs + 1) * l);
    auto fits = [&](double level) {
      double f = 0;
      for (int p = 0; p < m.pairs; ++p)
        if (level > load[p]) f += (int)((level - load[p]) / l);
      return f;
    };
    for (int k = 0; k < 24; ++k) {
      const double mid = 0.5 * (low + high);
      (fits(mid) >= want ? high : low) = mid;
    }
    int64_t over = -(int64_t)want;
    int got[FDMOE_PAIR_MOST];
    for (int p = 0; p < m.pairs; ++p) over += got[p] = high > load[p] ? (int)((high - load[p]) / l) : 0;
    for (int p = m.pairs - 1; p >= 0 && over > 0; --p)  // those that reach the level itself give one back
      if (got[p] > 0 && load[p] + got[p] * l > high - l) --got[p], --over;
    if (over != 0) return m;
    for (int p = 0; p < m.pairs; ++p) {
      load[p] += got[p] * l;
      held[p] += got[p];
      if (got[p] > 255 || held[p] > FDMOE_PAIR_LIST - 3) return m;
      m.count[i][p] = (uint8_t)got[p];
    }
  }
  m.use = *std::max_element(load, load + m.pairs) + 3000 < apart;
  return m;
}

// Whether the streaming kernel takes the products of `tokens` rows instead of the pair kernel.  It reads weights faster,
// which counts by their bytes, and its partial sums and epilogue cost more with every token.  Whole block of `bytes` of
// weights, streaming and pair kernels in us: 96 tokens of 512 x 1024 10.9 and 10.5, of 2048 x 768 12.7 and 13.9; 128
// tokens of 2048 x 768 14.4 and 14.1, of 1024 x 4096 18.2 and 18.1, of 2048 x 6144 27.4 and 29.6; 160 tokens of
// 2048 x 6144 29.7 and 29.7, of 4096 x 4096 32.2 and 34.0, of 4096 x 12288 66 and 83, of 8192 x 28672 249 and 289.
inline bool UseStream(int64_t tokens, int64_t bytes) {
  return tokens <= std::min<int64_t>(96 + (bytes >> 20), FDMOE_STREAM_TOKENS);
}
// 4-bit operands: one tile of tokens, or two where the pair kernel's tiles leave most pairs idle.  128 tokens times
// 4096 x 12288 (rows, columns) 10.3 and 14.1 us, 2048 x 6144 7.2 and 9.2, 12288 x 4096 10.8 and 10.7, gated 16.4 and
// 18.2, gated 8192 x 8192 19.4 and 18.1; 256 tokens times 1024 x 4096 6.3 and 8.8, 4096 x 12288 13.3 and 14.2,
// 8192 x 8192 14.5 and 13.7, gated 1024 x 4096 9.7 and 9.4.
inline bool UseStreamMx4(int64_t tokens, int64_t rows, bool gated) {
  return tokens <= (!gated && rows <= 4096 ? 2 * FDMOE_STREAM_TOKENS_MX4 : FDMOE_STREAM_TOKENS_MX4);
}

// The kernel for a 4-bit product.  The streaming kernel writes results whose rows do not start on 16 bytes, at any number
// of tokens (it then reads the weights again for every 128); its grid has a block per 128 weight rows along y and one
// per tile of tokens along z, which a launch has no more than 65535 of.
enum class Mx4Kernel { kStream, kPair, kNone };
inline Mx4Kernel ChooseMx4Kernel(int64_t tokens, int64_t rows, bool gated, bool f32) {
  constexpr int64_t kGrid = 65535;
  const bool aligned = rows % (f32 ? 4 : 8) == 0;
  const bool fits = (rows + FDMOE_STREAM_ROWS - 1) / FDMOE_STREAM_ROWS <= kGrid &&
                    (tokens + FDMOE_STREAM_TOKENS_MX4 - 1) / FDMOE_STREAM_TOKENS_MX4 <= kGrid;
  if (fits && (!aligned || UseStreamMx4(tokens, rows, gated))) return Mx4Kernel::kStream;
  return aligned ? Mx4Kernel::kPair : Mx4Kernel::kNone;
}

inline size_t AlignBytes(size_t v) { return (v + 255) / 256 * 256; }

// 512-byte blocks of scales per 128 rows: an even number, as many as the stages of 256 columns take.
inline int64_t ScaleChunks(int64_t cols) { return (cols + FDMOE_MX4_STAGE_K - 1) / FDMOE_MX4_STAGE_K * 2; }
inline size_t ScaleBytes(int64_t batch, int64_t rows, int64_t cols) {
  return (size_t)(batch * ((rows + 127) / 128) * ScaleChunks(cols) * 512);
}

}  // namespace fdmoe
