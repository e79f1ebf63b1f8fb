// Checks the launch plans of the streaming kernel over the range of sizes: shared memory, TMEM columns, stages and the
// split of the k axis stay within what the kernel and the hardware allow.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../flash_distributed_moe_b200/csrc/dense_plan.h"

#define CHECK(cond)                                                                                              \
  do {                                                                                                           \
    if (!(cond)) {                                                                                               \
      std::printf("line %d: %s (rows %d tokens %d kblocks %d gated %d mx4 %d)\n", __LINE__, #cond, rows, tokens, \
                  kb, gated, mx4);                                                                               \
      return 1;                                                                                                  \
    }                                                                                                            \
  } while (0)

int main() {
  using namespace fdmoe;
  const int row_list[] = {1, 8, 127, 128, 129, 768, 1544, 4096, 12288, 65536};
  const int token_list[] = {1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 80, 96, 100, 112, 127, 128, 129, 255, 256, 1531, 8192, 65536};
  const int kb_list[] = {1, 2, 3, 5, 8, 12, 16, 33, 64, 192, 1000};
  for (int rows : row_list)
    for (int tokens : token_list)
      for (int kb : kb_list)
        for (int gated = 0; gated < 2; ++gated)
          for (int mx4 = 0; mx4 < 2; ++mx4)
            for (int sms : {148, 132, 8}) {
              DeviceSlots dev;
              for (int n = 1; n <= FDMOE_STREAM_SPLIT; ++n) dev.stream_one[n] = sms / n, dev.stream_two[n] = 2 * sms / n;
              for (int n = 1; n <= FDMOE_PAIR_SPLIT; ++n) dev.pair[n] = sms / (2 * n);
              const StreamPlan s = MakeStreamPlan(rows, tokens, kb, gated, mx4, dev);
              const int parts = gated ? 2 : 1;
              const int stage = parts * 16384 + s.tile_tokens * 128 + (mx4 ? (parts + 1) * 1024 : 0);
              CHECK(s.tile_tokens % 16 == 0 && s.tile_tokens >= 16 && s.tile_tokens <= (mx4 ? FDMOE_STREAM_TOKENS_MX4 : FDMOE_STREAM_TOKENS));
              CHECK((int64_t)s.tile_tokens * s.token_tiles >= tokens && (int64_t)s.tile_tokens * (s.token_tiles - 1) < tokens);
              // a tile of tokens lies within one block of 128 rows of scales and starts on a column of them
              if (s.token_tiles > 1 && mx4) CHECK(s.tile_tokens == 128 || (128 % s.tile_tokens == 0 && s.tile_tokens % 32 == 0));
              CHECK(s.row_tiles * FDMOE_STREAM_ROWS >= rows && s.row_tiles <= 65535);
              CHECK(s.split >= 1 && s.split <= FDMOE_STREAM_SPLIT && s.split <= kb);
              CHECK(s.stages >= 1 && s.stages <= FDMOE_STREAM_STAGES);
              CHECK(s.stages * stage + kStreamSlack <= s.smem);
              const int in_tile = tokens < s.tile_tokens ? tokens : s.tile_tokens;  // partial sums, if the k axis is split
              if (s.split > 1) CHECK(RoundUp(in_tile, 4 * s.split) * parts * 512 + kStreamSlack <= s.smem);
              CHECK(s.smem <= 226 * 1024 && (s.per_sm == 1 || s.smem <= 112 * 1024));
              const int cols = parts * s.tile_tokens + (mx4 ? s.stages * (parts + 1) * 8 : 0);
              CHECK(s.tmem_cols >= cols && s.tmem_cols >= 32 && (s.tmem_cols & (s.tmem_cols - 1)) == 0);
              CHECK(s.tmem_cols * s.per_sm <= 512);
              // No CTA may wait for another's columns while a CTA of its cluster on another SM already holds some:
              // wherever the shared memory of several has room, their columns have too.
              const int taken = s.smem + 1024, sm = 228 * 1024;
              CHECK(taken / 1024 * 544 > sm / 1024 * s.tmem_cols);  // the sum of columns is a multiple of 32
              CHECK(taken + 196 * 1024 > sm);                       // kernels that take all 512 columns
              const PairPlan q = MakePairPlan(tokens, rows, kb, gated, mx4, dev);
              const int cols_tile = gated ? q.tile_n / 2 : q.tile_n;
              CHECK(q.tile_n == 256 || ((q.tile_n == 128 || q.tile_n == 192) && !mx4));
              CHECK((q.split == 1 || q.split == 2 || q.split == 4) && q.split <= kb);
              CHECK(q.tiles_m * 256 >= tokens && q.tiles_n * cols_tile >= rows && q.clusters >= 1);
              CHECK(q.split == 1 ? q.clusters <= q.tiles_m * q.tiles_n : q.clusters == q.tiles_m * q.tiles_n);
            }
  // Several products in one launch: every tile is dealt out once, in the order in which the kernel lists them.
  const int dims[] = {8, 72, 256, 777, 1000, 2048, 4096, 12288};
  for (int tokens : dims)
    for (int rows : dims)
      for (int kb : dims)
        for (int n = 2; n <= 3; ++n) {
          const int gated = n, mx4 = 0;  // for the message
          DeviceSlots dev = {};
          dev.pair[1] = 74, dev.pair[2] = 33, dev.pair[4] = 15;
          const int T = tokens, H = rows, I = kb;
          const ManyShape shape[3] = {{T, H, (2 * I + 63) / 64}, {2 * I, H, (T + 63) / 64}, {H, I, (T + 63) / 64}};
          const ManyPlan m = MakeManyPlan(shape, n, dev);
          if (!m.use) continue;
          CHECK(m.pairs == 74);
          std::vector<int> held(m.pairs, 0);
          for (int i = 0; i < n; ++i) {
            const int x = m.order[i];
            CHECK(m.tile_n[x] == 256 || m.tile_n[x] == 192 || m.tile_n[x] == 128);
            const long tiles = ((shape[x].rows + 255) / 256) * ((shape[x].cols + m.tile_n[x] - 1) / m.tile_n[x]);
            std::vector<char> seen(tiles, 0);
            long base = 0;
            for (int r = 0; r < 256; ++r) {
              long all = 0;
              for (int p = 0; p < m.pairs; ++p)
                if (m.count[i][p] > r) {
                  CHECK(base + all < tiles && !seen[base + all]);
                  seen[base + all] = 1;
                  ++all, ++held[p];
                }
              base += all;
            }
            CHECK(base == tiles);
          }
          for (int p = 0; p < m.pairs; ++p) CHECK(held[p] <= FDMOE_PAIR_LIST - 3);
        }
  {
    const int rows = 0, tokens = 0, kb = 0, gated = 0, mx4 = 0;
    CHECK(ScaleChunks(32) == 2 && ScaleChunks(256) == 2 && ScaleChunks(288) == 4);
    CHECK(ScaleBytes(1, 1, 32) == 1024 && ScaleBytes(2, 129, 512) == 2 * 2 * 4 * 512 && ScaleBytes(1, 0, 32) == 0);
  }
  std::printf("ok\n");
  return 0;
}
