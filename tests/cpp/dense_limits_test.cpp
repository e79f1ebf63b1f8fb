// Checks that every 4-bit product that is accepted has a kernel whose grid can be launched, up to the largest sizes.
#include <cstdio>

#include "../../flash_distributed_moe_b200/csrc/dense_plan.h"

#define CHECK(cond)                                                                                                    \
  do {                                                                                                                 \
    if (!(cond)) {                                                                                                     \
      std::printf("line %d: %s (rows %lld tokens %lld gated %d f32 %d)\n", __LINE__, #cond, (long long)rows,           \
                  (long long)tokens, gated, f32);                                                                      \
      return 1;                                                                                                        \
    }                                                                                                                  \
  } while (0)

int main() {
  using namespace fdmoe;
  const int64_t list[] = {1, 8, 12, 127, 128, 129, 256, 257, 4096, 12288, 65536, 8388479, 8388480, 8388481, 8388484, 8388488,
                          8388608, 100000001, 1 << 30};
  DeviceSlots dev = {};
  for (int n = 1; n <= FDMOE_STREAM_SPLIT; ++n) dev.stream_one[n] = 148 / n, dev.stream_two[n] = 296 / n;
  for (int n = 1; n <= FDMOE_PAIR_SPLIT; ++n) dev.pair[n] = 74 / n;
  int chosen[3] = {};
  for (int64_t rows : list)
    for (int64_t tokens : list)
      for (int gated = 0; gated < 2; ++gated)
        for (int f32 = 0; f32 < 2; ++f32) {
          const Mx4Kernel k = ChooseMx4Kernel(tokens, rows, gated, f32);
          ++chosen[(int)k];
          const bool aligned = rows % (f32 ? 4 : 8) == 0;
          if (k == Mx4Kernel::kPair) CHECK(aligned);
          if (k == Mx4Kernel::kNone) CHECK(!aligned && (rows > 8388480 || tokens > 8388480));
          if (rows <= 8388480 && tokens <= 8388480) CHECK((k == Mx4Kernel::kStream) == (!aligned || UseStreamMx4(tokens, rows, gated)));
          if (k == Mx4Kernel::kStream) {
            const StreamPlan s = MakeStreamPlan((int)rows, (int)tokens, 1, gated, true, dev);
            CHECK(s.row_tiles >= 1 && s.row_tiles <= 65535 && s.token_tiles >= 1 && s.token_tiles <= 65535);
            CHECK(s.token_tiles == 1 || s.tile_tokens == 128);  // a tile of tokens begins with a block of scales
          }
        }
  const int64_t rows = 0, tokens = 0;
  const int gated = 0, f32 = 0;
  CHECK(chosen[0] > 0 && chosen[1] > 0 && chosen[2] > 0);
  std::printf("ok\n");
  return 0;
}
