// Plain structs shared by the host side (dense_ops.cpp) and the device side (dense_kernels.cu, mx4_kernels.cu) of the
// dense gated feed-forward block and of the 4-bit microscaled products.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "moe_types.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
  FDMOE_PAIR_TILE = 256,      // rows of a tile of the pair kernel, and most columns
  FDMOE_PAIR_SPLIT = 4,       // most pairs that share the k axis of a tile of the pair kernel
  FDMOE_PAIR_PRODUCTS = 3,    // most products that a launch of the pair kernel works on
  FDMOE_PAIR_MOST = 96,       // most pairs of such a launch
  FDMOE_PAIR_LIST = 64,       // most tiles of a pair in it
  FDMOE_STREAM_ROWS = 128,    // weight rows of a tile of the streaming kernel
  FDMOE_STREAM_TOKENS = 192,  // most tokens of a tile of the streaming kernel: the room for a gated tile's partial sums
  FDMOE_STREAM_TOKENS_MX4 = 128,  // with 4-bit operands: a tile is one block of 128 rows of scales, or part of the only one
  FDMOE_STREAM_SPLIT = 8,     // most CTAs that share the k axis of a tile of the streaming kernel
  FDMOE_STREAM_STAGES = 12,   // most shared-memory stages of the streaming kernel
  FDMOE_MX4_BLOCK = 32,       // elements that share a scale
  FDMOE_MX4_STAGE_K = 256,    // elements of k per stage: 128 bytes of 4-bit values
};

// What the epilogue makes of a tile.
enum {
  FDMOE_EPI_HALF = 0,        // rounded to bf16 or fp16
  FDMOE_EPI_F32 = 1,         // as it is
  FDMOE_EPI_GATED = 2,       // silu(gate) * up, rounded to bf16 or fp16
  FDMOE_EPI_GATED_F32 = 3,   // silu(gate) * up
  FDMOE_EPI_GATED_GRAD = 4,  // gradients of gate and up
  FDMOE_EPI_GATED_SAVE = 5,  // as FDMOE_EPI_GATED, and the gate and up projections
};

// Status codes of the dense kernels (first error wins).
enum {
  FDMOE_DENSE_TIMEOUT_EMPTY = 21,  // a stage was not freed
  FDMOE_DENSE_TIMEOUT_FULL = 22,   // a stage was not filled
  FDMOE_DENSE_TIMEOUT_ACC = 23,    // an accumulator was not freed
  FDMOE_DENSE_TIMEOUT_DONE = 24,   // an accumulator was not completed
};

// One product of a launch of the pair kernel.
typedef struct {
  FdmoeTensorMap a, b;        // operands; `a` gives the rows of the result, `b` its columns
  FdmoeTensorMap out[3];      // results: the tile | h | h, upper halves of gate, up | d gate, d up
  int32_t rows, cols;         // of the result
  int32_t tiles_m, tiles_n;
  int32_t tile_n;             // 256, 192 or 128 (4-bit operands: 256)
  int32_t kblocks;
  int32_t a_mn, b_mn;         // operand stored with its rows along M (N) instead of along K
} FdmoePairProduct;

typedef struct {
  FdmoePairProduct product[FDMOE_PAIR_PRODUCTS];
  FdmoeTensorMap sfa, sfb;    // scales of 4-bit operands
  FdmoeTensorMap gu[2];       // upper halves of gate and up projections (FDMOE_EPI_GATED_GRAD)
  void* lower;                // [rows, cols] lower bytes of both (FDMOE_EPI_GATED_SAVE and FDMOE_EPI_GATED_GRAD)
  void* to[3];                // product[0].out and `gu` as pointers, for tiles whose k axis is shared
  const void* from[2];
  uint32_t* status;
  uint64_t timeout_ns;
  int32_t products;           // above 1: FDMOE_EPI_HALF, `split` 1, tiles dealt out by `count`
  int32_t split;              // 1, 2 or 4 pairs per tile; above 1 a launch has a cluster per tile
  int32_t up_row;             // row of `b` at which the up projection starts (gated)
  int32_t sf_chunks;          // 512-byte blocks of scales per 128 rows
  int32_t sf_up_block;        // block of 128 rows at which the up projection's scales start
  int32_t bf16;               // 16-bit operands and results are bf16, otherwise fp16
  int32_t stall;              // test hook: nothing is loaded, every wait runs out
  uint8_t count[FDMOE_PAIR_PRODUCTS][FDMOE_PAIR_MOST];  // tiles of each product for each pair
} FdmoePairParams;

typedef struct {
  FdmoeTensorMap a, b;        // weights (rows of the tile) and tokens (columns of the tile)
  FdmoeTensorMap sfa, sfb;
  void* out;                  // [tokens, rows], row stride `ld` elements
  uint32_t* status;
  uint64_t timeout_ns;
  int64_t ld;
  int32_t rows, tokens;
  int32_t tile_tokens;        // a multiple of 16, up to FDMOE_STREAM_TOKENS or FDMOE_STREAM_TOKENS_MX4
  int32_t split;              // CTAs per tile along k: the cluster
  int32_t kblocks_each, kblocks_more;  // stages of k of every CTA; one more for the first few
  int32_t stages;
  int32_t up_row;
  int32_t sf_chunks;
  int32_t sf_up_block;
  int32_t bf16;
  int32_t tmem_cols;
  int32_t early_weights;      // the launch before this one does not write the weights: load them before it has ended
  int32_t stall;              // test hook, as above
} FdmoeStreamParams;

// Launchers; return a cudaError_t.  `mx4` selects 4-bit operands.
// Every kernel of the dense operators may start before the launch before it on the stream has ended, and waits for
// that itself before it touches global memory (programmatic dependent launch): set-up and launch latency overlap.
int fdmoe_pair_launch(const FdmoePairParams* p, int epi, int mx4, int clusters, void* stream);
int fdmoe_stream_launch(const FdmoeStreamParams* p, int epi, int mx4, int smem, void* stream);

// Clusters of `size` CTAs of the pair kernel, or of the streaming kernel with `smem` bytes, that the current device
// runs at once.
int fdmoe_pair_clusters(int size, int* out);
int fdmoe_stream_clusters(int size, int smem, int* out);

int fdmoe_mx4_quantize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int64_t batch_stride,
                       int64_t row_stride, void* values, void* scales, void* stream);
int fdmoe_mx4_dequantize(const void* values, const void* scales, int64_t batch, int64_t rows, int64_t cols, int dtype,
                         void* out, void* stream);

#ifdef __cplusplus
}
#endif
