// Host side of the dense operators: argument checks, TMA descriptors, workspaces and launches of the gated
// feed-forward block (forward, backward) and of the 4-bit microscaled products.  Every call only enqueues work on the
// caller's stream, keeps nothing between calls and takes all scratch from the caller, so calls on different streams
// may overlap and every call can be captured into a CUDA graph.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <initializer_list>
#include <mutex>

#include "../../include/flashmoe_c.h"
#include "dense_plan.h"
#include "dense_types.h"
#include "host_layout.h"

#undef MOE_ERROR_LOG
#define MOE_ERROR_LOG(...)                                   \
  do {                                                       \
    fprintf(stderr, "[MOE ERROR: %s:%d] ", __FILE__, __LINE__); \
    fprintf(stderr, __VA_ARGS__);                            \
    fprintf(stderr, "\n");                                   \
  } while (0)

#define DENSE_CHECK(expr)                                                                              \
  do {                                                                                                 \
    const cudaError_t _e = static_cast<cudaError_t>(expr);                                             \
    if (_e != cudaSuccess) {                                                                           \
      fprintf(stderr, "[MOE CUDA ERROR: %s:%d] %s\n", __FILE__, __LINE__, cudaGetErrorString(_e));     \
      return (int)_e;                                                                                  \
    }                                                                                                  \
  } while (0)

namespace {

using fdmoe::EncodeTiledFn;

enum { kBf16 = 0, kF32 = 1, kF16 = 2 };  // FlashMoeConfig's numbering, and fp16

// One word of mapped host memory: the first device-side error of any dense call in this process.
struct Shared {
  std::mutex mutex;
  uint32_t* status = nullptr;
  EncodeTiledFn encode = nullptr;
  CUresult (*context)(CUcontext*) = nullptr;  // cuCtxGetCurrent
  bool known[64] = {};
  fdmoe::DeviceSlots slots[64];
} g_shared;

struct Call {
  uint32_t* status;
  EncodeTiledFn encode;
  const fdmoe::DeviceSlots* slots;
  uint64_t timeout_ns;
  cudaStream_t stream;
  bool stall;
};

thread_local bool g_stall = false;  // test hook: products load nothing

// After a device-side error nothing is launched on what it has left.  The caller holds the mutex.
int RefuseAfterError() {
  const uint32_t seen = g_shared.status ? *static_cast<volatile uint32_t*>(g_shared.status) : 0;
  if (!seen) return 0;
  MOE_ERROR_LOG("refused after device-side error %u; see FlashMoeDenseStatus", seen);
  return (int)cudaErrorUnknown;
}

int BeginCall(Call* c, void* stream) {
  int dev = 0;
  DENSE_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_shared.mutex);
  if (!g_shared.context) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    DENSE_CHECK(cudaGetDriverEntryPoint("cuCtxGetCurrent", &fn, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess) return (int)cudaErrorUnknown;
    g_shared.context = reinterpret_cast<CUresult (*)(CUcontext*)>(fn);
  }
  // A thread that has made no CUDA call yet (autograd's) has no context, which the descriptors need; one that has keeps
  // its own.
  CUcontext context = nullptr;
  if (g_shared.context(&context) != CUDA_SUCCESS || !context) DENSE_CHECK(cudaSetDevice(dev));
  if (!g_shared.status) {
    // the first call of the process may be inside a stream capture, which this allocation is no part of
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    DENSE_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable);
    cudaThreadExchangeStreamCaptureMode(&mode);
    DENSE_CHECK(e);
    memset(p, 0, 64);
    g_shared.status = static_cast<uint32_t*>(p);
  }
  if (!g_shared.encode) g_shared.encode = fdmoe::GetEncodeTiled();
  if (!g_shared.encode) {
    MOE_ERROR_LOG("cuTensorMapEncodeTiled is not available from this driver");
    return (int)cudaErrorUnknown;
  }
  if (!g_shared.known[dev]) {
    fdmoe::DeviceSlots& d = g_shared.slots[dev];
    for (int n = 1; n <= FDMOE_STREAM_SPLIT; ++n) {
      DENSE_CHECK(fdmoe_stream_clusters(n, fdmoe::kStreamSmemOne, &d.stream_one[n]));
      DENSE_CHECK(fdmoe_stream_clusters(n, fdmoe::kStreamSmemTwo, &d.stream_two[n]));
    }
    for (int n = 1; n <= FDMOE_PAIR_SPLIT; n *= 2) DENSE_CHECK(fdmoe_pair_clusters(2 * n, &d.pair[n]));
    g_shared.known[dev] = true;
  }
  if (const int refused = RefuseAfterError()) return refused;
  c->status = g_shared.status;
  c->encode = g_shared.encode;
  c->slots = &g_shared.slots[dev];
  const char* env = getenv("FLASHMOE_TIMEOUT_MS");
  c->timeout_ns = (uint64_t)std::max(1, env && *env ? atoi(env) : 2000) * 1000000ull;
  c->stream = static_cast<cudaStream_t>(stream);
  c->stall = g_stall;
  return 0;
}

// Row-major matrix [rows, cols] of `size`-byte elements, rows `stride` bytes apart.
int MakeMap(const Call& c, FdmoeTensorMap* out, const void* base, int size, int64_t rows, int64_t cols, int64_t stride,
            int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = size == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const int span = box_cols * size;  // bytes of a row in shared memory
  const CUtensorMapSwizzle swizzle = span == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : span == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                  : CU_TENSOR_MAP_SWIZZLE_NONE;
  const CUresult r = c.encode(reinterpret_cast<CUtensorMap*>(out), type, 2, const_cast<void*>(base), dims, strides, box,
                              estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    MOE_ERROR_LOG("cuTensorMapEncodeTiled failed with %d (rows %lld cols %lld)", (int)r, (long long)rows, (long long)cols);
    return (int)cudaErrorInvalidValue;
  }
  return 0;
}

#define DENSE_TRY(expr)          \
  do {                           \
    const int _r = (expr);       \
    if (_r != 0) return _r;      \
  } while (0)

bool Aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------ products of 16-bit operands
struct Operand {
  const void* base;
  int64_t rows, cols;  // as stored
  bool mn;             // rows run along M (N): stored [k, m] instead of [m, k]
};

int OperandMap(const Call& c, FdmoeTensorMap* out, const Operand& o, int box_rows) {
  return MakeMap(c, out, o.base, 2, o.rows, o.cols, o.cols * 2, 64, o.mn ? 64 : box_rows);
}

int KBlocks(int64_t k, bool mx4) { return (int)((k + (mx4 ? FDMOE_MX4_STAGE_K : 64) - 1) / (mx4 ? FDMOE_MX4_STAGE_K : 64)); }

// A launch of the pair kernel with one product of this shape; returns its number of clusters.
int PairShape(FdmoePairParams& p, const Call& c, int64_t rows, int64_t cols, int64_t k, bool gated, bool mx4) {
  FdmoePairProduct& q = p.product[0];
  p.status = c.status;
  p.timeout_ns = c.timeout_ns;
  p.stall = c.stall;
  p.products = 1;
  q.rows = (int32_t)rows;
  q.cols = (int32_t)cols;
  q.kblocks = KBlocks(k, mx4);
  const fdmoe::PairPlan plan = fdmoe::MakePairPlan(rows, cols, q.kblocks, gated, mx4, *c.slots);
  p.split = plan.split;
  q.tile_n = plan.tile_n;
  q.tiles_m = plan.tiles_m;
  q.tiles_n = plan.tiles_n;
  return plan.clusters;
}

// out = A B^T, both operands given as stored.
struct Product {
  Operand a, b;
  void* out;
  int64_t rows() const { return a.mn ? a.cols : a.rows; }
  int64_t cols() const { return b.mn ? b.cols : b.rows; }
  int64_t k() const { return a.mn ? a.rows : a.cols; }
};

int ProductMaps(const Call& c, FdmoePairProduct& q, const Product& w) {
  q.a_mn = w.a.mn;
  q.b_mn = w.b.mn;
  DENSE_TRY(OperandMap(c, &q.a, w.a, 128));
  DENSE_TRY(OperandMap(c, &q.b, w.b, q.tile_n / 2));
  return MakeMap(c, &q.out[0], w.out, 2, w.rows(), w.cols(), w.cols() * 2, 64, 32);
}

int PairProduct(const Call& c, const Product& w, bool bf16) {
  FdmoePairParams p;
  memset(&p, 0, sizeof(p));
  const int clusters = PairShape(p, c, w.rows(), w.cols(), w.k(), false, false);
  DENSE_TRY(ProductMaps(c, p.product[0], w));
  p.to[0] = w.out;
  p.bf16 = bf16;
  return fdmoe_pair_launch(&p, FDMOE_EPI_HALF, 0, clusters, c.stream);
}

// MakeManyPlan takes some ten microseconds; the plans of the last shapes are kept.
void CachedManyPlan(const fdmoe::ManyShape* shape, int n, const fdmoe::DeviceSlots* slots, fdmoe::ManyPlan* out) {
  struct Entry {
    const fdmoe::DeviceSlots* slots = nullptr;  // of the device
    int n = 0;
    int64_t key[3 * FDMOE_PAIR_PRODUCTS];
    fdmoe::ManyPlan plan;
  };
  static std::mutex mutex;
  static Entry cache[32];
  static int next = 0;
  int64_t key[3 * FDMOE_PAIR_PRODUCTS] = {};
  for (int i = 0; i < n; ++i) key[3 * i] = shape[i].rows, key[3 * i + 1] = shape[i].cols, key[3 * i + 2] = shape[i].kblocks;
  std::lock_guard<std::mutex> lock(mutex);
  for (const Entry& e : cache)
    if (e.slots == slots && e.n == n && memcmp(e.key, key, sizeof(key)) == 0) {
      *out = e.plan;
      return;
    }
  Entry& e = cache[next];
  next = (next + 1) % 32;
  e.plan = fdmoe::MakeManyPlan(shape, n, *slots);
  e.slots = slots;
  e.n = n;
  memcpy(e.key, key, sizeof(key));
  *out = e.plan;
}

// Up to three products that do not depend on each other, in one launch if that is faster.
int PairProducts(const Call& c, const Product* w, int n, bool bf16) {
  fdmoe::ManyShape shape[FDMOE_PAIR_PRODUCTS];
  for (int i = 0; i < n; ++i) shape[i] = {w[i].rows(), w[i].cols(), KBlocks(w[i].k(), false)};
  fdmoe::ManyPlan m;
  CachedManyPlan(shape, n, c.slots, &m);
  if (!m.use) {
    for (int i = 0; i < n; ++i) DENSE_TRY(PairProduct(c, w[i], bf16));
    return 0;
  }
  FdmoePairParams p;
  memset(&p, 0, sizeof(p));
  p.status = c.status;
  p.timeout_ns = c.timeout_ns;
  p.stall = c.stall;
  p.products = n;
  p.split = 1;
  p.bf16 = bf16;
  for (int i = 0; i < n; ++i) {
    const int x = m.order[i];
    FdmoePairProduct& q = p.product[i];
    q.rows = (int32_t)shape[x].rows;
    q.cols = (int32_t)shape[x].cols;
    q.kblocks = shape[x].kblocks;
    q.tile_n = m.tile_n[x];
    q.tiles_m = (int32_t)((shape[x].rows + FDMOE_PAIR_TILE - 1) / FDMOE_PAIR_TILE);
    q.tiles_n = (int32_t)((shape[x].cols + q.tile_n - 1) / q.tile_n);
    DENSE_TRY(ProductMaps(c, q, w[x]));
  }
  memcpy(p.count, m.count, sizeof(p.count));
  return fdmoe_pair_launch(&p, FDMOE_EPI_HALF, 0, m.pairs, c.stream);
}

// out[tokens, rows] = x w^T (gated: silu(x w[:rows]^T) * (x w[rows:]^T)) for few tokens.
int StreamProduct(const Call& c, const void* x, const void* w, void* out, int64_t tokens, int64_t rows, int64_t k,
                  bool gated, bool bf16, bool early_weights) {
  FdmoeStreamParams p;
  memset(&p, 0, sizeof(p));
  const int kblocks = (int)((k + 63) / 64);
  const fdmoe::StreamPlan s = fdmoe::MakeStreamPlan((int)rows, (int)tokens, kblocks, gated, false, *c.slots);
  DENSE_TRY(MakeMap(c, &p.a, w, 2, gated ? 2 * rows : rows, k, k * 2, 64, 128));
  DENSE_TRY(MakeMap(c, &p.b, x, 2, tokens, k, k * 2, 64, s.tile_tokens));
  p.out = out;
  p.status = c.status;
  p.timeout_ns = c.timeout_ns;
  p.stall = c.stall;
  p.ld = rows;
  p.rows = (int32_t)rows;
  p.tokens = (int32_t)tokens;
  p.tile_tokens = s.tile_tokens;
  p.split = s.split;
  p.kblocks_each = kblocks / s.split;
  p.kblocks_more = kblocks % s.split;
  p.stages = s.stages;
  p.up_row = (int32_t)rows;
  p.bf16 = bf16;
  p.tmem_cols = s.tmem_cols;
  p.early_weights = early_weights;
  return fdmoe_stream_launch(&p, gated ? FDMOE_EPI_GATED : FDMOE_EPI_HALF, 0, s.smem, c.stream);
}

// What a forward call keeps for the backward pass: the upper halves of the projections [T, 2I], their lower bytes
// [T, I], and h [T, I], 16 bits each.
struct Saved {
  uint8_t *gu = nullptr, *lower = nullptr, *h = nullptr;
  static size_t Bytes(int64_t T, int64_t I) {
    return fdmoe::AlignBytes((size_t)T * I * 4) + 2 * fdmoe::AlignBytes((size_t)T * I * 2);
  }
  Saved() = default;
  Saved(const void* base, int64_t T, int64_t I) {
    gu = static_cast<uint8_t*>(const_cast<void*>(base));
    lower = gu + fdmoe::AlignBytes((size_t)T * I * 4);
    h = lower + fdmoe::AlignBytes((size_t)T * I * 2);
  }
};

// h[T, I] = silu(g) * u with [g, u] = x w13^T; also what is to be kept, where `saved` has room for it.
int GatedProduct(const Call& c, const void* x, const void* w13, void* h, const Saved& saved, int64_t T, int64_t H,
                 int64_t I, bool bf16) {
  FdmoePairParams p;
  memset(&p, 0, sizeof(p));
  const int clusters = PairShape(p, c, T, I, H, true, false);
  FdmoePairProduct& q = p.product[0];
  DENSE_TRY(MakeMap(c, &q.a, x, 2, T, H, H * 2, 64, 128));
  DENSE_TRY(MakeMap(c, &q.b, w13, 2, 2 * I, H, H * 2, 64, q.tile_n / 2));
  DENSE_TRY(MakeMap(c, &q.out[0], h, 2, T, I, I * 2, 64, 32));
  p.to[0] = h;
  if (saved.gu) {
    // two matrices side by side: what a tile has beyond column I of the gate projection is not stored
    DENSE_TRY(MakeMap(c, &q.out[1], saved.gu, 2, T, I, I * 4, 64, 32));
    DENSE_TRY(MakeMap(c, &q.out[2], saved.gu + I * 2, 2, T, I, I * 4, 64, 32));
    p.to[1] = saved.gu;
    p.to[2] = saved.gu + I * 2;
    p.lower = saved.lower;
  }
  p.up_row = (int32_t)I;
  p.bf16 = bf16;
  return fdmoe_pair_launch(&p, saved.gu ? FDMOE_EPI_GATED_SAVE : FDMOE_EPI_GATED, 0, clusters, c.stream);
}

// From dy: dgu [T, 2I].
int GatedGradient(const Call& c, const void* dy, const void* w2, const Saved& saved, void* dgu, int64_t T, int64_t H,
                  int64_t I, bool bf16) {
  FdmoePairParams p;
  memset(&p, 0, sizeof(p));
  const int clusters = PairShape(p, c, T, I, H, false, false);
  FdmoePairProduct& q = p.product[0];
  DENSE_TRY(MakeMap(c, &q.a, dy, 2, T, H, H * 2, 64, 128));
  DENSE_TRY(MakeMap(c, &q.b, w2, 2, H, I, I * 2, 64, 64));
  for (int i = 0; i < 2; ++i) {
    DENSE_TRY(MakeMap(c, &p.gu[i], saved.gu + i * I * 2, 2, T, I, I * 4, 64, 32));
    DENSE_TRY(MakeMap(c, &q.out[i], static_cast<uint8_t*>(dgu) + i * I * 2, 2, T, I, I * 4, 64, 32));
    p.from[i] = saved.gu + i * I * 2;
    p.to[i] = static_cast<uint8_t*>(dgu) + i * I * 2;
  }
  p.lower = saved.lower;
  q.b_mn = 1;
  p.bf16 = bf16;
  return fdmoe_pair_launch(&p, FDMOE_EPI_GATED_GRAD, 0, clusters, c.stream);
}

// ------------------------------------------------------ products of 4-bit operands
struct Mx4 {
  const void *values, *scales;
  int64_t rows;   // of one matrix
  int64_t batch;  // matrices one after another
};

int Mx4Maps(const Call& c, FdmoeTensorMap* values, FdmoeTensorMap* scales, const Mx4& m, int64_t k, int box_rows) {
  const int64_t chunks = fdmoe::ScaleChunks(k), blocks = m.batch * ((m.rows + 127) / 128);
  if (blocks * chunks > INT32_MAX) return (int)cudaErrorInvalidValue;  // a coordinate has 32 bits
  DENSE_TRY(MakeMap(c, values, m.values, 1, m.batch * m.rows, k / 2, k / 2, 128, box_rows));
  return MakeMap(c, scales, m.scales, 4, blocks * chunks, 128, 512, 128, 2);
}

int Mx4Product(const Call& c, const Mx4& a, const Mx4& b, void* out, int dtype, int64_t k, bool gated,
               bool early_weights) {
  const int64_t tokens = a.rows, rows = b.rows;
  const int kblocks = (int)((k + FDMOE_MX4_STAGE_K - 1) / FDMOE_MX4_STAGE_K);
  const int chunks = (int)fdmoe::ScaleChunks(k), up_block = (int)((rows + 127) / 128);
  const int epi = gated ? (dtype == kF32 ? FDMOE_EPI_GATED_F32 : FDMOE_EPI_GATED)
                        : (dtype == kF32 ? FDMOE_EPI_F32 : FDMOE_EPI_HALF);
  if (fdmoe::ChooseMx4Kernel(tokens, rows, gated, dtype == kF32) == fdmoe::Mx4Kernel::kStream) {
    FdmoeStreamParams p;
    memset(&p, 0, sizeof(p));
    const fdmoe::StreamPlan s = fdmoe::MakeStreamPlan((int)rows, (int)tokens, kblocks, gated, true, *c.slots);
    DENSE_TRY(Mx4Maps(c, &p.a, &p.sfa, b, k, 128));
    DENSE_TRY(Mx4Maps(c, &p.b, &p.sfb, a, k, s.tile_tokens));
    p.out = out;
    p.status = c.status;
    p.timeout_ns = c.timeout_ns;
    p.stall = c.stall;
    p.ld = rows;
    p.rows = (int32_t)rows;
    p.tokens = (int32_t)tokens;
    p.tile_tokens = s.tile_tokens;
    p.split = s.split;
    p.kblocks_each = kblocks / s.split;
    p.kblocks_more = kblocks % s.split;
    p.stages = s.stages;
    p.up_row = (int32_t)rows;
    p.sf_chunks = chunks;
    p.sf_up_block = up_block;
    p.bf16 = dtype == kBf16;
    p.tmem_cols = s.tmem_cols;
    p.early_weights = early_weights;
    return fdmoe_stream_launch(&p, epi, 1, s.smem, c.stream);
  }
  FdmoePairParams p;
  memset(&p, 0, sizeof(p));
  const int clusters = PairShape(p, c, tokens, rows, k, gated, true);
  DENSE_TRY(Mx4Maps(c, &p.product[0].a, &p.sfa, a, k, 128));
  DENSE_TRY(Mx4Maps(c, &p.product[0].b, &p.sfb, b, k, 128));
  const int size = dtype == kF32 ? 4 : 2;
  DENSE_TRY(MakeMap(c, &p.product[0].out[0], out, size, tokens, rows, rows * size, 128 / size, 32));
  p.to[0] = out;
  p.up_row = (int32_t)rows;
  p.sf_chunks = chunks;
  p.sf_up_block = up_block;
  p.bf16 = dtype == kBf16;
  return fdmoe_pair_launch(&p, epi, 1, clusters, c.stream);
}

// ------------------------------------------------------------------- checks
constexpr int64_t kMaxDim = 1 << 20;      // of a layer: hidden, intermediate, columns
constexpr int64_t kMaxTokens = 1 << 30;

int CheckFfn(const FlashMoeFfnConfig* cfg, int64_t tokens) {
  if (!cfg) return (int)cudaErrorInvalidValue;
  const int64_t H = cfg->hiddenSize, I = cfg->intermediateSize;
  if (H <= 0 || I <= 0 || H % 8 || I % 8 || H > kMaxDim || I > kMaxDim || (cfg->dtype != kBf16 && cfg->dtype != kF16)) {
    MOE_ERROR_LOG("unsupported block hidden=%lld intermediate=%lld dtype=%d (sizes multiples of 8; bf16 or fp16)",
                  (long long)H, (long long)I, cfg->dtype);
    return (int)cudaErrorInvalidValue;
  }
  if (tokens < 0 || tokens > kMaxTokens) return (int)cudaErrorInvalidValue;
  return 0;
}

int CheckMx4(int64_t batch, int64_t rows, int64_t cols) {
  if (batch < 0 || batch > 65535 || rows < 0 || rows > kMaxTokens || cols <= 0 || cols % FDMOE_MX4_BLOCK || cols > kMaxDim ||
      batch * rows > kMaxTokens) {
    MOE_ERROR_LOG("unsupported matrix batch=%lld rows=%lld cols=%lld (columns: a multiple of 32)", (long long)batch,
                  (long long)rows, (long long)cols);
    return (int)cudaErrorInvalidValue;
  }
  return 0;
}

// Memory of a call.  What it writes may lie on nothing that it reads or writes elsewhere: launches of a call overlap, and
// the products of a backward pass are one launch.
struct Range {
  const void* base;  // NULL: not there
  size_t bytes;
};
bool Apart(const Range& a, const Range& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.base), y = reinterpret_cast<uintptr_t>(b.base);
  return !x || !y || x + a.bytes <= y || y + b.bytes <= x;
}
int CheckApart(std::initializer_list<Range> written, std::initializer_list<Range> read) {
  for (auto w = written.begin(); w != written.end(); ++w) {
    bool apart = true;
    for (const Range& r : read) apart = apart && Apart(*w, r);
    for (auto other = written.begin(); other != w; ++other) apart = apart && Apart(*w, *other);
    if (!apart) {
      MOE_ERROR_LOG("results or scratch lie on other memory of the call");
      return (int)cudaErrorInvalidValue;
    }
  }
  return 0;
}
size_t Bytes(int64_t rows, int64_t cols, int size) { return (size_t)rows * cols * size; }

}  // namespace

// ---------------------------------------------------------------- C exports
extern "C" int FlashMoeDenseStatus(uint32_t* code, int reset) {
  std::lock_guard<std::mutex> lock(g_shared.mutex);
  volatile uint32_t* s = g_shared.status;
  if (code) *code = s ? *s : 0;
  if (reset && s) *s = 0;
  return 0;
}

// Scratch of a forward call: h, unless it is kept; of a backward call: the gradients of the projections.
extern "C" size_t FlashMoeFfnWorkspaceBytes(const FlashMoeFfnConfig* cfg, int64_t tokensNum, int backward) {
  if (CheckFfn(cfg, tokensNum) != 0) return 0;
  return fdmoe::AlignBytes((size_t)tokensNum * cfg->intermediateSize * (backward ? 4 : 2));
}

extern "C" size_t FlashMoeFfnSavedBytes(const FlashMoeFfnConfig* cfg, int64_t tokensNum) {
  if (CheckFfn(cfg, tokensNum) != 0) return 0;
  return Saved::Bytes(tokensNum, cfg->intermediateSize);
}

extern "C" int FlashMoeFfnForward(const FlashMoeFfnConfig* cfg, const void* x, const void* w13, const void* w2, void* y,
                                  void* savedFor, void* workspace, size_t workspaceBytes, int64_t T, void* stream) {
  DENSE_TRY(CheckFfn(cfg, T));
  if (T == 0) return 0;
  if (!x || !w13 || !w2 || !y || !Aligned(x) || !Aligned(w13) || !Aligned(w2) || !Aligned(y) || !Aligned(savedFor) ||
      !Aligned(workspace) || (!savedFor && (!workspace || workspaceBytes < FlashMoeFfnWorkspaceBytes(cfg, T, 0))))
    return (int)cudaErrorInvalidValue;
  const int64_t H = cfg->hiddenSize, I = cfg->intermediateSize;
  const Range scratch = savedFor ? Range{savedFor, Saved::Bytes(T, I)} : Range{workspace, Bytes(T, I, 2)};
  DENSE_TRY(CheckApart({{y, Bytes(T, H, 2)}, scratch}, {{w13, Bytes(2 * I, H, 2)}, {w2, Bytes(H, I, 2)}}));
  DENSE_TRY(CheckApart({scratch}, {{x, Bytes(T, H, 2)}}));  // the last product writes y, the first reads x
  Call c;
  DENSE_TRY(BeginCall(&c, stream));
  const bool bf16 = cfg->dtype == kBf16;
  if (!savedFor && fdmoe::UseStream(T, 6 * H * I)) {
    DENSE_TRY(StreamProduct(c, x, w13, workspace, T, I, H, true, bf16, false));
    return StreamProduct(c, workspace, w2, y, T, H, I, false, bf16, true);
  }
  const Saved saved = savedFor ? Saved(savedFor, T, I) : Saved();
  void* h = savedFor ? saved.h : workspace;
  DENSE_TRY(GatedProduct(c, x, w13, h, saved, T, H, I, bf16));
  return PairProduct(c, {{h, T, I, false}, {w2, H, I, false}, y}, bf16);
}

extern "C" int FlashMoeTestDenseStall(int on) {
  g_stall = on != 0;
  return 0;
}

extern "C" int FlashMoeTestFfnStall(const FlashMoeFfnConfig* cfg, const void* x, const void* w13, const void* w2, void* y,
                                    void* workspace, size_t workspaceBytes, int64_t tokensNum, void* stream) {
  const bool before = g_stall;
  g_stall = true;
  const int r = FlashMoeFfnForward(cfg, x, w13, w2, y, nullptr, workspace, workspaceBytes, tokensNum, stream);
  g_stall = before;
  return r;
}

extern "C" int FlashMoeFfnBackward(const FlashMoeFfnConfig* cfg, const void* dy, const void* x, const void* w13,
                                   const void* w2, const void* savedBy, void* dx, void* dw13, void* dw2, void* workspace,
                                   size_t workspaceBytes, int64_t T, void* stream) {
  DENSE_TRY(CheckFfn(cfg, T));
  const int64_t H = cfg->hiddenSize, I = cfg->intermediateSize;
  if (!Aligned(dx) || !Aligned(dw13) || !Aligned(dw2)) return (int)cudaErrorInvalidValue;
  if (T == 0) {
    if (dw13) DENSE_CHECK(cudaMemsetAsync(dw13, 0, (size_t)(2 * I * H) * 2, static_cast<cudaStream_t>(stream)));
    if (dw2) DENSE_CHECK(cudaMemsetAsync(dw2, 0, (size_t)(I * H) * 2, static_cast<cudaStream_t>(stream)));
    return 0;
  }
  if (!dy || !x || !w13 || !w2 || !savedBy || !workspace || !Aligned(dy) || !Aligned(x) || !Aligned(w13) || !Aligned(w2) ||
      !Aligned(savedBy) || !Aligned(workspace) || workspaceBytes < FlashMoeFfnWorkspaceBytes(cfg, T, 1))
    return (int)cudaErrorInvalidValue;
  if (!dx && !dw13 && !dw2) return 0;
  DENSE_TRY(CheckApart({{dx, Bytes(T, H, 2)}, {dw13, Bytes(2 * I, H, 2)}, {dw2, Bytes(H, I, 2)},
                        {workspace, Bytes(T, I, 4)}},
                       {{dy, Bytes(T, H, 2)}, {x, Bytes(T, H, 2)}, {w13, Bytes(2 * I, H, 2)}, {w2, Bytes(H, I, 2)},
                        {savedBy, Saved::Bytes(T, I)}}));
  Call c;
  DENSE_TRY(BeginCall(&c, stream));
  const bool bf16 = cfg->dtype == kBf16;
  const Saved saved(savedBy, T, I);
  void* dgu = workspace;
  if (dx || dw13) DENSE_TRY(GatedGradient(c, dy, w2, saved, dgu, T, H, I, bf16));
  Product work[FDMOE_PAIR_PRODUCTS];
  int n = 0;
  if (dx) work[n++] = {{dgu, T, 2 * I, false}, {w13, 2 * I, H, true}, dx};
  if (dw13) work[n++] = {{dgu, T, 2 * I, true}, {x, T, H, true}, dw13};
  if (dw2) work[n++] = {{dy, T, H, true}, {saved.h, T, I, true}, dw2};
  return PairProducts(c, work, n, bf16);
}

extern "C" size_t FlashMoeMx4ScaleBytes(int64_t batch, int64_t rows, int64_t cols) {
  if (CheckMx4(batch, rows, cols) != 0) return 0;
  return fdmoe::ScaleBytes(batch, rows, cols);
}

extern "C" int FlashMoeMx4Quantize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols,
                                   int64_t batchStride, int64_t rowStride, void* values, void* scales, void* stream) {
  DENSE_TRY(CheckMx4(batch, rows, cols));
  if (dtype != kBf16 && dtype != kF32 && dtype != kF16) return (int)cudaErrorInvalidValue;
  if (batch == 0 || rows == 0) return 0;
  const int64_t per16 = dtype == kF32 ? 4 : 8;
  if (!x || !values || !scales || !Aligned(x) || !Aligned(values) || !Aligned(scales) || batchStride < 0 || rowStride < 0 ||
      batchStride % per16 || rowStride % per16)
    return (int)cudaErrorInvalidValue;
  const int64_t span = (batch - 1) * batchStride + (rows - 1) * rowStride + cols;
  DENSE_TRY(CheckApart({{values, Bytes(batch * rows, cols / 2, 1)}, {scales, fdmoe::ScaleBytes(batch, rows, cols)}},
                       {{x, Bytes(span, 1, dtype == kF32 ? 4 : 2)}}));
  {
    std::lock_guard<std::mutex> lock(g_shared.mutex);
    DENSE_TRY(RefuseAfterError());
  }
  return fdmoe_mx4_quantize(x, dtype, batch, rows, cols, batchStride, rowStride, values, scales, stream);
}

extern "C" int FlashMoeMx4Dequantize(const void* values, const void* scales, int64_t batch, int64_t rows, int64_t cols,
                                     int dtype, void* out, void* stream) {
  DENSE_TRY(CheckMx4(batch, rows, cols));
  if (dtype != kBf16 && dtype != kF32 && dtype != kF16) return (int)cudaErrorInvalidValue;
  if (batch == 0 || rows == 0) return 0;
  if (!values || !scales || !out || !Aligned(values) || !Aligned(scales) || !Aligned(out)) return (int)cudaErrorInvalidValue;
  DENSE_TRY(CheckApart({{out, Bytes(batch * rows, cols, dtype == kF32 ? 4 : 2)}},
                       {{values, Bytes(batch * rows, cols / 2, 1)}, {scales, fdmoe::ScaleBytes(batch, rows, cols)}}));
  {
    std::lock_guard<std::mutex> lock(g_shared.mutex);
    DENSE_TRY(RefuseAfterError());
  }
  return fdmoe_mx4_dequantize(values, scales, batch, rows, cols, dtype, out, stream);
}

extern "C" int FlashMoeMx4Matmul(const void* aValues, const void* aScales, const void* bValues, const void* bScales,
                                 void* out, int dtype, int64_t m, int64_t n, int64_t k, int gated, void* stream) {
  DENSE_TRY(CheckMx4(1, m, k));
  DENSE_TRY(CheckMx4(gated ? 2 : 1, n, k));
  if (dtype != kBf16 && dtype != kF32 && dtype != kF16) return (int)cudaErrorInvalidValue;
  if (m == 0 || n == 0) return 0;
  if (!aValues || !aScales || !bValues || !bScales || !out || !Aligned(aValues) || !Aligned(aScales) || !Aligned(bValues) ||
      !Aligned(bScales) || !Aligned(out))
    return (int)cudaErrorInvalidValue;
  if (fdmoe::ChooseMx4Kernel(m, n, gated != 0, dtype == kF32) == fdmoe::Mx4Kernel::kNone) {
    MOE_ERROR_LOG("unsupported product m=%lld n=%lld (above 8388480 of either, n is a multiple of 8, of fp32 results of 4)",
                  (long long)m, (long long)n);
    return (int)cudaErrorInvalidValue;
  }
  const int parts = gated ? 2 : 1;
  DENSE_TRY(CheckApart({{out, Bytes(m, n, dtype == kF32 ? 4 : 2)}},
                       {{aValues, Bytes(m, k / 2, 1)}, {aScales, fdmoe::ScaleBytes(1, m, k)},
                        {bValues, Bytes(parts * n, k / 2, 1)}, {bScales, fdmoe::ScaleBytes(parts, n, k)}}));
  Call c;
  DENSE_TRY(BeginCall(&c, stream));
  return Mx4Product(c, {aValues, aScales, m, 1}, {bValues, bScales, n, gated ? 2 : 1}, out, dtype, k, gated != 0, false);
}

// Workspace of the block on 4-bit weights: 4-bit tokens, activations, 4-bit activations.
namespace {
struct Mx4FfnLayout {
  size_t xv, xs, h, hv, hs, total;
};
Mx4FfnLayout MakeMx4FfnLayout(int64_t T, int64_t H, int64_t I) {
  Mx4FfnLayout l;
  size_t at = 0;
  l.xv = at;
  at += fdmoe::AlignBytes((size_t)T * H / 2);
  l.xs = at;
  at += fdmoe::AlignBytes(fdmoe::ScaleBytes(1, T, H));
  l.h = at;
  at += fdmoe::AlignBytes((size_t)T * I * 2);
  l.hv = at;
  at += fdmoe::AlignBytes((size_t)T * I / 2);
  l.hs = at;
  at += fdmoe::AlignBytes(fdmoe::ScaleBytes(1, T, I));
  l.total = at;
  return l;
}
}  // namespace

extern "C" size_t FlashMoeMx4FfnWorkspaceBytes(const FlashMoeFfnConfig* cfg, int64_t tokensNum) {
  if (CheckFfn(cfg, tokensNum) != 0 || cfg->hiddenSize % FDMOE_MX4_BLOCK || cfg->intermediateSize % FDMOE_MX4_BLOCK) return 0;
  return MakeMx4FfnLayout(tokensNum, cfg->hiddenSize, cfg->intermediateSize).total;
}

extern "C" int FlashMoeMx4FfnForward(const FlashMoeFfnConfig* cfg, const void* x, const void* w13Values,
                                     const void* w13Scales, const void* w2Values, const void* w2Scales, void* y,
                                     void* workspace, size_t workspaceBytes, int64_t T, void* stream) {
  DENSE_TRY(CheckFfn(cfg, T));
  const int64_t H = cfg->hiddenSize, I = cfg->intermediateSize;
  DENSE_TRY(CheckMx4(1, T, H));
  DENSE_TRY(CheckMx4(2, I, H));
  DENSE_TRY(CheckMx4(1, H, I));
  if (T == 0) return 0;
  if (!x || !w13Values || !w13Scales || !w2Values || !w2Scales || !y || !workspace || !Aligned(x) || !Aligned(w13Values) ||
      !Aligned(w13Scales) || !Aligned(w2Values) || !Aligned(w2Scales) || !Aligned(y) || !Aligned(workspace) ||
      workspaceBytes < FlashMoeMx4FfnWorkspaceBytes(cfg, T))
    return (int)cudaErrorInvalidValue;
  const Mx4FfnLayout l = MakeMx4FfnLayout(T, H, I);
  DENSE_TRY(CheckApart({{y, Bytes(T, H, 2)}, {workspace, l.total}},
                       {{w13Values, Bytes(2 * I, H / 2, 1)}, {w13Scales, fdmoe::ScaleBytes(2, I, H)},
                        {w2Values, Bytes(H, I / 2, 1)}, {w2Scales, fdmoe::ScaleBytes(1, H, I)}}));
  DENSE_TRY(CheckApart({{workspace, l.total}}, {{x, Bytes(T, H, 2)}}));  // x is quantised before y is written
  Call c;
  DENSE_TRY(BeginCall(&c, stream));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  DENSE_TRY(fdmoe_mx4_quantize(x, cfg->dtype, 1, T, H, 0, H, ws + l.xv, ws + l.xs, stream));
  DENSE_TRY(Mx4Product(c, {ws + l.xv, ws + l.xs, T, 1}, {w13Values, w13Scales, I, 2}, ws + l.h, cfg->dtype, H, true, true));
  DENSE_TRY(fdmoe_mx4_quantize(ws + l.h, cfg->dtype, 1, T, I, 0, I, ws + l.hv, ws + l.hs, stream));
  return Mx4Product(c, {ws + l.hv, ws + l.hs, T, 1}, {w2Values, w2Scales, H, 1}, y, cfg->dtype, I, false, true);
}
