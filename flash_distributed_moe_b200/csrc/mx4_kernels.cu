// 4-bit microscaled values: quantisation, its inverse, and the instances of the matrix products on them.
//
// Values: E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even element in the low half.  Every 32
// elements along a row share a scale 2^(byte - 127) with byte = max(exponent field of the largest magnitude - 2, 0),
// i.e. 2^(floor(log2 max) - 2), so that the largest element lands in [4, 8) and saturates at 6.  A block that holds a
// NaN or an infinity gets the scale 255, which stands for NaN.
// Scales lie in blocks of 512 bytes for 128 rows and 128 columns, as the tensor cores take them: the scale of row r
// and block c of 32 columns is byte (r % 32) * 16 + (r / 32) * 4 + c of it.  Blocks of the same rows follow each other
// (an even number of them), and a matrix of a batch starts with a new block of rows.  Scales of rows and columns that
// do not exist are 0, values of no consequence there.
#include "dense_launch.cuh"

namespace fdmoe {
namespace dense {
namespace {

constexpr int kQuantRows = 128, kQuantBlocks = 8;  // a CTA's tile: 128 rows x 256 columns, 1 KB of scales
constexpr int kQuantThreads = 256;
constexpr int kQuantBatch = 4;  // rows that a thread loads before it works on the first

// Four lanes share a block of 32 elements, eight each.

// Eight elements as they are stored, and in 32 bits.
template <bool F32>
struct Eight {
  uint4 w[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* x, int64_t at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) w[i] = __ldg(p + i);
  }
  __device__ __forceinline__ void get(bool bf16, float (&v)[8]) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 8; i += F32 ? 1 : 2) {
      if constexpr (F32)
        v[i] = __uint_as_float(u[i]);
      else
        unpack2(u[i / 2], bf16, v[i], v[i + 1]);
    }
  }
};

__device__ __forceinline__ uint32_t to_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ void from_e2m1x8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(h[i], false, v[2 * i], v[2 * i + 1]);
}

struct QuantParams {
  const void* x;
  uint8_t* values;
  uint8_t* scales;
  int64_t rows, cols, batch_stride, row_stride;
  int dtype;  // 0 bf16, 1 fp32, 2 fp16
};

template <bool F32>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantize_kernel(const QuantParams p) {
  __shared__ __align__(16) uint8_t sc[2 * kScaleBlock];
  ptx::grid_wait_dependency();
  ptx::grid_launch_dependents();
  const int64_t batch = blockIdx.z, row0 = (int64_t)blockIdx.x * kQuantRows;
  const int64_t blocks = p.cols / FDMOE_MX4_BLOCK, blk0 = (int64_t)blockIdx.y * kQuantBlocks;
  const int rows = (int)min((int64_t)kQuantRows, p.rows - row0);
  if (threadIdx.x < 64) reinterpret_cast<uint4*>(sc)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int part = threadIdx.x & 3, b = (threadIdx.x >> 2) & 7, r0 = threadIdx.x >> 5;
  const int64_t col = (blk0 + b) * FDMOE_MX4_BLOCK + part * 8;
  const bool in_cols = blk0 + b < blocks;
  const uint32_t group = 0xFu << (threadIdx.x & 28);
  if (in_cols) {
    for (int r1 = r0; r1 < rows; r1 += kQuantBatch * kQuantThreads / 32) {
      Eight<F32> in[kQuantBatch];
#pragma unroll
      for (int i = 0; i < kQuantBatch; ++i) {
        const int r = r1 + i * kQuantThreads / 32;
        if (r < rows) in[i].load(p.x, batch * p.batch_stride + (row0 + r) * p.row_stride + col);
      }
#pragma unroll
      for (int i = 0; i < kQuantBatch; ++i) {
        const int r = r1 + i * kQuantThreads / 32;
        if (r >= rows) break;
        float v[8];
        in[i].get(p.dtype == 0, v);
        uint32_t top = 0;  // bits of the largest magnitude: infinities and NaN are above every number
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(group, top, 1));
        top = max(top, __shfl_xor_sync(group, top, 2));
        const uint32_t field = top >> 23;
        const uint32_t scale = field == 255 ? 255 : (field > 2 ? field - 2 : 0);
        const float inv = __uint_as_float((254u - min(scale, 253u)) << 23);  // 2^-(scale - 127), exact
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= inv;
        reinterpret_cast<uint32_t*>(p.values)[((batch * p.rows + row0 + r) * p.cols + col) >> 3] = to_e2m1x8(v);
        if (part == 0) sc[(b >> 2) * kScaleBlock + (r & 31) * 16 + (r >> 5) * 4 + (b & 3)] = (uint8_t)scale;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int64_t chunks = (int64_t)gridDim.y * 2;
    uint8_t* dst = p.scales + ((batch * gridDim.x + blockIdx.x) * chunks + blockIdx.y * 2) * kScaleBlock;
    reinterpret_cast<uint4*>(dst)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
  }
}

struct DequantParams {
  const uint8_t* values;
  const uint8_t* scales;
  void* out;
  int64_t rows, cols;
  int dtype;
};

template <bool F32>
__global__ void __launch_bounds__(kQuantThreads) mx4_dequantize_kernel(const DequantParams p) {
  __shared__ __align__(16) uint8_t sc[2 * kScaleBlock];
  ptx::grid_wait_dependency();
  ptx::grid_launch_dependents();
  const int64_t batch = blockIdx.z, row0 = (int64_t)blockIdx.x * kQuantRows;
  const int64_t blocks = p.cols / FDMOE_MX4_BLOCK, blk0 = (int64_t)blockIdx.y * kQuantBlocks;
  const int rows = (int)min((int64_t)kQuantRows, p.rows - row0);
  if (threadIdx.x < 64) {
    const int64_t chunks = (int64_t)gridDim.y * 2;
    const uint8_t* src = p.scales + ((batch * gridDim.x + blockIdx.x) * chunks + blockIdx.y * 2) * kScaleBlock;
    reinterpret_cast<uint4*>(sc)[threadIdx.x] = reinterpret_cast<const uint4*>(src)[threadIdx.x];
  }
  __syncthreads();
  const int part = threadIdx.x & 3, b = (threadIdx.x >> 2) & 7, r0 = threadIdx.x >> 5;
  const int64_t col = (blk0 + b) * FDMOE_MX4_BLOCK + part * 8;
  if (blk0 + b >= blocks) return;
  for (int r1 = r0; r1 < rows; r1 += kQuantBatch * kQuantThreads / 32) {
    uint32_t in[kQuantBatch];
#pragma unroll
    for (int i = 0; i < kQuantBatch; ++i) {
      const int r = r1 + i * kQuantThreads / 32;
      if (r < rows) in[i] = __ldg(reinterpret_cast<const uint32_t*>(p.values) + (((batch * p.rows + row0 + r) * p.cols + col) >> 3));
    }
#pragma unroll
    for (int i = 0; i < kQuantBatch; ++i) {
      const int r = r1 + i * kQuantThreads / 32;
      if (r >= rows) break;
      const int64_t at = (batch * p.rows + row0 + r) * p.cols + col;
      const uint32_t byte = sc[(b >> 2) * kScaleBlock + (r & 31) * 16 + (r >> 5) * 4 + (b & 3)];
      const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
      float v[8];
      from_e2m1x8(in[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= scale;
      if constexpr (F32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        const bool bf16 = p.dtype == 0;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) =
            make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16), pack2(v[6], v[7], bf16));
      }
    }
  }
}

dim3 quant_grid(int64_t batch, int64_t rows, int64_t cols) {
  return dim3((unsigned)((rows + kQuantRows - 1) / kQuantRows),
              (unsigned)((cols + FDMOE_MX4_STAGE_K - 1) / FDMOE_MX4_STAGE_K), (unsigned)batch);
}

}  // namespace
}  // namespace dense
}  // namespace fdmoe

using namespace fdmoe::dense;

extern "C" int fdmoe_mx4_quantize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols,
                                  int64_t batch_stride, int64_t row_stride, void* values, void* scales, void* stream) {
  const QuantParams p{x, static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales), rows, cols, batch_stride,
                      row_stride, dtype};
  const LaunchConfig l(quant_grid(batch, rows, cols), kQuantThreads, 0, 1, static_cast<cudaStream_t>(stream));
  return dtype == 1 ? cudaLaunchKernelEx(&l.cfg, mx4_quantize_kernel<true>, p) : cudaLaunchKernelEx(&l.cfg, mx4_quantize_kernel<false>, p);
}

extern "C" int fdmoe_mx4_dequantize(const void* values, const void* scales, int64_t batch, int64_t rows, int64_t cols,
                                    int dtype, void* out, void* stream) {
  const DequantParams p{static_cast<const uint8_t*>(values), static_cast<const uint8_t*>(scales), out, rows, cols, dtype};
  const LaunchConfig l(quant_grid(batch, rows, cols), kQuantThreads, 0, 1, static_cast<cudaStream_t>(stream));
  return dtype == 1 ? cudaLaunchKernelEx(&l.cfg, mx4_dequantize_kernel<true>, p) : cudaLaunchKernelEx(&l.cfg, mx4_dequantize_kernel<false>, p);
}

cudaError_t fdmoe_pair_launch_mx4(const FdmoePairParams& p, int epi, int clusters, cudaStream_t s) {
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_pair<true, FDMOE_EPI_HALF>(p, clusters, s);
    case FDMOE_EPI_F32: return launch_pair<true, FDMOE_EPI_F32>(p, clusters, s);
    case FDMOE_EPI_GATED: return launch_pair<true, FDMOE_EPI_GATED>(p, clusters, s);
    case FDMOE_EPI_GATED_F32: return launch_pair<true, FDMOE_EPI_GATED_F32>(p, clusters, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t fdmoe_stream_launch_mx4(const FdmoeStreamParams& p, int epi, int smem, cudaStream_t s) {
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_stream<true, FDMOE_EPI_HALF>(p, smem, s);
    case FDMOE_EPI_F32: return launch_stream<true, FDMOE_EPI_F32>(p, smem, s);
    case FDMOE_EPI_GATED: return launch_stream<true, FDMOE_EPI_GATED>(p, smem, s);
    case FDMOE_EPI_GATED_F32: return launch_stream<true, FDMOE_EPI_GATED_F32>(p, smem, s);
  }
  return cudaErrorInvalidValue;
}
