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

// A CTA's tile: 128 rows x 128 columns, which share a block of scales.  Four lanes share a block of 32 elements, eight
// each; a thread has the same columns of every 16th row, and loads a batch of those rows before it works on the first:
// with 16-bit elements all eight, so that a CTA waits for memory once.
constexpr int kQuantRows = 128, kQuantThreads = 256, kQuantStep = 16;
enum { kBf16 = 0, kF32 = 1, kF16 = 2 };  // element types as in the C interface
template <int T>
constexpr int kQuantBatch = T == kF32 ? 4 : 8;

// Eight elements as they are stored, and in 32 bits.
template <int T>
struct Eight {
  uint4 w[T == kF32 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t* at) {
#pragma unroll
    for (int i = 0; i < (T == kF32 ? 2 : 1); ++i) w[i] = ptx::ld_global_u32x4(at + 16 * i);
  }
  // Bits of the largest magnitude, as stored: infinities and NaN are above every number.
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if constexpr (T == kF32) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) t = max(t, u[i] & 0x7FFFFFFFu);
      return t;
    } else {
      const uint32_t m = 0x7FFF7FFFu;
      const uint32_t t = __vmaxu2(__vmaxu2(u[0] & m, u[1] & m), __vmaxu2(u[2] & m, u[3] & m));
      return max(t & 0xFFFFu, t >> 16);
    }
  }
  // The exponent field that this magnitude has in 32 bits.
  static __device__ __forceinline__ uint32_t exponent_field(uint32_t top) {
    if constexpr (T == kF32) return top >> 23;
    if constexpr (T == kBf16) return top >> 7;
    float v, unused;
    unpack2(top, false, v, unused);
    return __float_as_uint(v) >> 23;
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 8; i += T == kF32 ? 1 : 2) {
      if constexpr (T == kF32)
        v[i] = __uint_as_float(u[i]);
      else
        unpack2(u[i / 2], T == kBf16, v[i], v[i + 1]);
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
  const uint8_t* x;
  uint8_t* values;
  uint8_t* scales;
  int64_t rows, cols, batch_stride, row_stride;  // strides in elements
};

template <int T>
__global__ void __launch_bounds__(kQuantThreads) mx4_quantize_kernel(const QuantParams p) {
  __shared__ __align__(16) uint8_t sc[kScaleBlock];
  ptx::grid_wait_dependency();
  ptx::grid_launch_dependents();
  constexpr int kSize = T == kF32 ? 4 : 2, kBatch = kQuantBatch<T>;
  const int64_t batch = blockIdx.z, row0 = (int64_t)blockIdx.x * kQuantRows;
  const int rows = (int)min((int64_t)kQuantRows, p.rows - row0);
  const int part = threadIdx.x & 3, b = (threadIdx.x >> 2) & 3, r0 = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.y * 128 + b * FDMOE_MX4_BLOCK + part * 8;
  const bool in_cols = col < p.cols;
  const uint32_t group = 0xFu << (threadIdx.x & 28);
  if (rows < kQuantRows || (int64_t)(blockIdx.y + 1) * 128 > p.cols) {  // scales that do not exist are 0
    if (threadIdx.x < kScaleBlock / 16) reinterpret_cast<uint4*>(sc)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  if (in_cols) {
    const uint8_t* x = p.x + (batch * p.batch_stride + (row0 + r0) * p.row_stride + col) * kSize;
    const int64_t x_step = p.row_stride * kQuantStep * kSize;
    uint8_t* values = p.values + (((batch * p.rows + row0 + r0) * p.cols + col) >> 1);
    const int64_t v_step = p.cols * kQuantStep / 2;
    uint8_t* scale_at = sc + r0 * 16 + b;
#pragma unroll
    for (int j = 0; j < kQuantRows / kQuantStep; j += kBatch) {
      if (r0 + j * kQuantStep >= rows) break;
      Eight<T> in[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (r0 + (j + i) * kQuantStep < rows) in[i].load(x + (j + i) * x_step);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (r0 + (j + i) * kQuantStep >= rows) break;
        uint32_t top = in[i].top();
        top = max(top, __shfl_xor_sync(group, top, 1));
        top = max(top, __shfl_xor_sync(group, top, 2));
        const uint32_t field = Eight<T>::exponent_field(top);
        const uint32_t scale = field == 255 ? 255 : (field > 2 ? field - 2 : 0);
        const float inv = __uint_as_float((254u - min(scale, 253u)) << 23);  // 2^-(scale - 127), exact
        float v[8];
        in[i].get(v);
#pragma unroll
        for (int q = 0; q < 8; q += 2) (F2(v[q], v[q + 1]) * F2(inv, inv)).get(v[q], v[q + 1]);
        *reinterpret_cast<uint32_t*>(values + (j + i) * v_step) = to_e2m1x8(v);
        // row r0 + 16 (j + i) of the tile
        if (part == 0) scale_at[((j + i) & 1) * 256 + ((j + i) >> 1) * 4] = (uint8_t)scale;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < kScaleBlock / 16) {
    uint8_t* dst = p.scales + ((batch * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y) * kScaleBlock;
    reinterpret_cast<uint4*>(dst)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
  }
}

struct DequantParams {
  const uint8_t* values;
  const uint8_t* scales;
  uint8_t* out;
  int64_t rows, cols;
  bool out32;  // `out` starts on 32 bytes
};

template <int T>
__global__ void __launch_bounds__(kQuantThreads) mx4_dequantize_kernel(const DequantParams p) {
  __shared__ __align__(16) uint8_t sc[kScaleBlock];
  ptx::grid_wait_dependency();
  ptx::grid_launch_dependents();
  constexpr int kSize = T == kF32 ? 4 : 2, kRows = kQuantRows / kQuantStep;
  const int64_t batch = blockIdx.z, row0 = (int64_t)blockIdx.x * kQuantRows;
  const int rows = (int)min((int64_t)kQuantRows, p.rows - row0);
  const int part = threadIdx.x & 3, b = (threadIdx.x >> 2) & 3, r0 = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.y * 128 + b * FDMOE_MX4_BLOCK + part * 8;
  const bool in_cols = col < p.cols;
  const int64_t at = (batch * p.rows + row0 + r0) * p.cols + col, step = p.cols * kQuantStep;
  uint32_t in[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (in_cols && r0 + i * kQuantStep < rows) in[i] = ptx::ld_global_u32(p.values + ((at + i * step) >> 1));
  if (threadIdx.x < kScaleBlock / 16) {
    const uint8_t* src = p.scales + ((batch * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y) * kScaleBlock;
    reinterpret_cast<uint4*>(sc)[threadIdx.x] = ptx::ld_global_u32x4(src + 16 * threadIdx.x);
  }
  __syncthreads();
  if (!in_cols) return;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (r0 + i * kQuantStep >= rows) break;
    const uint32_t byte = sc[r0 * 16 + b + (i & 1) * 256 + (i >> 1) * 4];
    const float scale = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
    float v[8];
    from_e2m1x8(in[i], v);
#pragma unroll
    for (int q = 0; q < 8; q += 2) (F2(v[q], v[q + 1]) * F2(scale, scale)).get(v[q], v[q + 1]);
    uint8_t* o = p.out + (at + i * step) * kSize;
    if constexpr (T == kF32) {
      if (p.out32) {  // whole sectors
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                     "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
      } else {
        reinterpret_cast<float4*>(o)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(o)[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
      constexpr bool bf16 = T == kBf16;
      *reinterpret_cast<uint4*>(o) =
          make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16), pack2(v[6], v[7], bf16));
    }
  }
}

dim3 quant_grid(int64_t batch, int64_t rows, int64_t cols) {
  return dim3((unsigned)((rows + kQuantRows - 1) / kQuantRows),
              (unsigned)((cols + FDMOE_MX4_STAGE_K - 1) / FDMOE_MX4_STAGE_K * 2), (unsigned)batch);
}

}  // namespace
}  // namespace dense
}  // namespace fdmoe

using namespace fdmoe::dense;

extern "C" int fdmoe_mx4_quantize(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols,
                                  int64_t batch_stride, int64_t row_stride, void* values, void* scales, void* stream) {
  const QuantParams p{static_cast<const uint8_t*>(x), static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales), rows,
                      cols, batch_stride, row_stride};
  const LaunchConfig l(quant_grid(batch, rows, cols), kQuantThreads, 0, 1, static_cast<cudaStream_t>(stream));
  switch (dtype) {
    case kBf16: return cudaLaunchKernelEx(&l.cfg, mx4_quantize_kernel<kBf16>, p);
    case kF32: return cudaLaunchKernelEx(&l.cfg, mx4_quantize_kernel<kF32>, p);
    case kF16: return cudaLaunchKernelEx(&l.cfg, mx4_quantize_kernel<kF16>, p);
  }
  return cudaErrorInvalidValue;
}

extern "C" int fdmoe_mx4_dequantize(const void* values, const void* scales, int64_t batch, int64_t rows, int64_t cols,
                                    int dtype, void* out, void* stream) {
  const DequantParams p{static_cast<const uint8_t*>(values), static_cast<const uint8_t*>(scales), static_cast<uint8_t*>(out),
                        rows, cols, (reinterpret_cast<uintptr_t>(out) & 31) == 0};
  const LaunchConfig l(quant_grid(batch, rows, cols), kQuantThreads, 0, 1, static_cast<cudaStream_t>(stream));
  switch (dtype) {
    case kBf16: return cudaLaunchKernelEx(&l.cfg, mx4_dequantize_kernel<kBf16>, p);
    case kF32: return cudaLaunchKernelEx(&l.cfg, mx4_dequantize_kernel<kF32>, p);
    case kF16: return cudaLaunchKernelEx(&l.cfg, mx4_dequantize_kernel<kF16>, p);
  }
  return cudaErrorInvalidValue;
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
