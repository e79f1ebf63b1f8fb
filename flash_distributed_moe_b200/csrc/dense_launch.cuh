// Launching the kernels of dense_gemm.cuh.
#pragma once
#include <atomic>

#include "dense_gemm.cuh"

namespace fdmoe {
namespace dense {

// Raises a kernel's shared-memory limit once per device.
template <typename F>
cudaError_t prepare_kernel(F kernel, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

// A launch with clusters of `cluster` CTAs along x.
struct LaunchConfig {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  LaunchConfig(dim3 grid, int threads, int smem, int cluster, cudaStream_t stream) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
};

template <bool MX4, int EPI, bool BF16>
cudaError_t launch_pair_of(const FdmoePairParams& p, int clusters, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = PairShape<MX4, EPI>::kSmem;
  cudaError_t e = prepare_kernel(pair_gemm<MX4, EPI, BF16>, smem, done);
  if (e != cudaSuccess) return e;
  const LaunchConfig l(dim3(clusters * 2 * p.split), kPairThreads, smem, 2 * p.split, stream);
  return cudaLaunchKernelEx(&l.cfg, pair_gemm<MX4, EPI, BF16>, p);
}
template <bool MX4, int EPI>
cudaError_t launch_pair(const FdmoePairParams& p, int clusters, cudaStream_t stream) {
  if constexpr (EPI == FDMOE_EPI_F32 || EPI == FDMOE_EPI_GATED_F32)
    return launch_pair_of<MX4, EPI, true>(p, clusters, stream);
  return p.bf16 ? launch_pair_of<MX4, EPI, true>(p, clusters, stream) : launch_pair_of<MX4, EPI, false>(p, clusters, stream);
}

constexpr int kStreamSmemMax = 227 * 1024 - 1024;  // beside the barriers in static shared memory

template <bool MX4, int EPI>
cudaError_t launch_stream(const FdmoeStreamParams& p, int smem, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  cudaError_t e = prepare_kernel(stream_gemm<MX4, EPI>, kStreamSmemMax, done);
  if (e != cudaSuccess) return e;
  const LaunchConfig l(dim3(p.split, (p.rows + FDMOE_STREAM_ROWS - 1) / FDMOE_STREAM_ROWS,
                            (p.tokens + p.tile_tokens - 1) / p.tile_tokens),
                       kStreamThreads, smem, p.split, stream);
  return cudaLaunchKernelEx(&l.cfg, stream_gemm<MX4, EPI>, p);
}

}  // namespace dense
}  // namespace fdmoe
