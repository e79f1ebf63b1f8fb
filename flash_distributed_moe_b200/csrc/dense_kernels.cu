// Kernels of the dense gated feed-forward block (16-bit operands) and the entry that picks an instance.
#include "dense_launch.cuh"

using namespace fdmoe::dense;

cudaError_t fdmoe_pair_launch_mx4(const FdmoePairParams& p, int epi, int clusters, cudaStream_t stream);
cudaError_t fdmoe_stream_launch_mx4(const FdmoeStreamParams& p, int epi, int smem, cudaStream_t stream);

extern "C" int fdmoe_pair_launch(const FdmoePairParams* p, int epi, int mx4, int clusters, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mx4) return fdmoe_pair_launch_mx4(*p, epi, clusters, s);
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_pair<false, FDMOE_EPI_HALF>(*p, clusters, s);
    case FDMOE_EPI_GATED: return launch_pair<false, FDMOE_EPI_GATED>(*p, clusters, s);
    case FDMOE_EPI_GATED_GRAD: return launch_pair<false, FDMOE_EPI_GATED_GRAD>(*p, clusters, s);
  }
  return cudaErrorInvalidValue;
}

// All instances of a kernel have the same threads and nearly the same shared memory, so one stands for all.
extern "C" int fdmoe_pair_clusters(int size, int* out) {
  constexpr int smem = PairShape<false, FDMOE_EPI_HALF>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(pair_gemm<false, FDMOE_EPI_HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const LaunchConfig l(dim3(size), kPairThreads, smem, size, nullptr);
  return cudaOccupancyMaxActiveClusters(out, pair_gemm<false, FDMOE_EPI_HALF>, &l.cfg);
}
extern "C" int fdmoe_stream_clusters(int size, int smem, int* out) {
  const cudaError_t e = cudaFuncSetAttribute(stream_gemm<false, FDMOE_EPI_GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kStreamSmemMax);
  if (e != cudaSuccess) return e;
  const LaunchConfig l(dim3(size), kStreamThreads, smem, size, nullptr);
  return cudaOccupancyMaxActiveClusters(out, stream_gemm<false, FDMOE_EPI_GATED>, &l.cfg);
}

extern "C" int fdmoe_stream_launch(const FdmoeStreamParams* p, int epi, int mx4, int smem, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mx4) return fdmoe_stream_launch_mx4(*p, epi, smem, s);
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_stream<false, FDMOE_EPI_HALF>(*p, smem, s);
    case FDMOE_EPI_GATED: return launch_stream<false, FDMOE_EPI_GATED>(*p, smem, s);
  }
  return cudaErrorInvalidValue;
}
