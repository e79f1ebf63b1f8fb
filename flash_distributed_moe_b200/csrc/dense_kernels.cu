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
    case FDMOE_EPI_GATED_SAVE: return launch_pair<false, FDMOE_EPI_GATED_SAVE>(*p, clusters, s);
    case FDMOE_EPI_GATED_GRAD: return launch_pair<false, FDMOE_EPI_GATED_GRAD>(*p, clusters, s);
  }
  return cudaErrorInvalidValue;
}

// What the device holds at once is asked for kernels that do nothing and have the shape of the real ones, whose use
// of TMEM the occupancy calculator takes for all of an SM's.
namespace {
__global__ void __launch_bounds__(kPairThreads) pair_shape() {}
__global__ void __launch_bounds__(kStreamThreads) stream_shape() {
  __shared__ volatile uint8_t barriers[256];
  barriers[0] = 0;
}

template <typename F>
int count_clusters(F kernel, int threads, int smem, int size, int* out) {
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const LaunchConfig l(dim3(size), threads, smem, size, nullptr);
  return cudaOccupancyMaxActiveClusters(out, kernel, &l.cfg);
}
}  // namespace

extern "C" int fdmoe_pair_clusters(int size, int* out) {
  return count_clusters(pair_shape, kPairThreads, PairShape<false, FDMOE_EPI_HALF>::kSmem, size, out);
}
extern "C" int fdmoe_stream_clusters(int size, int smem, int* out) {
  return count_clusters(stream_shape, kStreamThreads, smem, size, out);
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
