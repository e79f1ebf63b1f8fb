// Kernels of the dense gated feed-forward block (16-bit operands) and the entry that picks an instance.
#include "dense_launch.cuh"

using namespace fdmoe::dense;

cudaError_t fdmoe_pair_launch_mx4(const FdmoePairParams& p, int epi, int sms, cudaStream_t stream);
cudaError_t fdmoe_stream_launch_mx4(const FdmoeStreamParams& p, int epi, int smem, bool dependent, cudaStream_t stream);

extern "C" int fdmoe_pair_launch(const FdmoePairParams* p, int epi, int mx4, int sms, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mx4) return fdmoe_pair_launch_mx4(*p, epi, sms, s);
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_pair<false, FDMOE_EPI_HALF>(*p, sms, s);
    case FDMOE_EPI_GATED: return launch_pair<false, FDMOE_EPI_GATED>(*p, sms, s);
    case FDMOE_EPI_GATED_GRAD: return launch_pair<false, FDMOE_EPI_GATED_GRAD>(*p, sms, s);
  }
  return cudaErrorInvalidValue;
}

extern "C" int fdmoe_stream_launch(const FdmoeStreamParams* p, int epi, int mx4, int smem, int dependent, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mx4) return fdmoe_stream_launch_mx4(*p, epi, smem, dependent != 0, s);
  switch (epi) {
    case FDMOE_EPI_HALF: return launch_stream<false, FDMOE_EPI_HALF>(*p, smem, dependent != 0, s);
    case FDMOE_EPI_GATED: return launch_stream<false, FDMOE_EPI_GATED>(*p, smem, dependent != 0, s);
  }
  return cudaErrorInvalidValue;
}
