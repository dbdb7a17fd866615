// Attention weights on the tensor cores, head_dim 256 (kernels: weights_tc.cuh).
#include "weights_tc.cuh"

namespace kvb {
cudaError_t launch_weights_tc_256(const WeightsArgs& a, cudaStream_t s) {
  return weights_tc::launch<256>(a, s);
}
}  // namespace kvb
