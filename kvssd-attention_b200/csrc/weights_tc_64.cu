// Attention weights on the tensor cores, head_dim 64 (kernels: weights_tc.cuh).
#include "weights_tc.cuh"

namespace kvb {
cudaError_t launch_weights_tc_64(const WeightsArgs& a, cudaStream_t s) {
  return weights_tc::launch<64>(a, s);
}
}  // namespace kvb
