// Attention weights on the tensor cores, head_dim 64 (weights_step.cuh, weights_window.cuh).
#include "weights_tc_launch.cuh"

namespace kvb {
cudaError_t launch_weights_tc_64(const WeightsArgs& a, cudaStream_t s) {
  return weights_tc::launch<64>(a, s);
}
}  // namespace kvb
