// Attention weights on the tensor cores, head_dim 96 (weights_step.cuh, weights_window.cuh).
#include "weights_tc_launch.cuh"

namespace kvb {
cudaError_t launch_weights_tc_96(const WeightsArgs& a, cudaStream_t s) {
  return weights_tc::launch<96>(a, s);
}
}  // namespace kvb
