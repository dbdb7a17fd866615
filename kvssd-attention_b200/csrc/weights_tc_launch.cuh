// Choice and launches of the tensor-core kernels of one head_dim.
#pragma once

#include "weights_step.cuh"
#include "weights_umma.cuh"
#include "weights_window.cuh"

namespace kvb {
namespace weights_tc {

template <int BITS, int D, int UNIT, bool LO>
cudaError_t launch_shape(const WeightsArgs& a, cudaStream_t s) {
  if constexpr (D <= 128 || BITS == 2 || !LO)
    if (weights_umma::takes<BITS, D, LO>(a)) return weights_umma::launch<BITS, D, LO>(a, s);
  Job j{};
  j.a = a;
  j.rows = a.queries * (a.qh / a.kvh);
  j.tiles_per_block = (a.bt + tile_rows(D, UNIT) - 1) / tile_rows(D, UNIT);
  j.total_tiles = a.n_sel * j.tiles_per_block;
  if (!a.lse_in) {
    j.parts = grid_x(j.total_tiles, a.kvh, 1, kWarps, resident(D, LO));
    if (j.parts > a.parts_room) return cudaErrorInvalidValue;
    const cudaError_t e = launch_mode<BITS, D, UNIT, LO, kLse>(j, s);
    if (e != cudaSuccess) return e;
  }
  if (j.rows <= 8) return launch_step<BITS, D, UNIT, LO>(j, s);
  return launch_mode<BITS, D, UNIT, LO, kWindow>(j, s);
}

template <int D>
cudaError_t launch(const WeightsArgs& a, cudaStream_t s) {
  const bool lo = a.dtype == kQF32 || a.dtype == kQF64;
  if (a.bits == 4) {
    if (a.group % 32 == 0) return lo ? launch_shape<4, D, 32, true>(a, s) : launch_shape<4, D, 32, false>(a, s);
    return lo ? launch_shape<4, D, 16, true>(a, s) : launch_shape<4, D, 16, false>(a, s);
  }
  if (a.group % 32 == 0) return lo ? launch_shape<2, D, 32, true>(a, s) : launch_shape<2, D, 32, false>(a, s);
  return lo ? launch_shape<2, D, 16, true>(a, s) : launch_shape<2, D, 16, false>(a, s);
}

}  // namespace weights_tc
}  // namespace kvb
