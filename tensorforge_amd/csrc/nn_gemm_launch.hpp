// One element type's product kernels and their choice by operand layout, tile
// and loader.  Included by one translation unit a type.
#pragma once

#include "nn_gemm.hpp"

namespace tfnn {

template <typename T, typename O, bool AMN, bool BMN>
hipError_t launch_layout(const GemmParams &p, int tile, bool dma, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.tiles_m) * p.tiles_n * p.splits);
  if (dma) {
    if (tile == TILE_256) gemm_tile_kernel<T, O, AMN, BMN, 256, 256, 2, 4, 2, true><<<grid, 512, 0, stream>>>(p);
    else if (tile == TILE_128) gemm_tile_kernel<T, O, AMN, BMN, 128, 128, 2, 2, 2, true><<<grid, 256, 0, stream>>>(p);
    else gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 3, true><<<grid, 256, 0, stream>>>(p);
  } else {
    if (tile == TILE_128) gemm_tile_kernel<T, O, AMN, BMN, 128, 128, 2, 2, 2, false><<<grid, 256, 0, stream>>>(p);
    else gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 2, false><<<grid, 256, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace tfnn
