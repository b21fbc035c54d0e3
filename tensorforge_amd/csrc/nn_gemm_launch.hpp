// One element type's product kernels and their choice by operand layout, tile
// and loader.  Included by one translation unit a type.
#pragma once

#include "nn_gemm.hpp"
#include "nn_wide.hpp"

namespace tfnn {

template <typename T, typename O, bool AMN, bool BMN>
hipError_t launch_layout(const GemmParams &p, int tile, bool dma, hipStream_t stream) {
  if constexpr (!AMN) {
    if (tile == TILE_ROWS) {
      const dim3 grid(static_cast<unsigned>((p.n + (BMN ? 31 : 15)) / (BMN ? 32 : 16)));
      if (p.m <= 16) gemm_rows_kernel<T, O, BMN, 1><<<grid, 64 * rows_waves(BMN, 1), 0, stream>>>(p);
      else if (p.m <= 32) gemm_rows_kernel<T, O, BMN, 2><<<grid, 64 * rows_waves(BMN, 2), 0, stream>>>(p);
      else gemm_rows_kernel<T, O, BMN, 4><<<grid, 64 * rows_waves(BMN, 4), 0, stream>>>(p);
      return hipGetLastError();
    }
  }
  const dim3 grid(static_cast<unsigned>(p.tiles_m) * p.tiles_n * p.splits);
  if (dma) {
    if (tile == TILE_256) gemm_wide_kernel<T, O, AMN, BMN><<<grid, 512, 0, stream>>>(p);
    else if (tile == TILE_128) gemm_tile_kernel<T, O, AMN, BMN, 128, 128, 2, 2, 2, true><<<grid, 256, 0, stream>>>(p);
    else if (grid.x <= 256) gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 8, true><<<grid, 256, 0, stream>>>(p);
    else gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 3, true><<<grid, 256, 0, stream>>>(p);
  } else {
    if (tile == TILE_128) gemm_tile_kernel<T, O, AMN, BMN, 128, 128, 2, 2, 2, false><<<grid, 256, 0, stream>>>(p);
    else gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 2, false><<<grid, 256, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace tfnn
