// One element type's product kernels and their choice by operand layout, tile
// and loader.  Included by one translation unit a type.
#pragma once

#include "nn_gemm.hpp"
#include "nn_wide.hpp"

namespace tfnn {

template <typename T, typename O, bool AMN, bool BMN, int TERMS>
hipError_t launch_tile(const GemmParams &p, int tile, bool dma, hipStream_t stream) {
  const long blocks = static_cast<long>(p.tiles_m) * p.tiles_n * p.splits;
  if (dma) {  // one-sided: plan_product leaves out what does not fit
    const dim3 grid(static_cast<unsigned>(blocks));
    if (tile == TILE_128) gemm_tile_kernel<T, O, AMN, BMN, 128, 128, 2, 2, 2, true, TERMS><<<grid, 256, 0, stream>>>(p);
    else if (tile == TILE_64x128) gemm_tile_kernel<T, O, AMN, BMN, 64, 128, 2, 2, 3, true, TERMS><<<grid, 256, 0, stream>>>(p);
    // Three slabs of LDS leave room for three workgroups on a CU, two for five: 1024 x
    // 2048 x 4096 (512 workgroups) 28.0 us with three, 35.4 with two; 1024 x 4096 x 4096
    // (1024) 55.7 and 48.7.
    else if (grid.x <= 768) gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 3, true, TERMS><<<grid, 256, 0, stream>>>(p);
    else gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 2, true, TERMS><<<grid, 256, 0, stream>>>(p);
  } else {
    gemm_tile_kernel<T, O, AMN, BMN, 64, 64, 2, 2, 2, false, TERMS><<<grid_of(blocks, 256), 256, 0, stream>>>(p);
  }
  return hipGetLastError();
}

template <typename T, typename O, bool AMN, bool BMN>
hipError_t launch_layout(const GemmParams &p, int tile, bool dma, hipStream_t stream) {
  if constexpr (!AMN) {
    if (tile == TILE_ROWS) {
      const dim3 grid(static_cast<unsigned>((p.n + (BMN ? 31 : 15)) / (BMN ? 32 : 16)));
      if ((p.m + 15) / 16 * p.terms <= 1) gemm_rows_kernel<T, O, BMN, 1><<<grid, 64 * rows_waves(BMN, 1), 0, stream>>>(p);
      else if ((p.m + 15) / 16 * p.terms <= 2) gemm_rows_kernel<T, O, BMN, 2><<<grid, 64 * rows_waves(BMN, 2), 0, stream>>>(p);
      else gemm_rows_kernel<T, O, BMN, 4><<<grid, 64 * rows_waves(BMN, 4), 0, stream>>>(p);
      return hipGetLastError();
    }
  }
  if (tile == TILE_256) {  // loads straight into LDS, one term
    gemm_wide_kernel<T, O, AMN, BMN><<<dim3(static_cast<unsigned>(p.tiles_m) * p.tiles_n * p.splits), 512, 0, stream>>>(p);
    return hipGetLastError();
  }
  if constexpr (sizeof(T) == 2) {
    if (p.terms == 2) return launch_tile<T, O, AMN, BMN, 2>(p, tile, dma, stream);
  }
  return launch_tile<T, O, AMN, BMN, 1>(p, tile, dma, stream);
}

template <typename T>
hipError_t launch_pair(const GemmParams &dx, bool bmn, const GemmParams &dw, const ShareParams &sum, hipStream_t stream) {
  const int first = dx.tiles_m * dx.tiles_n * dx.splits, second = dw.tiles_m * dw.tiles_n * dw.splits;
  const dim3 grid(static_cast<unsigned>(first + second + (sum.d + 15) / 16));
  const bool two = dx.terms == 2;
  if (bmn && two) gemm_pair_kernel<T, true, 2><<<grid, 256, 0, stream>>>(dx, dw, sum, first, second);
  else if (bmn) gemm_pair_kernel<T, true, 1><<<grid, 256, 0, stream>>>(dx, dw, sum, first, second);
  else if (two) gemm_pair_kernel<T, false, 2><<<grid, 256, 0, stream>>>(dx, dw, sum, first, second);
  else gemm_pair_kernel<T, false, 1><<<grid, 256, 0, stream>>>(dx, dw, sum, first, second);
  return hipGetLastError();
}

}  // namespace tfnn
