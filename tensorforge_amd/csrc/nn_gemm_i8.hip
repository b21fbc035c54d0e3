// The products of 8-bit integers: k contiguous on both sides, 16-bit results.
#include "nn_gemm_launch.hpp"

namespace tfnn {

hipError_t launch_gemm_i8(const GemmParams &p, int out_type, int tile, bool dma, hipStream_t stream) {
  if (out_type == TYPE_BF16) return launch_layout<i8, bf16, false, false>(p, tile, dma, stream);
  return launch_layout<i8, f16, false, false>(p, tile, dma, stream);
}

}  // namespace tfnn
