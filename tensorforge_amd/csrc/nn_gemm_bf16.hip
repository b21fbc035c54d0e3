// The bfloat16 products.
#include "nn_gemm_launch.hpp"

namespace tfnn {

hipError_t launch_gemm_bf16(const GemmParams &p, bool amn, bool bmn, int tile, bool dma, hipStream_t stream) {
  if (amn) return launch_layout<bf16, bf16, true, true>(p, tile, dma, stream);  // weight gradients: both operands by columns of k
  if (bmn) return launch_layout<bf16, bf16, false, true>(p, tile, dma, stream);
  return launch_layout<bf16, bf16, false, false>(p, tile, dma, stream);
}

hipError_t launch_gemm_pair_bf16(const GemmParams &dx, bool bmn, const GemmParams &dw, const ShareParams &sum, hipStream_t stream) {
  return launch_pair<bf16>(dx, bmn, dw, sum, stream);
}

}  // namespace tfnn
