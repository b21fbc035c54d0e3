// The bfloat16 products of the loss over a vocabulary.
#include "nn_xent_gemm.hpp"

namespace tfnn {

hipError_t launch_xent_bf16(const XentParams &p, XentProduct what, bool amn, bool bmn, int tile, bool dma, hipStream_t stream) {
  return launch_xent<bf16>(p, what, amn, bmn, tile, dma, stream);
}

}  // namespace tfnn
