// The 16-bit products that keep their pre-activation in 8 bits.
#include "nn_gemm_kept.hpp"

namespace tfnn {

hipError_t launch_gemm_kept(const KeptGemmParams &p, int type, bool bmn, int tile, hipStream_t stream) {
  if (type == TYPE_BF16) return bmn ? launch_kept_as<bf16, true>(p, tile, stream) : launch_kept_as<bf16, false>(p, tile, stream);
  return bmn ? launch_kept_as<f16, true>(p, tile, stream) : launch_kept_as<f16, false>(p, tile, stream);
}

}  // namespace tfnn
