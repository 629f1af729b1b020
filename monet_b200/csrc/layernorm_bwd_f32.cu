// Layer norm backward for fp32 activations.
#include "layernorm_bwd.cuh"

namespace mb {
int layer_norm_bwd_f32(const LnArgs& p, const mb_ln_desc* d, bool from_y, bool granules, const Grads& g, cudaStream_t st) {
  return from_y ? bwd<float, true>(p, d, granules, g, st) : bwd<float, false>(p, d, granules, g, st);
}
}  // namespace mb
