// Layer norm backward for float16 activations.
#include "layernorm_bwd.cuh"

namespace mb {
int layer_norm_bwd_f16(const LnArgs& p, const mb_ln_desc* d, bool from_y, bool granules, const Grads& g, cudaStream_t st) {
  return from_y ? bwd<__half, true>(p, d, granules, g, st) : bwd<__half, false>(p, d, granules, g, st);
}
}  // namespace mb
