// Layer norm backward for bfloat16 activations.
#include "layernorm_bwd.cuh"

namespace mb {
int layer_norm_bwd_bf16(const LnArgs& p, const mb_ln_desc* d, bool from_y, bool granules, const Grads& g, cudaStream_t st) {
  return from_y ? bwd<__nv_bfloat16, true>(p, d, granules, g, st) : bwd<__nv_bfloat16, false>(p, d, granules, g, st);
}
}  // namespace mb
