// Layer norm backward: entry points (layernorm_bwd.cuh).
#include "layernorm.cuh"

namespace mb {
int layer_norm_bwd_f32(const LnArgs&, const mb_ln_desc*, bool from_y, bool granules, const Grads&, cudaStream_t);
int layer_norm_bwd_bf16(const LnArgs&, const mb_ln_desc*, bool from_y, bool granules, const Grads&, cudaStream_t);
int layer_norm_bwd_f16(const LnArgs&, const mb_ln_desc*, bool from_y, bool granules, const Grads&, cudaStream_t);
}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_layer_norm_bwd_workspace_bytes(const mb_ln_desc* d) {
  if (!d || d->cols == 0 || d->cols > 0x7fffffffULL || d->rows == 0 || !dtype_bytes(d->dtype)) return 0;
  // which kernel runs also depends on addresses: enough for any
  size_t floats = static_cast<size_t>(column_parts(d)) * 2 * d->cols;
  for (int form = 0; form < 4; ++form) {
    RowPlan q;
    size_t n = 0;
    const bool fits = plan_bwd(d, 2 + form / 2, form % 2, &q);
    if (fits) n = static_cast<size_t>(q.grid / q.cluster) * 2 * d->cols;
    if (n > floats) floats = n;
    if ((!fits || q.cluster > 1) && plan_bwd_long(d, 2 + form / 2, form % 2, &q))
      n = static_cast<size_t>(q.grid / q.cluster) * 2 * d->cols + 2 * d->rows * (1 + static_cast<size_t>(q.cluster) * (q.team / 32));
    if (n > floats) floats = n;
  }
  return floats * sizeof(float);
}

int mb_layer_norm_bwd(const void* dy, const void* kept, int kept_is_output, const void* dsum, const void* weight,
                      const void* bias, const float* mean, const float* rstd, void* dv, void* dx, void* dweight,
                      void* dbias, const mb_ln_desc* d, const mb_dropout_desc* drop, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* who = "mb_layer_norm_bwd";
  if (int rc = check_desc(who, d)) return rc;
  LnArgs p{dy, kept, dsum, weight, bias, dv, dx, const_cast<float*>(mean), const_cast<float*>(rstd),
           d->rows, d->cols, d->ld_a, d->ld_b, d->ld_c, d->param_dtype == MB_F32, aligned(weight, 16) && aligned(bias, 16), d->eps, {}};
  if (int rc = make_drop(who, drop, &p.drop)) return rc;
  cudaStream_t st = as_stream(stream);
  if (!natural_param(d, weight) || !natural_param(d, bias) || !natural_param(d, dweight) || !natural_param(d, dbias))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  if (d->rows == 0) {      // empty sums
    for (void* g : {dweight, dbias})
      if (g && cudaMemsetAsync(g, 0, d->cols * dtype_bytes(d->param_dtype), st) != cudaSuccess)
        return fail(MB_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(cudaGetLastError()));
    return MB_OK;
  }
  if (!dy || !kept || !rstd || !dv || (!kept_is_output && !mean)) return fail(MB_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (dv == dx) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dv and dx must not be the same buffer", who);
  for (const void* o : {static_cast<const void*>(dv), static_cast<const void*>(dx)})
    if (o && ((o == dy && d->ld_a != d->cols) || (o == kept && d->ld_b != d->cols) || (o == dsum && d->ld_c != d->cols)))
      return fail(MB_ERR_INVALID_ARGUMENT, "%s: only dense rows can be overwritten", who);
  if (drop && !dx) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout needs dx", who);
  if (!natural(d, dy) || !natural(d, kept) || !natural(d, dsum) || !natural(d, dv) || !natural(d, dx) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < mb_layer_norm_bwd_workspace_bytes(d))
    return fail(MB_ERR_WORKSPACE, "%s: workspace too small or misaligned", who);
  const Grads g{dweight, dbias, static_cast<float*>(workspace)};
  const bool granules = d->ld_a == d->cols && d->ld_b == d->cols && (!dsum || d->ld_c == d->cols) &&
                        on_granules(d, {{dy, d->cols}, {kept, d->cols}, {dsum, d->cols}, {dv, d->cols}, {dx, d->cols}});
  const bool from_y = kept_is_output != 0;
  if (d->dtype == MB_F32) return layer_norm_bwd_f32(p, d, from_y, granules, g, st);
  if (d->dtype == MB_BF16) return layer_norm_bwd_bf16(p, d, from_y, granules, g, st);
  return layer_norm_bwd_f16(p, d, from_y, granules, g, st);
}

}  // extern "C"
