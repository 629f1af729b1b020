// Layer norm forward: kernels and entry point (layernorm.cuh).
#include "layernorm.cuh"

namespace mb {
namespace {

// Row statistics of `n` values: every warp centres on its own mean, and the warps' (count, mean,
// squared deviations) are combined - no difference of large sums is ever formed.
template <bool CLUSTER>
__device__ __forceinline__ void combine_stats(WarpSums& red, float4 (*peer)[8], const RowPlan& q, const RowWalk& at, int buf,
                                              float count, float& mean, float& m2, float n) {
  const int warps = q.team >> 5, w0 = at.group * warps;
  if ((threadIdx.x & 31) == 0) red.v[buf][threadIdx.x >> 5] = make_float4(count, mean, m2, 0.f);
  team_barrier(at.group, q.team);
  float s = 0.f, c = 0.f;
  for (int i = 0; i < warps; ++i) {
    const float4 f = red.v[buf][w0 + i];
    s = fmaf(f.x, f.y, s);
    c += f.x;
  }
  mean = c > 0.f ? s / c : 0.f;
  m2 = 0.f;
  for (int i = 0; i < warps; ++i) {
    const float4 f = red.v[buf][w0 + i];
    const float d = f.y - mean;
    m2 += fmaf(f.x * d, d, f.z);
  }
  if (CLUSTER) {
    if (threadIdx.x < q.cluster) put_remote(&peer[buf][at.rank], threadIdx.x, make_float4(c, mean, m2, 0.f));
    cluster_barrier();
    s = 0.f;
    for (int i = 0; i < q.cluster; ++i) s = fmaf(peer[buf][i].x, peer[buf][i].y, s);
    mean = s / n;
    m2 = 0.f;
    for (int i = 0; i < q.cluster; ++i) {
      const float4 f = peer[buf][i];
      const float d = f.y - mean;
      m2 += fmaf(f.x * d, d, f.z);
    }
  }
}

template <typename T, int K, bool RES, bool EDGE, bool CLUSTER>
__global__ void __launch_bounds__(kMaxTeam) ln_fwd_rows(LnArgs p, RowPlan q) {
  extern __shared__ __align__(128) uint4 ring[];
  if (CLUSTER) cluster_barrier();      // every CTA has started before one writes into another
  __shared__ WarpSums red;
  __shared__ float4 peer[2][8];
  constexpr int kOps = RES ? 2 : 1;
  constexpr bool kKeep = K <= 2 && !CLUSTER;      // parameters of the thread's columns stay in registers
  const RowWalk at(q, static_cast<int>(p.cols));
  const int granules = EDGE ? static_cast<int>((at.m + p.cols + 7) >> 3) : static_cast<int>(p.cols >> 3);
  const size_t total = p.rows * p.cols;
  const float n = static_cast<float>(p.cols), inv_n = 1.f / n;
  const unsigned long long key = p.drop.on ? __ldg(p.drop.seed) : 0;

  long long col[K];
  uint32_t mask[K];
  float wk[kKeep ? K : 1][8], bk[kKeep ? K : 1][8];
  float count = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int jl = at.t + k * q.team, j = at.rank * q.chunk + jl;
    col[k] = static_cast<long long>(j) * 8 - at.m;
    mask[k] = jl < q.chunk && j < granules ? 0xffu : 0u;
    if (EDGE && mask[k]) {
      if (col[k] < 0) mask[k] &= 0xffu << -col[k];
      if (col[k] + 8 > static_cast<long long>(p.cols)) mask[k] &= 0xffu >> (col[k] + 8 - static_cast<long long>(p.cols));
    }
    count += static_cast<float>(__popc(mask[k]));
    if (kKeep) {
      param8<T>(p.w, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 1.f, wk[k]);
      param8<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 0.f, bk[k]);
    }
  }
  const float warp_count = warp_sum(count);

  const int plane = q.chunk;                                   // granules per plane of one stage
  const int per_op = plane * kPlanes<T>, per_stage = per_op * kOps;
  uint4* mine = ring + static_cast<size_t>(at.group) * q.stages * per_stage + at.t;
  const uint32_t mine_u = sm100::smem_u32(mine);

  auto fetch = [&](size_t row, int stage) {
    if (row < p.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        const int j = at.rank * q.chunk + at.t + k * q.team;
        const uint32_t dst = mine_u + (stage * per_stage + k * q.team) * 16;
        if (EDGE) {
          const size_t e = ((row * p.cols) >> 3) * 8 + static_cast<size_t>(j) * 8;
          ring_fetch<T>(dst, plane, static_cast<const T*>(p.a) + e, total - e);
          if (RES) ring_fetch<T>(dst + per_op * 16, plane, static_cast<const T*>(p.b) + e, total - e);
        } else {
          ring_fetch<T>(dst, plane, static_cast<const T*>(p.a) + row * p.ld_a + static_cast<size_t>(j) * 8);
          if (RES) ring_fetch<T>(dst + per_op * 16, plane, static_cast<const T*>(p.b) + row * p.ld_b + static_cast<size_t>(j) * 8);
        }
      }
    }
    cp_async_commit();
  };

  size_t ahead = at.first;
  for (int s = 0; s < q.stages - 1; ++s, ahead += at.step) fetch(ahead, s);
  // the teams of a warp shuffle together, so they leave the loop together
  const size_t lead = q.team < 32 ? at.first - static_cast<size_t>(at.group - (threadIdx.x & ~31) / q.team) * q.period : at.first;
  int stage = 0, fill = q.stages - 1, buf = 0;
  size_t row = at.first;
  for (size_t go = lead; go < p.rows; go += at.step, row += at.step, buf ^= 1) {
    cp_async_wait(q.stages - 2);
    float v[K][8];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (mask[k] && row < p.rows) {
        const uint4* src = mine + stage * per_stage + k * q.team;
        ring_read<T>(src, plane, v[k]);
        if (RES) {
          float r[8];
          ring_read<T>(src + per_op, plane, r);
          uint32_t keep = 0xffu;
          if (p.drop.on) {
            const int j = at.rank * q.chunk + at.t + k * q.team;
            keep = keep8(key, ((row * p.cols) >> 3) + j, p.drop.stream, p.drop.last);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[k][i] = __fadd_rn(r[i], !p.drop.on ? v[k][i] : (keep >> i) & 1u ? __fmul_rn(v[k][i], p.drop.scale) : 0.f);
        }
        if (EDGE && mask[k] != 0xffu) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[k][i] = (mask[k] >> i) & 1u ? v[k][i] : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[k][i];
    }
    fetch(ahead, fill);
    ahead += at.step;
    stage = stage + 1 == q.stages ? 0 : stage + 1;
    fill = fill + 1 == q.stages ? 0 : fill + 1;

    auto deviations = [&](float mean) {
      float d2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = (EDGE ? (mask[k] >> i) & 1u : mask[k]) ? v[k][i] - mean : 0.f;
          d2 = fmaf(d, d, d2);
        }
      return d2;
    };
    float mean, m2;
    if (q.team <= 32) {
      mean = lanes_sum(s, q.team) * inv_n;
      m2 = lanes_sum(deviations(mean), q.team);
    } else {
      mean = warp_count > 0.f ? warp_sum(s) / warp_count : 0.f;
      m2 = warp_sum(deviations(mean));
      combine_stats<CLUSTER>(red, peer, q, at, buf, warp_count, mean, m2, n);
    }
    const float rstd = 1.f / sqrtf(m2 * inv_n + p.eps);
    if (row < p.rows) {
      if (at.t == 0 && at.rank == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
      const size_t base = EDGE ? ((row * p.cols) >> 3) * 8 : row * p.cols;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        const size_t e = base + static_cast<size_t>(at.rank * q.chunk + at.t + k * q.team) * 8;
        if (p.out2) {
          if (EDGE) store8_masked(static_cast<T*>(p.out2) + e, v[k], mask[k]);
          else store8(static_cast<T*>(p.out2) + e, v[k]);
        }
        float w[8], b[8], y[8];
        if (!kKeep) {
          param8<T>(p.w, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 1.f, w);
          param8<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 0.f, b);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf((v[k][i] - mean) * rstd, kKeep ? wk[kKeep ? k : 0][i] : w[i], kKeep ? bk[kKeep ? k : 0][i] : b[i]);
        if (EDGE) store8_masked(static_cast<T*>(p.out) + e, y, mask[k]);
        else store8(static_cast<T*>(p.out) + e, y);
      }
    }
  }
  if (CLUSTER) cluster_barrier();      // no CTA leaves while a peer may still write into it
}

template <typename T>
__global__ void __launch_bounds__(kBlock) ln_fwd_any(LnArgs p) {
  __shared__ float red[kBlock / 32];
  const unsigned long long key = p.drop.on ? __ldg(p.drop.seed) : 0;
  const float inv_n = 1.f / static_cast<float>(p.cols);
  for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.a) + r * p.ld_a;
    const T* res = p.b ? static_cast<const T*>(p.b) + r * p.ld_b : nullptr;
    T* y = static_cast<T*>(p.out) + r * p.cols;
    T* sum = p.out2 ? static_cast<T*>(p.out2) + r * p.cols : nullptr;
    auto value = [&](size_t i) {
      float v = to_f32(x[i]);
      if (p.drop.on) v = kept(p.drop, key, r * p.cols + i) ? __fmul_rn(v, p.drop.scale) : 0.f;
      return res ? __fadd_rn(to_f32(res[i]), v) : v;
    };
    float s = 0.f;
    for (size_t i = threadIdx.x; i < p.cols; i += kBlock) s += value(i);
    const float mean = block_sum(s, red) * inv_n;
    float q = 0.f;
    for (size_t i = threadIdx.x; i < p.cols; i += kBlock) {
      const float c = value(i) - mean;
      q = fmaf(c, c, q);
    }
    const float rstd = 1.f / sqrtf(block_sum(q, red) * inv_n + p.eps);
    for (size_t i = threadIdx.x; i < p.cols; i += kBlock) {
      const float v = value(i);
      const float w = p.w ? param<T>(p.w, p.w_f32, i) : 1.f, b = p.bias ? param<T>(p.bias, p.w_f32, i) : 0.f;
      if (sum) sum[i] = from_f32<T>(v);
      y[i] = from_f32<T>(fmaf((v - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
  }
}


template <typename T, int K, bool RES, bool EDGE, bool CLUSTER>
int launch_fwd(const LnArgs& p, RowPlan q, cudaStream_t st) {
  static std::atomic<int> cache[64];
  auto kernel = ln_fwd_rows<T, K, RES, EDGE, CLUSTER>;
  int regs = 0;
  if (int rc = prepare("layer_norm_fwd", kernel, cache, &regs)) return rc;
  size_grid(p.rows, resident(q.groups * q.team, regs, q.smem), &q);
  fit_clusters(kernel, &q);
  return launch_rows("layer_norm_fwd", kernel, q, st, p, q);
}

template <typename T, bool RES, bool EDGE>
int pick_fwd(const LnArgs& p, const RowPlan& q, cudaStream_t st) {
  if (q.cluster > 1) return q.per_thread <= 4 ? launch_fwd<T, 4, RES, EDGE, true>(p, q, st) : launch_fwd<T, 8, RES, EDGE, true>(p, q, st);
  if (q.per_thread == 1) return launch_fwd<T, 1, RES, EDGE, false>(p, q, st);
  if (q.per_thread == 2) return launch_fwd<T, 2, RES, EDGE, false>(p, q, st);
  return launch_fwd<T, 4, RES, EDGE, false>(p, q, st);
}

template <typename T>
int fwd(const LnArgs& p, bool granules, cudaStream_t st) {
  RowPlan q;
  if (granules && plan_rows(p.rows, p.cols, sizeof(T), p.b ? 2 : 1, false, false, &q)) {
    const bool edge = p.cols % 8 != 0;
    if (p.b) return edge ? pick_fwd<T, true, true>(p, q, st) : pick_fwd<T, true, false>(p, q, st);
    return edge ? pick_fwd<T, false, true>(p, q, st) : pick_fwd<T, false, false>(p, q, st);
  }
  ln_fwd_any<T><<<grid_for(p.rows, 1, 8), kBlock, 0, st>>>(p);
  return after_launch("layer_norm_fwd");
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" {

int mb_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* y,
                      void* sum, float* mean, float* rstd, const mb_ln_desc* d, const mb_dropout_desc* drop,
                      void* stream) {
  const char* who = "mb_layer_norm_fwd";
  if (int rc = check_desc(who, d)) return rc;
  LnArgs p{x, residual, nullptr, weight, bias, y, sum, mean, rstd, d->rows, d->cols, d->ld_a, d->ld_b, 0, d->param_dtype == MB_F32, aligned(weight, 16) && aligned(bias, 16), d->eps, {}};
  if (int rc = make_drop(who, drop, &p.drop)) return rc;
  if (d->rows == 0) return MB_OK;
  if (!x || !y || !mean || !rstd) return fail(MB_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (drop && !residual) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout needs a residual", who);
  if (!natural(d, x) || !natural(d, residual) || !natural(d, y) || !natural(d, sum) || !natural_param(d, weight) ||
      !natural_param(d, bias) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  cudaStream_t st = as_stream(stream);
  const bool granules = on_granules(d, {{x, d->ld_a}, {residual, d->ld_b}, {y, d->cols}, {sum, d->cols}});
  if (d->dtype == MB_F32) return fwd<float>(p, granules, st);
  if (d->dtype == MB_BF16) return fwd<__nv_bfloat16>(p, granules, st);
  return fwd<__half>(p, granules, st);
}

}  // extern "C"
