// Layer norm backward: kernels and entry point (layernorm.cuh).
#include "layernorm.cuh"

namespace mb {
namespace {

// Backward.  partial[blockIdx.x][0][col] = sum of dy xhat, [1][col] = sum of dy over this CTA's rows.
template <typename T, int K, bool FROM_Y, bool DSUM, bool EDGE, bool CLUSTER>
__global__ void __launch_bounds__(kMaxThreads) ln_bwd_rows(LnArgs p, RowPlan q, float* partial) {
  extern __shared__ __align__(128) uint4 ring[];
  if (CLUSTER) cluster_barrier();      // every CTA has started before one writes into another
  __shared__ WarpSums red;
  __shared__ float4 peer[2][8];
  constexpr int kOps = DSUM ? 3 : 2;
  const RowWalk at(q, static_cast<int>(p.cols));
  const int granules = EDGE ? static_cast<int>((at.m + p.cols + 7) >> 3) : static_cast<int>(p.cols >> 3);
  const size_t total = p.rows * p.cols;
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const unsigned long long key = p.drop.on ? __ldg(p.drop.seed) : 0;

  long long col[K];
  uint32_t mask[K];
  float w[K][8], iw[FROM_Y ? K : 1][8], b[FROM_Y ? K : 1][8];
  float aw[K][8], ab[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int jl = at.t + k * q.team, j = at.rank * q.chunk + jl;
    col[k] = static_cast<long long>(j) * 8 - at.m;
    mask[k] = jl < q.chunk && j < granules ? 0xffu : 0u;
    if (EDGE && mask[k]) {
      if (col[k] < 0) mask[k] &= 0xffu << -col[k];
      if (col[k] + 8 > static_cast<long long>(p.cols)) mask[k] &= 0xffu >> (col[k] + 8 - static_cast<long long>(p.cols));
    }
    param8<T>(p.w, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 1.f, w[k]);
    if (FROM_Y) {
      param8<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col[k], mask[k], 0.f, b[FROM_Y ? k : 0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) iw[FROM_Y ? k : 0][i] = 1.f / w[k][i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) aw[k][i] = ab[k][i] = 0.f;
  }

  const int plane = q.chunk;
  const int per_op = plane * kPlanes<T>, per_stage = per_op * kOps;
  uint4* mine = ring + static_cast<size_t>(at.group) * q.stages * per_stage + at.t;
  const uint32_t mine_u = sm100::smem_u32(mine);
  const T* const src[3] = {static_cast<const T*>(p.a), static_cast<const T*>(p.b), static_cast<const T*>(p.c)};
  const size_t ld[3] = {p.ld_a, p.ld_b, p.ld_c};

  auto fetch = [&](size_t row, int stage) {
    if (row < p.rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        const int j = at.rank * q.chunk + at.t + k * q.team;
        const uint32_t dst = mine_u + (stage * per_stage + k * q.team) * 16;
#pragma unroll
        for (int o = 0; o < kOps; ++o) {
          if (EDGE) {
            const size_t e = ((row * p.cols) >> 3) * 8 + static_cast<size_t>(j) * 8;
            ring_fetch<T>(dst + o * per_op * 16, plane, src[o] + e, total - e);
          } else {
            ring_fetch<T>(dst + o * per_op * 16, plane, src[o] + row * ld[o] + static_cast<size_t>(j) * 8);
          }
        }
      }
    }
    cp_async_commit();
  };

  size_t ahead = at.first;
  for (int s = 0; s < q.stages - 1; ++s, ahead += at.step) fetch(ahead, s);
  const size_t lead = q.team < 32 ? at.first - static_cast<size_t>(at.group - (threadIdx.x & ~31) / q.team) * q.period : at.first;
  int stage = 0, fill = q.stages - 1, buf = 0;
  size_t row = at.first;
  float mean = 0.f, rstd = 0.f;
  if (row < p.rows) {
    if (!FROM_Y) mean = __ldg(p.mean + row);
    rstd = __ldg(p.rstd + row);
  }
  for (size_t go = lead; go < p.rows; go += at.step, row += at.step, buf ^= 1) {
    float mean_next = 0.f, rstd_next = 0.f;
    if (row + at.step < p.rows) {
      if (!FROM_Y) mean_next = __ldg(p.mean + row + at.step);
      rstd_next = __ldg(p.rstd + row + at.step);
    }
    cp_async_wait(q.stages - 2);
    float h[K][8], dy[K][8], ds[DSUM ? K : 1][8];
    float s1 = 0.f, s2 = 0.f;
    const bool live = row < p.rows;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (mask[k] && live) {
        const uint4* from = mine + stage * per_stage + k * q.team;
        ring_read<T>(from, plane, dy[k]);
        ring_read<T>(from + per_op, plane, h[k]);
        if (DSUM) ring_read<T>(from + 2 * per_op, plane, ds[DSUM ? k : 0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[k][i] = FROM_Y ? (h[k][i] - b[FROM_Y ? k : 0][i]) * iw[FROM_Y ? k : 0][i] : (h[k][i] - mean) * rstd;
        if (EDGE && mask[k] != 0xffu) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            h[k][i] = (mask[k] >> i) & 1u ? h[k][i] : 0.f;
            dy[k][i] = (mask[k] >> i) & 1u ? dy[k][i] : 0.f;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[k][i] = dy[k][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float g = dy[k][i] * w[k][i];
        s1 += g;
        s2 = fmaf(g, h[k][i], s2);
        aw[k][i] = fmaf(dy[k][i], h[k][i], aw[k][i]);
        ab[k][i] += dy[k][i];
      }
    }
    fetch(ahead, fill);
    ahead += at.step;
    stage = stage + 1 == q.stages ? 0 : stage + 1;
    fill = fill + 1 == q.stages ? 0 : fill + 1;

    if (q.team <= 32) {
      s1 = lanes_sum(s1, q.team);
      s2 = lanes_sum(s2, q.team);
    } else {
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      const int warps = q.team >> 5, w0 = at.group * warps;
      if ((threadIdx.x & 31) == 0) red.v[buf][threadIdx.x >> 5] = make_float4(s1, s2, 0.f, 0.f);
      team_barrier(at.group, q.team);
      s1 = s2 = 0.f;
      for (int i = 0; i < warps; ++i) {
        const float4 f = red.v[buf][w0 + i];
        s1 += f.x;
        s2 += f.y;
      }
      if (CLUSTER) {
        if (threadIdx.x < q.cluster) put_remote(&peer[buf][at.rank], threadIdx.x, make_float4(s1, s2, 0.f, 0.f));
        cluster_barrier();
        s1 = s2 = 0.f;
        for (int i = 0; i < q.cluster; ++i) {
          s1 += peer[buf][i].x;
          s2 += peer[buf][i].y;
        }
      }
    }
    s1 *= inv_n;
    s2 *= inv_n;
    if (live) {
      const size_t base = EDGE ? ((row * p.cols) >> 3) * 8 : row * p.cols;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        const int j = at.rank * q.chunk + at.t + k * q.team;
        const size_t e = base + static_cast<size_t>(j) * 8;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          d[i] = (dy[k][i] * w[k][i] - s1 - h[k][i] * s2) * rstd;
          if (DSUM) d[i] += ds[DSUM ? k : 0][i];
        }
        if (EDGE) store8_masked(static_cast<T*>(p.out) + e, d, mask[k]);
        else store8(static_cast<T*>(p.out) + e, d);
        if (p.out2) {
          if (p.drop.on) {
            const uint32_t keep = keep8(key, ((row * p.cols) >> 3) + j, p.drop.stream, p.drop.last);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = (keep >> i) & 1u ? d[i] * p.drop.scale : 0.f;
          }
          if (EDGE) store8_masked(static_cast<T*>(p.out2) + e, d, mask[k]);
          else store8(static_cast<T*>(p.out2) + e, d);
        }
      }
    }
    mean = mean_next;
    rstd = rstd_next;
  }
  if (CLUSTER) cluster_barrier();
  if (!partial) return;
  // the CTA's teams hold the same columns: halve their number until one is left
  float* sums = reinterpret_cast<float*>(ring);
  for (int n = q.groups; n > 1;) {
    const int low = (n + 1) / 2;
    __syncthreads();
    if (at.group >= low && at.group < n) {
      float* to = sums + (static_cast<size_t>(at.group - low) * q.team + at.t);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          to[(k * 16 + i) * (low * q.team)] = aw[k][i];
          to[(k * 16 + 8 + i) * (low * q.team)] = ab[k][i];
        }
    }
    __syncthreads();
    if (at.group < n - low) {
      const float* from = sums + (static_cast<size_t>(at.group) * q.team + at.t);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          aw[k][i] += from[(k * 16 + i) * (low * q.team)];
          ab[k][i] += from[(k * 16 + 8 + i) * (low * q.team)];
        }
    }
    n = low;
  }
  if (at.group == 0) {
    float* to = partial + static_cast<size_t>(blockIdx.x / q.cluster) * 2 * p.cols;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((mask[k] >> i) & 1u) {
          to[col[k] + i] = aw[k][i];
          to[p.cols + col[k] + i] = ab[k][i];
        }
  }
}

template <typename T, bool FROM_Y>
__device__ __forceinline__ float xhat_any(const LnArgs& p, const T* kept_row, size_t i, float w, float b, float mean, float rstd) {
  const float v = to_f32(kept_row[i]);
  return FROM_Y ? (v - b) / w : (v - mean) * rstd;
}

template <typename T, bool FROM_Y>
__global__ void __launch_bounds__(kBlock) ln_bwd_any(LnArgs p) {
  __shared__ float red[kBlock / 32];
  const unsigned long long key = p.drop.on ? __ldg(p.drop.seed) : 0;
  const float inv_n = 1.f / static_cast<float>(p.cols);
  for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* dy = static_cast<const T*>(p.a) + r * p.ld_a;
    const T* kp = static_cast<const T*>(p.b) + r * p.ld_b;
    const T* ds = p.c ? static_cast<const T*>(p.c) + r * p.ld_c : nullptr;
    T* dv = static_cast<T*>(p.out) + r * p.cols;
    T* dx = p.out2 ? static_cast<T*>(p.out2) + r * p.cols : nullptr;
    const float mean = FROM_Y ? 0.f : p.mean[r], rstd = p.rstd[r];
    auto get = [&](size_t i, float& g, float& h) {
      const float w = p.w ? param<T>(p.w, p.w_f32, i) : 1.f;
      const float b = FROM_Y && p.bias ? param<T>(p.bias, p.w_f32, i) : 0.f;
      g = to_f32(dy[i]) * w;
      h = xhat_any<T, FROM_Y>(p, kp, i, w, b, mean, rstd);
    };
    float s1 = 0.f, s2 = 0.f, g, h;
    for (size_t i = threadIdx.x; i < p.cols; i += kBlock) {
      get(i, g, h);
      s1 += g;
      s2 = fmaf(g, h, s2);
    }
    s1 = block_sum(s1, red) * inv_n;
    s2 = block_sum(s2, red) * inv_n;
    for (size_t i = threadIdx.x; i < p.cols; i += kBlock) {
      get(i, g, h);
      float d = (g - s1 - h * s2) * rstd;
      if (ds) d += to_f32(ds[i]);
      if (dx) dx[i] = from_f32<T>(!p.drop.on ? d : kept(p.drop, key, r * p.cols + i) ? d * p.drop.scale : 0.f);
      dv[i] = from_f32<T>(d);
    }
  }
}

// Partial sums over rows: CTA (x, y) covers 32 columns and every gridDim.y-th group of 8 rows.
// partial[y][0][col] = sum dy xhat, partial[y][1][col] = sum dy.
template <typename T, bool FROM_Y>
__global__ void __launch_bounds__(256) ln_bwd_columns_any(LnArgs p, float* partial) {
  __shared__ float sw[8][33], sb[8][33];
  const size_t col = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.x;
  float aw = 0.f, ab = 0.f;
  if (col < p.cols) {
    const float w = p.w ? param<T>(p.w, p.w_f32, col) : 1.f;
    const float b = FROM_Y && p.bias ? param<T>(p.bias, p.w_f32, col) : 0.f;
    for (size_t r = static_cast<size_t>(blockIdx.y) * 8 + threadIdx.y; r < p.rows; r += static_cast<size_t>(gridDim.y) * 8) {
      const float g = to_f32(static_cast<const T*>(p.a)[r * p.ld_a + col]);
      aw = fmaf(g, xhat_any<T, FROM_Y>(p, static_cast<const T*>(p.b) + r * p.ld_b, col, w, b, FROM_Y ? 0.f : p.mean[r], p.rstd[r]), aw);
      ab += g;
    }
  }
  sw[threadIdx.y][threadIdx.x] = aw;
  sb[threadIdx.y][threadIdx.x] = ab;
  __syncthreads();
  if (threadIdx.y == 0 && col < p.cols) {
    for (int k = 1; k < 8; ++k) {
      aw += sw[k][threadIdx.x];
      ab += sb[k][threadIdx.x];
    }
    partial[(static_cast<size_t>(blockIdx.y) * 2) * p.cols + col] = aw;
    partial[(static_cast<size_t>(blockIdx.y) * 2 + 1) * p.cols + col] = ab;
  }
}

// dw, db from `parts` partials per column: 32 columns a CTA, 32 threads a column.
template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_finish(const float* partial, int parts, size_t cols, void* dw, void* db, bool w_f32) {
  __shared__ float sw[32][33], sb[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");      // launched while the partials are still being written
  const size_t col = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.x;
  float aw = 0.f, ab = 0.f;
  if (col < cols)
#pragma unroll 4
    for (int k = threadIdx.y; k < parts; k += 32) {
      aw += partial[(static_cast<size_t>(k) * 2) * cols + col];
      ab += partial[(static_cast<size_t>(k) * 2 + 1) * cols + col];
    }
  sw[threadIdx.y][threadIdx.x] = aw;
  sb[threadIdx.y][threadIdx.x] = ab;
  __syncthreads();
  // warp y adds the 32 values of column y of the tile
  aw = warp_sum(sw[threadIdx.x][threadIdx.y]);
  ab = warp_sum(sb[threadIdx.x][threadIdx.y]);
  const size_t mine = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.y;
  if (threadIdx.x == 0 && mine < cols) {
    if (dw) put_param<T>(dw, w_f32, mine, aw);
    if (db) put_param<T>(db, w_f32, mine, ab);
  }
}

template <typename T>
int finish(const float* partial, int parts, size_t cols, void* dw, void* db, bool w_f32, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((cols + 31) / 32));
  cfg.blockDim = dim3(32, 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, ln_bwd_finish<T>, partial, parts, cols, dw, db, w_f32);
  return after_launch("layer_norm_bwd_finish");
}

int column_parts(const mb_ln_desc* d) {
  const size_t tiles = (d->cols + 31) / 32, groups = (d->rows + 7) / 8;
  size_t want = (static_cast<size_t>(num_sms()) * 8 + tiles - 1) / tiles;
  if (want > groups) want = groups;
  return static_cast<int>(want < 1 ? 1 : want > 1024 ? 1024 : want);
}


// Plan of the row kernel: one CTA per SM, so that there are few partials and much shared memory.
bool plan_bwd(const mb_ln_desc* d, int ops, RowPlan* q) {
  if (!plan_rows(d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, true, kMaxThreads, q)) return false;
  size_grid(d->rows, 1, q);
  return true;
}

struct Grads { void *dw, *db; float* ws; };

template <typename T, int K, bool FROM_Y, bool DSUM, bool EDGE, bool CLUSTER>
int launch_bwd(const LnArgs& p, RowPlan q, const Grads& g, cudaStream_t st) {
  static std::atomic<int> cache[64];
  auto kernel = ln_bwd_rows<T, K, FROM_Y, DSUM, EDGE, CLUSTER>;
  int regs = 0;
  if (int rc = prepare("layer_norm_bwd", kernel, cache, &regs)) return rc;
  fit_clusters(kernel, &q);
  const bool sums = g.dw || g.db;
  if (int rc = launch_rows("layer_norm_bwd", kernel, q, st, p, q, sums ? g.ws : nullptr)) return rc;
  return sums ? finish<T>(g.ws, q.grid / q.cluster, p.cols, g.dw, g.db, p.w_f32, st) : MB_OK;
}

template <typename T, bool FROM_Y, bool DSUM, bool EDGE>
int pick_bwd(const LnArgs& p, const RowPlan& q, const Grads& g, cudaStream_t st) {
  if (q.cluster > 1) return launch_bwd<T, 2, FROM_Y, DSUM, EDGE, true>(p, q, g, st);
  if (q.per_thread == 1) return launch_bwd<T, 1, FROM_Y, DSUM, EDGE, false>(p, q, g, st);
  return launch_bwd<T, 2, FROM_Y, DSUM, EDGE, false>(p, q, g, st);
}

template <typename T, bool FROM_Y>
int bwd(const LnArgs& p, const mb_ln_desc* d, bool granules, const Grads& g, cudaStream_t st) {
  RowPlan q;
  if (granules && plan_bwd(d, p.c ? 3 : 2, &q)) {
    const bool edge = p.cols % 8 != 0;
    if (p.c) return edge ? pick_bwd<T, FROM_Y, true, true>(p, q, g, st) : pick_bwd<T, FROM_Y, true, false>(p, q, g, st);
    return edge ? pick_bwd<T, FROM_Y, false, true>(p, q, g, st) : pick_bwd<T, FROM_Y, false, false>(p, q, g, st);
  }
  if (g.dw || g.db) {      // before the outputs, which may lie over the inputs
    const int parts = column_parts(d);
    ln_bwd_columns_any<T, FROM_Y><<<dim3(static_cast<unsigned>((p.cols + 31) / 32), parts), dim3(32, 8), 0, st>>>(p, g.ws);
    if (int rc = after_launch("layer_norm_bwd_columns")) return rc;
    if (int rc = finish<T>(g.ws, parts, p.cols, g.dw, g.db, p.w_f32, st)) return rc;
  }
  ln_bwd_any<T, FROM_Y><<<grid_for(p.rows, 1, 8), kBlock, 0, st>>>(p);
  return after_launch("layer_norm_bwd");
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_layer_norm_workspace_bytes(const mb_ln_desc* d) {
  if (!d || d->cols == 0 || d->rows == 0 || !dtype_bytes(d->dtype)) return 0;
  // which kernel runs also depends on addresses: enough for any
  int parts = column_parts(d);
  RowPlan q;
  for (int ops = 2; ops <= 3; ++ops)
    if (plan_bwd(d, ops, &q) && q.grid / q.cluster > parts) parts = q.grid / q.cluster;
  return static_cast<size_t>(parts) * 2 * d->cols * sizeof(float);
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
  if (drop && !dx) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout needs dx", who);
  if (!natural(d, dy) || !natural(d, kept) || !natural(d, dsum) || !natural(d, dv) || !natural(d, dx) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  if ((dweight || dbias) && (!workspace || !aligned(workspace, 16) || workspace_bytes < mb_layer_norm_workspace_bytes(d)))
    return fail(MB_ERR_WORKSPACE, "%s: workspace too small or misaligned", who);
  const Grads g{dweight, dbias, static_cast<float*>(workspace)};
  const bool granules = on_granules(d, {{dy, d->ld_a}, {kept, d->ld_b}, {dsum, d->ld_c}, {dv, d->cols}, {dx, d->cols}});
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return kept_is_output ? bwd<T, true>(p, d, granules, g, st) : bwd<T, false>(p, d, granules, g, st);
  };
  if (d->dtype == MB_F32) return go(0.f);
  if (d->dtype == MB_BF16) return go(__nv_bfloat16{});
  return go(__half{});
}

}  // extern "C"
