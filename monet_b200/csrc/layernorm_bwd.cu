// Layer norm backward: kernels and entry point (layernorm.cuh).
#include "layernorm.cuh"

namespace mb {
namespace {

// Backward.  partial[team CTA][0][col] = sum of dy xhat, [1][col] = sum of dy over the CTA's rows.
//
// kRows rows are handled between two barriers: their sums (mean(g), mean(g xhat)) are formed from a
// first reading of the ring, then the rows are read a second time to form dv.  Reading twice costs
// shared-memory loads but no registers, which the column sums need; the parameters lie in shared
// memory for the same reason.  With 64 registers a thread two CTAs share an SM, and one computes
// while the other waits for its barrier.
template <typename T, int K, bool FROM_Y, bool DSUM, bool DROP, bool EDGE, bool CLUSTER>
__global__ void __launch_bounds__(K == 1 ? kMaxTeam : kMaxThreads, K == 1 ? 2 : 1) ln_bwd_rows(LnArgs p, RowPlan q, float* partial) {
  extern __shared__ __align__(128) uint4 ring[];
  if (CLUSTER) cluster_barrier();      // every CTA has started before one writes into another
  __shared__ WarpSums red;
  __shared__ float4 peer[2][8];
  constexpr int kOps = DSUM ? 3 : 2;
  const RowWalk at(q, static_cast<int>(p.cols));
  const int granules = EDGE ? static_cast<int>((at.m + p.cols + 7) >> 3) : static_cast<int>(p.cols >> 3);
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const int j0 = at.rank * q.chunk + at.t;           // the thread's granules: j0 + k * team
  const int rows = static_cast<int>(p.rows), step = static_cast<int>(at.step);

  uint32_t mask[K];
  float2 aw[K][4], ab[K][4];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    mask[k] = column_mask<EDGE>(at, q, granules, static_cast<int>(p.cols), k);
#pragma unroll
    for (int i = 0; i < 4; ++i) aw[k][i] = ab[k][i] = make_float2(0.f, 0.f);
  }

  const int plane = q.chunk;
  const int per_op = plane * kPlanes<T>, per_stage = per_op * kOps;
  uint4* mine = ring + at.group * q.stages * per_stage + at.t;
  float4* const ws = reinterpret_cast<float4*>(ring) + q.stages * q.groups * per_stage + at.t;

  auto fetch = [&](int row, int stage) {
    if (row < rows) {
      const uint32_t dst = sm100::smem_u32(mine) + stage * per_stage * 16;
#pragma unroll
      for (int o = 0; o < kOps; ++o) {
        const T* from = static_cast<const T*>(o == 0 ? p.a : o == 1 ? p.b : p.c);
        const size_t ld = o == 0 ? p.ld_a : o == 1 ? p.ld_b : p.ld_c;
        fetch_row<T, K, EDGE>(from, ld, row, p.rows, p.cols, j0, q.team, mask, dst + o * per_op * 16, plane);
      }
    }
    cp_async_commit();
  };
  // xhat, dy and dy * weight of one granule; zero outside the row
  auto read = [&](const uint4* from, int k, float mean, float rstd, float2 h[4], float2 dy[4], float2 g[4]) {
    const float4* wk = ws + k * q.team;
    ring_read<T>(from + per_op, plane, h);
    if (FROM_Y) {
      get8(wk + 4 * q.chunk, q.chunk, g);
      get8(wk + 2 * q.chunk, q.chunk, dy);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = mul2(add2(h[i], make_float2(-g[i].x, -g[i].y)), dy[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = mul2(add2(h[i], both(-mean)), both(rstd));
    }
    ring_read<T>(from, plane, dy);
    get8(wk, q.chunk, g);
    if (EDGE && mask[k] != 0xffu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!((mask[k] >> (2 * i)) & 1u)) h[i].x = dy[i].x = 0.f;
        if (!((mask[k] >> (2 * i)) & 2u)) h[i].y = dy[i].y = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = mul2(g[i], dy[i]);
  };

  int row = static_cast<int>(at.first);
  for (int s = 0; s < q.stages; ++s) fetch(row + s * step, s);
  // the weight (with FROM_Y also 1 / weight and the bias) of the CTA's columns, granule by granule like the ring
  if (at.group == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!mask[k]) continue;
      const long long col = static_cast<long long>(j0 + k * q.team) * 8 - at.m;
      float v[8];
      param8<T>(p.w, p.w_f32, p.w_vec && !EDGE, col, mask[k], 1.f, v);
      put8(ws + k * q.team, q.chunk, v);
      if (FROM_Y) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 1.f / v[i];
        put8(ws + 2 * q.chunk + k * q.team, q.chunk, v);
        param8<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col, mask[k], 0.f, v);
        put8(ws + 4 * q.chunk + k * q.team, q.chunk, v);
      }
    }
  }
  if (q.groups > 1) __syncthreads();   // the parameters that group 0 put down
  // the teams of a warp shuffle together, so they leave the loop together
  int spare = q.team < 32 ? (at.group - (threadIdx.x & ~31) / q.team) * q.period : 0;
  float mean[kRows], rstd[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int i = row + r * step;
    mean[r] = !FROM_Y && i < rows ? __ldg(p.mean + i) : 0.f;
    rstd[r] = i < rows ? __ldg(p.rstd + i) : 0.f;
  }
  int stage = 0, buf = 0;
  for (; row - spare < rows; row += kRows * step, buf ^= 1) {
    // the next rows' statistics
    float mean_next[kRows], rstd_next[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int i = row + (kRows + r) * step;
      mean_next[r] = !FROM_Y && i < rows ? __ldg(p.mean + i) : 0.f;
      rstd_next[r] = i < rows ? __ldg(p.rstd + i) : 0.f;
    }
    cp_async_wait(q.stages - kRows);
    float s1[kRows], s2[kRows];
    int st = stage;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float2 t1 = make_float2(0.f, 0.f), t2 = t1;
      if (row + r * step < rows) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!mask[k]) continue;
          float2 h[4], dy[4], g[4];
          read(mine + st * per_stage + k * q.team, k, mean[r], rstd[r], h, dy, g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            t1 = add2(t1, g[i]);
            t2 = fma2(g[i], h[i], t2);
            aw[k][i] = fma2(dy[i], h[i], aw[k][i]);
            ab[k][i] = add2(ab[k][i], dy[i]);
          }
        }
      }
      s1[r] = t1.x + t1.y;
      s2[r] = t2.x + t2.y;
      st = st + 1 == q.stages ? 0 : st + 1;
    }
    if (q.team < 32) {
      for (int o = q.team >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          s1[r] += __shfl_xor_sync(0xffffffffu, s1[r], o);
          s2[r] += __shfl_xor_sync(0xffffffffu, s2[r], o);
        }
    } else {
      const float mine4 = warp_sum4(s1[0], s2[0], s1[1], s2[1]);
      float4 f;
      if (q.team == 32) {
        f = make_float4(__shfl_sync(0xffffffffu, mine4, 0), __shfl_sync(0xffffffffu, mine4, 8),
                        __shfl_sync(0xffffffffu, mine4, 16), __shfl_sync(0xffffffffu, mine4, 24));
      } else {
        if ((threadIdx.x & 7) == 0) reinterpret_cast<float*>(red.v[buf])[threadIdx.x >> 3] = mine4;
        team_barrier(at.group, q.team);
        f = gather4(red.v[buf] + at.group * (q.team >> 5), q.team >> 5);
      }
      if (CLUSTER) {
        if (threadIdx.x < q.cluster) put_remote(&peer[buf][at.rank], threadIdx.x, f);
        cluster_barrier();
        f = gather4(peer[buf], q.cluster);
      }
      s1[0] = f.x; s2[0] = f.y; s1[1] = f.z; s2[1] = f.w;
    }
#pragma unroll 1
    for (int r = 0; r < kRows; ++r) {
      const int here = row + r * step;
      if (here < rows) {
        const float mu = r ? mean[1] : mean[0], rs = r ? rstd[1] : rstd[0];
        const float2 c0 = both(rs), c1 = both(-rs * ((r ? s1[1] : s1[0]) * inv_n)), c2 = both(-rs * ((r ? s2[1] : s2[0]) * inv_n));
        const size_t base = static_cast<size_t>(here) * p.cols;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!mask[k]) continue;
          const size_t e = (EDGE ? base & ~size_t(7) : base) + static_cast<size_t>(j0 + k * q.team) * 8;
          const uint32_t keep = DROP ? keep8(__ldg(p.drop.seed), e >> 3, p.drop.stream, p.drop.last) : 0u;
          const uint4* from = mine + stage * per_stage + k * q.team;
          float2 h[4], dy[4], d[4];
          read(from, k, mu, rs, h, dy, d);
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = fma2(d[i], c0, fma2(h[i], c2, c1));     // rstd (g - mean(g) - xhat mean(g xhat))
          if (DSUM) {
            ring_read<T>(from + 2 * per_op, plane, h);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = add2(d[i], h[i]);
          }
          store8_row<EDGE>(static_cast<T*>(p.out) + e, d, mask[k]);
          if (DROP) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              d[i].x = (keep >> (2 * i)) & 1u ? d[i].x * p.drop.scale : 0.f;
              d[i].y = (keep >> (2 * i)) & 2u ? d[i].y * p.drop.scale : 0.f;
            }
            store8_row<EDGE>(static_cast<T*>(p.out2) + e, d, mask[k]);
          }
        }
      }
      fetch(here + q.stages * step, stage);     // into the slots just read for the last time
      stage = stage + 1 == q.stages ? 0 : stage + 1;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
  }
  if (CLUSTER) cluster_barrier();
  if (!partial) return;
  // the CTA's teams hold the same columns: halve their number until one is left
  float2* sums = reinterpret_cast<float2*>(ring);
  for (int n = q.groups; n > 1;) {
    const int low = (n + 1) / 2, pitch = low * q.team;
    __syncthreads();
    if (at.group >= low && at.group < n) {
      float2* to = sums + (at.group - low) * q.team + at.t;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          to[(k * 8 + i) * pitch] = aw[k][i];
          to[(k * 8 + 4 + i) * pitch] = ab[k][i];
        }
    }
    __syncthreads();
    if (at.group < n - low) {
      const float2* from = sums + at.group * q.team + at.t;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          aw[k][i] = add2(aw[k][i], from[(k * 8 + i) * pitch]);
          ab[k][i] = add2(ab[k][i], from[(k * 8 + 4 + i) * pitch]);
        }
    }
    n = low;
  }
  if (at.group == 0) {
    float* to = partial + static_cast<size_t>(blockIdx.x / q.cluster) * 2 * p.cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long col = static_cast<long long>(j0 + k * q.team) * 8 - at.m;
      if (!EDGE) {
        if (mask[k]) {
          store8(to + col, aw[k]);
          store8(to + p.cols + col, ab[k]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((mask[k] >> i) & 1u) {
            to[col + i] = i & 1 ? aw[k][i / 2].y : aw[k][i / 2].x;
            to[p.cols + col + i] = i & 1 ? ab[k][i / 2].y : ab[k][i / 2].x;
          }
      }
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


// Plan of the row kernel; two CTAs per SM where the registers allow.
bool plan_bwd(const mb_ln_desc* d, int ops, bool from_y, RowPlan* q) {
  if (!plan_rows(d->rows, d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, true, from_y, q)) return false;
  size_grid(d->rows, q->per_thread == 1 ? 2 : 1, q);
  return true;
}

struct Grads { void *dw, *db; float* ws; };

template <typename T, int K, bool FROM_Y, bool DSUM, bool DROP, bool EDGE, bool CLUSTER>
int launch_bwd(const LnArgs& p, RowPlan q, const Grads& g, cudaStream_t st) {
  static std::atomic<int> cache[64];
  auto kernel = ln_bwd_rows<T, K, FROM_Y, DSUM, DROP, EDGE, CLUSTER>;
  int regs = 0;
  if (int rc = prepare("layer_norm_bwd", kernel, cache, &regs)) return rc;
  fit_clusters(kernel, &q);
  const bool sums = g.dw || g.db;
  if (int rc = launch_rows("layer_norm_bwd", kernel, q, st, p, q, sums ? g.ws : nullptr)) return rc;
  return sums ? finish<T>(g.ws, q.grid / q.cluster, p.cols, g.dw, g.db, p.w_f32, st) : MB_OK;
}

template <typename T, bool FROM_Y, bool DSUM, bool DROP, bool EDGE>
int pick_bwd(const LnArgs& p, const RowPlan& q, const Grads& g, cudaStream_t st) {
  if (q.cluster > 1) return launch_bwd<T, 2, FROM_Y, DSUM, DROP, EDGE, true>(p, q, g, st);
  if (q.per_thread == 1) return launch_bwd<T, 1, FROM_Y, DSUM, DROP, EDGE, false>(p, q, g, st);
  return launch_bwd<T, 2, FROM_Y, DSUM, DROP, EDGE, false>(p, q, g, st);
}

template <typename T, bool FROM_Y, bool DSUM, bool DROP>
int pick_edge(const LnArgs& p, const RowPlan& q, const Grads& g, cudaStream_t st) {
  return p.cols % 8 ? pick_bwd<T, FROM_Y, DSUM, DROP, true>(p, q, g, st) : pick_bwd<T, FROM_Y, DSUM, DROP, false>(p, q, g, st);
}

template <typename T, bool FROM_Y>
int bwd(const LnArgs& p, const mb_ln_desc* d, bool granules, const Grads& g, cudaStream_t st) {
  RowPlan q;
  // (a dx that equals dv because nothing is dropped is rare enough for the element-wise kernels)
  if (granules && (p.drop.on || !p.out2) && plan_bwd(d, p.c ? 3 : 2, FROM_Y, &q)) {
    if (p.drop.on) return p.c ? pick_edge<T, FROM_Y, true, true>(p, q, g, st) : pick_edge<T, FROM_Y, false, true>(p, q, g, st);
    return p.c ? pick_edge<T, FROM_Y, true, false>(p, q, g, st) : pick_edge<T, FROM_Y, false, false>(p, q, g, st);
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
  for (int form = 0; form < 4; ++form)
    if (plan_bwd(d, 2 + form / 2, form % 2, &q) && q.grid / q.cluster > parts) parts = q.grid / q.cluster;
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
