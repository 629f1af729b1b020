// Layer norm forward: kernels and entry point (layernorm.cuh).
#include "layernorm.cuh"

namespace mb {
namespace {

// ---- rows in registers -----------------------------------------------------------------------
// Statistics: every thread centres on its own mean, and (sum, squared deviations) are merged pairwise
// over the lanes, then over the warps and the CTAs of a cluster: no difference of large sums is ever
// formed, and one pass over the lanes does.  (Where a warp's lanes hold different numbers of values it
// centres on the warp's mean instead.)
template <int P>
__device__ __forceinline__ void normalise(float2 (&y)[P], float mean, float rstd, const float2 (&w)[P], const float2 (&b)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) y[i] = fma2(mul2(add2(y[i], both(-mean)), both(rstd)), w[i], b[i]);
}
template <int P>
__device__ __forceinline__ float2 deviations(const float2 (&v)[P], float mean, uint32_t mask, bool whole, float2 sum) {
  float2 d[P];
#pragma unroll
  for (int i = 0; i < P; ++i) d[i] = add2(v[i], both(-mean));
  if (!whole) zero_outside(d, mask);
#pragma unroll
  for (int i = 0; i < P; ++i) sum = fma2(d[i], d[i], sum);
  return sum;
}

template <typename T, int K, int R, bool RES, bool EDGE, bool CLUSTER>
__global__ void __launch_bounds__(K * kE<T> >= 32 ? kMaxThreadsWide : kMaxThreads) ln_fwd_rows(LnArgs p, RowPlan q) {
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ float2 red[2][kMaxThreads / 32][R];      // double-buffered by row: one barrier a row
  __shared__ float counts[kMaxThreads / 32];
  __shared__ float peer[2][kMaxCluster][3];
  if (CLUSTER) cluster_barrier();      // every CTA has started before one writes into another
  constexpr int E = kE<T>, P = kPairs<T>, kOps = RES ? 2 : 1, kSlots = K * kOps;
  constexpr int kParam = kParamUnits<T> * kUnit;
  constexpr uint32_t kAll = (1u << E) - 1;
  constexpr bool kInRegs = K == 1;
  const RowWalk at(q, p.cols, E);
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const int rows = static_cast<int>(p.rows), step = at.step, lane = threadIdx.x & 31, warps = q.team >> 5;
  const unsigned long long key = RES && p.drop.on ? __ldg(p.drop.seed) : 0;
  const uint32_t stride = (blockDim.x >> 5) * (kSlots * kUnit);
  const uint32_t slots = sm100::smem_u32(ring) + (threadIdx.x >> 5) * (kSlots * kUnit) + lane * 16;
  const uint32_t params = sm100::smem_u32(ring) + q.stages * stride + (at.t >> 5) * (K * 2 * kParam) + (at.t & 31) * 16;
  const uint32_t kstep = q.team * 16;

  uint32_t mask[K];
  float count = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    mask[k] = column_mask<T, EDGE>(at, q, at.t + k * q.team, p.cols);
    count += static_cast<float>(__popc(mask[k]));
  }
  const int j0 = at.rank * q.chunk + at.t;           // the thread's granules: j0 + k * team
  const bool even = __all_sync(0xffffffffu, count == static_cast<float>(K * E));      // the warp's lanes have equal counts
  if (!kInRegs) {
    count = warp_sum(count);
    if (lane == 0) counts[threadIdx.x >> 5] = count;
  }

  size_t out = row_offset<T, EDGE>(at.first, p.cols, p.cols, j0) * sizeof(T);
  const size_t out_step = static_cast<size_t>(step) * p.cols * sizeof(T);
  // inputs may have gaps between their rows
  size_t in_a = row_offset<T, EDGE>(at.first, p.ld_a, p.cols, j0) * sizeof(T), in_b = RES ? row_offset<T, EDGE>(at.first, p.ld_b, p.cols, j0) * sizeof(T) : 0;
  int next = at.first;
  const int ends = last_rows<T, EDGE>(rows, p.cols);
  auto fetch = [&](uint32_t stage) {
    if (next < rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        ring_copy(stage + (k * kOps) * kUnit, p.a, in_a + k * kstep, EDGE && next >= ends, p.rows * p.cols * sizeof(T));
        if (RES) ring_copy(stage + (k * kOps + 1) * kUnit, p.b, in_b + k * kstep, EDGE && next >= ends, p.rows * p.cols * sizeof(T));
      }
      in_a += static_cast<size_t>(step) * p.ld_a * sizeof(T);
      if (RES) in_b += static_cast<size_t>(step) * p.ld_b * sizeof(T);
    }
    next += step;
  };
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (!mask[k])
      for (int s = 0; s < q.stages; ++s)
#pragma unroll
        for (int o = 0; o < kOps; ++o) smem_put(slots + s * stride + (k * kOps + o) * kUnit, make_uint4(0, 0, 0, 0));
  for (int s = 0; s < q.stages; s += R) {
#pragma unroll
    for (int r = 0; r < R; ++r) fetch(slots + (s + r) * stride);
    cp_async_commit();
  }

  float2 wr[P], br[P];
  if (kInRegs || at.group == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long col = static_cast<long long>(j0 + k * q.team) * E - at.m;
      load_params<T>(p.w, p.w_f32, p.w_vec && !EDGE, col, mask[k], 1.f, wr);
      load_params<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col, mask[k], 0.f, br);
      if (!kInRegs) {
        param_put<T>(params + (2 * k) * kParam, wr);
        param_put<T>(params + (2 * k + 1) * kParam, br);
      }
    }
  }
  if (!kInRegs) __syncthreads();       // the parameters that group 0 put down, and the counts
  // Combining the warps' statistics, a lane looks after the warp of its number.  Warps with equal counts,
  // a power of two of them, merge like lanes.
  const bool alike = !EDGE && q.chunk == K * q.team && (warps & (warps - 1)) == 0;
  const float part_count = q.team > 32 && lane < warps ? counts[at.group * warps + lane] : 0.f;
  const float part_inv = part_count > 0.f ? 1.f / part_count : 0.f, part_total = q.team > 32 ? warp_sum(part_count) : 0.f;
  const float part_each = part_total > 0.f ? 1.f / part_total : 0.f;

  uint32_t stage = slots;
  int row = at.first, buf = 0;
  const int spare = at.spare(q);
  for (; row - spare < rows; row += R * step, buf ^= 1) {
    cp_async_wait(q.stages / R - 1);
    float2 v[R][K][P];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 sum = both(0.f);
      Signs<T> gone[K];
      if (RES && p.drop.on) {
        size_t g[K];
#pragma unroll
        for (int k = 0; k < K; ++k) g[k] = (out + r * out_step + k * kstep) / 16;
        granule_signs<T, K>(p.drop, key, g, gone);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        ring_get<T>(stage + r * stride + (k * kOps) * kUnit, v[r][k]);
        if (RES) {
          float2 res[P];
          if (p.drop.on) apply_signs<T>(v[r][k], gone[k], p.drop.scale);
          ring_get<T>(stage + r * stride + (k * kOps + 1) * kUnit, res);
#pragma unroll
          for (int i = 0; i < P; ++i) v[r][k][i] = add2(res[i], v[r][k][i]);
        }
        if (EDGE && mask[k] != kAll) zero_outside(v[r][k], mask[k]);
#pragma unroll
        for (int i = 0; i < P; ++i) sum = add2(sum, v[r][k][i]);
      }
      s[r] = sum.x + sum.y;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) fetch(stage + r * stride);       // the slots are free again
    cp_async_commit();
    stage += R * stride;
    if (stage >= slots + q.stages * stride) stage = slots;

    float mean[R], m2[R];
    auto spread = [&](const float (&centre)[R], bool whole) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 sum = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) sum = deviations(v[r][k], centre[r], mask[k], whole || mask[k] == kAll, sum);
        m2[r] = sum.x + sum.y;
      }
    };
    if (even && !kInRegs) {
#pragma unroll
      for (int r = 0; r < R; ++r) mean[r] = s[r] * (1.f / (K * E));
      spread(mean, true);
      merge_lanes(s, m2, q.team < 32 ? q.team : 32, static_cast<float>(K * E));
    } else {
      const float each = kInRegs ? inv_n : count > 0.f ? 1.f / count : 0.f;
      lanes_sums(s, kInRegs ? q.team : 32);
#pragma unroll
      for (int r = 0; r < R; ++r) mean[r] = s[r] * each;
      spread(mean, false);
      lanes_sums(m2, kInRegs ? q.team : 32);
    }
    if (q.team > 32) {
      if (lane == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) red[buf][threadIdx.x >> 5][r] = make_float2(s[r], m2[r]);
      team_barrier(at.group, q.team);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2(*f)[R] = red[buf] + at.group * warps;
        float total, sq, n = part_total;
        if (alike) {
          float ts[1] = {f[lane & (warps - 1)][r].x}, tq[1] = {f[lane & (warps - 1)][r].y};
          merge_lanes(ts, tq, warps, static_cast<float>(32 * K * E));
          total = ts[0];
          sq = tq[0];
        } else {
          const float2 mine = lane < warps ? f[lane][r] : make_float2(0.f, 0.f);
          total = warp_sum(mine.x);
          const float d = mine.x * part_inv - total * part_each;
          sq = warp_sum(part_inv > 0.f ? fmaf(part_count * d, d, mine.y) : 0.f);
        }
        if (CLUSTER) {
          if (threadIdx.x < q.cluster) {
            put_remote(&peer[buf][at.rank][0], threadIdx.x, total);
            put_remote(&peer[buf][at.rank][1], threadIdx.x, sq);
            put_remote(&peer[buf][at.rank][2], threadIdx.x, n);
          }
          cluster_barrier();
          const bool have = lane < q.cluster;
          const float ps = have ? peer[buf][lane][0] : 0.f, pq = have ? peer[buf][lane][1] : 0.f, pn = have ? peer[buf][lane][2] : 0.f;
          total = warp_sum(ps);
          const float d = pn > 0.f ? ps / pn - total * inv_n : 0.f;
          sq = warp_sum(fmaf(pn * d, d, pq));
        }
        s[r] = total;
        m2[r] = sq;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = s[r] * inv_n;
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = 1.f / sqrtf(m2[r] * inv_n + p.eps);
      if (at.t == 0 && at.rank == 0 && row + r * step < rows) {
        p.mean[row + r * step] = mean[r];
        p.rstd[row + r * step] = rstd[r];
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 w[P], b[P];
      if constexpr (kInRegs) {
        copy_pairs(wr, w);
        copy_pairs(br, b);
      } else {
        param_get<T>(params + (2 * k) * kParam, w);
        param_get<T>(params + (2 * k + 1) * kParam, b);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!mask[k] || row + r * step >= rows) continue;
        const size_t e = out + r * out_step + k * kstep;
        if (RES && p.out2) store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out2) + e), v[r][k], mask[k]);
        normalise(v[r][k], mean[r], rstd[r], w, b);
        store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out) + e), v[r][k], mask[k]);
      }
    }
    out += R * out_step;
  }
  if (CLUSTER) cluster_barrier();      // no CTA leaves while a peer may still write into it
}

// ---- long rows ---------------------------------------------------------------------------------
// A row lies in the shared memory of up to eight CTAs: it is read from HBM once and walked three
// times there (sum, deviations, result).  Each granule's slot takes the next row's as soon as the
// result is written, so that row arrives while this one is stored.
template <typename T, bool RES, bool EDGE>
__global__ void __launch_bounds__(kMaxTeam, 2) ln_fwd_long(LnArgs p, RowPlan q) {
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ float2 red[2][kMaxTeam / 32];
  __shared__ float counts[kMaxTeam / 32];
  __shared__ float peer[2][kMaxCluster][3];
  constexpr int E = kE<T>, P = kPairs<T>, kOps = RES ? 2 : 1;
  constexpr uint32_t kAll = (1u << E) - 1;
  if (q.cluster > 1) cluster_barrier();      // every CTA has started before one writes into another
  const RowWalk at(q, p.cols, E);
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const int rows = static_cast<int>(p.rows), step = at.step, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long key = RES && p.drop.on ? __ldg(p.drop.seed) : 0;
  const int j0 = at.rank * q.chunk + at.t;
  const uint32_t slots = sm100::smem_u32(ring) + warp * (q.per_thread * kOps * kUnit) + lane * 16;
  constexpr uint32_t kStep = kMaxTeam * 16;

  auto mask_of = [&](int k) { return column_mask<T, EDGE>(at, q, at.t + k * kMaxTeam, p.cols); };
  const int mine = at.t < q.chunk ? (q.chunk - at.t + kMaxTeam - 1) / kMaxTeam : 0;      // granules of this thread, some perhaps empty
  float count = 0.f;
  for (int k = 0; k < mine; ++k) count += static_cast<float>(__popc(mask_of(k)));
  count = warp_sum(count);
  if (lane == 0) counts[warp] = count;

  const int ends = last_rows<T, EDGE>(rows, p.cols);
  auto fetch = [&](int row, int k) {
    if (row >= rows || !mask_of(k)) return;
    const size_t a = row_offset<T, EDGE>(row, p.ld_a, p.cols, j0) * sizeof(T) + static_cast<size_t>(k) * kStep;
    ring_copy(slots + (k * kOps) * kUnit, p.a, a, EDGE && row >= ends, p.rows * p.cols * sizeof(T));
    if (RES) {
      const size_t b = row_offset<T, EDGE>(row, p.ld_b, p.cols, j0) * sizeof(T) + static_cast<size_t>(k) * kStep;
      ring_copy(slots + (k * kOps + 1) * kUnit, p.b, b, EDGE && row >= ends, p.rows * p.cols * sizeof(T));
    }
  };
  // with a residual the sum is kept as fp32 in the granule's two slots
  auto value = [&](int k, float2 (&v)[P]) {
    if constexpr (RES) param_get<T>(slots + (k * kOps) * kUnit, v);
    else ring_get<T>(slots + (k * kOps) * kUnit, v);
  };

  for (int k = 0; k < mine; ++k) fetch(at.first, k);
  cp_async_commit();
  __syncthreads();
  int buf = 0;
  for (int row = at.first; row < rows; row += step, buf ^= 1) {
    const size_t out = row_offset<T, EDGE>(row, p.cols, p.cols, j0) * sizeof(T);
    cp_async_wait(0);
    float2 sum = both(0.f);
#pragma unroll 4
    for (int k = 0; k < mine; ++k) {
      const uint32_t m = mask_of(k);
      if (!m) continue;
      float2 v[P];
      ring_get<T>(slots + (k * kOps) * kUnit, v);
      if (RES) {
        float2 res[P];
        ring_get<T>(slots + (k * kOps + 1) * kUnit, res);
        if (p.drop.on) {
          const size_t g[1] = {(out + static_cast<size_t>(k) * kStep) / 16};
          Signs<T> gone[1];
          granule_signs<T, 1>(p.drop, key, g, gone);
          apply_signs<T>(v, gone[0], p.drop.scale);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = add2(res[i], v[i]);
        param_put<T>(slots + (k * kOps) * kUnit, v);
      }
      if (EDGE && m != kAll) zero_outside(v, m);
#pragma unroll
      for (int i = 0; i < P; ++i) sum = add2(sum, v[i]);
    }
    const float x = warp_sum(sum.x + sum.y), centre = count > 0.f ? x / count : 0.f;
    float2 dev = both(0.f);
#pragma unroll 4
    for (int k = 0; k < mine; ++k) {
      const uint32_t m = mask_of(k);
      if (!m) continue;
      float2 v[P];
      value(k, v);
      dev = deviations(v, centre, m, !EDGE || m == kAll, dev);
    }
    const float y = warp_sum(dev.x + dev.y);
    if (lane == 0) red[buf][warp] = make_float2(x, y);
    __syncthreads();
    float mean, m2;
    {
      constexpr int kWarps = kMaxTeam / 32;
      const float2 f = lane < kWarps ? red[buf][lane] : make_float2(0.f, 0.f);
      const float c = lane < kWarps ? counts[lane] : 0.f;
      const float total = warp_sum(f.x), n = warp_sum(c);
      const float m = n > 0.f ? total / n : 0.f;
      const float d = c > 0.f ? f.x / c - m : 0.f;
      m2 = warp_sum(fmaf(c * d, d, f.y));
      mean = m;
      if (q.cluster > 1) {
        if (threadIdx.x < q.cluster) {
          put_remote(&peer[buf][at.rank][0], threadIdx.x, total);
          put_remote(&peer[buf][at.rank][1], threadIdx.x, m2);
          put_remote(&peer[buf][at.rank][2], threadIdx.x, n);
        }
        cluster_barrier();
        const bool have = lane < q.cluster;
        const float ps = have ? peer[buf][lane][0] : 0.f, pq = have ? peer[buf][lane][1] : 0.f, pn = have ? peer[buf][lane][2] : 0.f;
        mean = warp_sum(ps) * inv_n;
        const float pd = pn > 0.f ? ps / pn - mean : 0.f;
        m2 = warp_sum(fmaf(pn * pd, pd, pq));
      }
    }
    const float rstd = 1.f / sqrtf(m2 * inv_n + p.eps);
    if (threadIdx.x == 0 && at.rank == 0) {
      p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
#pragma unroll 4
    for (int k = 0; k < mine; ++k) {
      const uint32_t m = mask_of(k);
      if (!m) continue;
      const long long col = static_cast<long long>(j0 + k * kMaxTeam) * E - at.m;
      float2 v[P], w[P], b[P];
      load_params<T>(p.w, p.w_f32, p.w_vec && !EDGE, col, m, 1.f, w);
      load_params<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col, m, 0.f, b);
      value(k, v);
      const size_t e = out + static_cast<size_t>(k) * kStep;
      if (RES && p.out2) store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out2) + e), v, m);
      normalise(v, mean, rstd, w, b);
      store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out) + e), v, m);
      fetch(row + step, k);
    }
    cp_async_commit();
  }
  if (q.cluster > 1) cluster_barrier();      // no CTA leaves while a peer may still write into it
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


template <typename Kernel>
int launch_fwd(Kernel kernel, std::atomic<int>* cache, const LnArgs& p, RowPlan q, cudaStream_t st) {
  int regs = 0;
  if (int rc = prepare("layer_norm_fwd", kernel, cache, &regs)) return rc;
  size_grid(p.rows, resident(q.groups * q.team, regs, q.smem), &q);
  if (!fit_clusters(kernel, &q)) return kDoesNotFit;
  return launch_rows("layer_norm_fwd", kernel, q, st, p, q);
}

template <typename T, int K, bool RES, bool EDGE, bool CLUSTER>
int rows_fwd(const LnArgs& p, const RowPlan& q, cudaStream_t st) {
  static std::atomic<int> cache[64];
  return launch_fwd(ln_fwd_rows<T, K, fwd_rows_between_barriers(K, kE<T>), RES, EDGE, CLUSTER>, cache, p, q, st);
}

template <typename T, bool RES, bool EDGE>
int long_fwd(const LnArgs& p, const RowPlan& q, cudaStream_t st) {
  static std::atomic<int> cache[64];
  return launch_fwd(ln_fwd_long<T, RES, EDGE>, cache, p, q, st);
}

template <typename T, bool RES, bool EDGE>
int pick_fwd(const LnArgs& p, const RowPlan& q, cudaStream_t st) {
  if (q.cluster > 1)
    return q.per_thread * kE<T> == 16 ? rows_fwd<T, 16 / kE<T>, RES, EDGE, true>(p, q, st) : rows_fwd<T, 32 / kE<T>, RES, EDGE, true>(p, q, st);
  switch (q.per_thread) {
    case 1: return rows_fwd<T, 1, RES, EDGE, false>(p, q, st);
    case 2: return rows_fwd<T, 2, RES, EDGE, false>(p, q, st);
    case 4: return rows_fwd<T, 4, RES, EDGE, false>(p, q, st);
    default: return rows_fwd<T, 32 / kE<T>, RES, EDGE, false>(p, q, st);
  }
}

template <typename T>
int fwd(const LnArgs& p, bool granules, cudaStream_t st) {
  RowPlan q;
  const int ops = p.b ? 2 : 1;
  const bool edge = p.cols % kE<T> != 0;
  int rc = kDoesNotFit;
  if (granules && plan_fwd_rows(p.rows, p.cols, sizeof(T), ops, &q)) {
    if (p.b) rc = edge ? pick_fwd<T, true, true>(p, q, st) : pick_fwd<T, true, false>(p, q, st);
    else rc = edge ? pick_fwd<T, false, true>(p, q, st) : pick_fwd<T, false, false>(p, q, st);
  }
  if (rc == kDoesNotFit && granules && plan_fwd_long(p.rows, p.cols, sizeof(T), ops, &q)) {
    if (p.b) rc = edge ? long_fwd<T, true, true>(p, q, st) : long_fwd<T, true, false>(p, q, st);
    else rc = edge ? long_fwd<T, false, true>(p, q, st) : long_fwd<T, false, false>(p, q, st);
  }
  if (rc != kDoesNotFit) return rc;
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
