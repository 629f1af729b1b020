// Layer norm forward: kernels and entry point (layernorm.cuh).
#include "layernorm.cuh"

namespace mb {
namespace {

// ---- rows in registers -----------------------------------------------------------------------
// Statistics: every thread centres on its own mean, and (sum, squared deviations) are merged pairwise
// over the lanes, then over the warps and the CTAs of a cluster: no large values are squared and
// subtracted, and one pass over the lanes does.  (Where a warp's lanes hold different numbers of values it
// centres on the warp's mean instead.)  The chain of shuffles is what a row waits for: bf16 16384 x 4096
// took 63 us with one pass for the mean and one for the deviations, 57 with the merge.
// Long rows (PASS): two passes, 184 x 200704 fp32 91 us on inputs that are not in L2.  Held in the shared memory
// of clusters of eight or sixteen CTAs it took 100 where two passes took 80, since those leave a fifth of the
// SMs without work.
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

template <typename T, int K, int R, bool RES, bool EDGE, int PASS>
__global__ void __launch_bounds__(fwd_threads(K, kE<T>, RES)) ln_fwd_rows(LnArgs p, RowPlan q, float* partial) {
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ float2 red[2][kMaxThreads / 32][R];      // double-buffered by row: one barrier a row
  __shared__ float counts[kMaxThreads / 32];
  __shared__ float peer[2][kMaxCluster][3];
  if (PASS == kCluster) cluster_barrier();      // every CTA has started before one writes into another
  if (PASS == kApply) asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int E = kE<T>, P = kPairs<T>, kOps = RES ? 2 : 1, kSlots = K * kOps;
  constexpr int kParam = kParamUnits<T> * kUnit;
  constexpr uint32_t kAll = (1u << E) - 1;
  constexpr bool kInRegs = K == 1;
  // the result's pass walks the rows backwards: the last ones are still in L2
  const RowWalk at(q, p.cols, E, PASS == kApply ? static_cast<int>(p.rows) - 1 : -1);
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const int rows = static_cast<int>(p.rows), step = at.step, lane = threadIdx.x & 31, warps = q.team >> 5;
  auto actual = [&](int i) { return PASS == kApply ? rows - 1 - i : i; };
  const size_t forth = PASS == kApply ? ~size_t(0) : 1;      // -1 or 1
  const int begin = at.first < rows ? actual(at.first) : 0;
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

  size_t out = row_offset<T, EDGE>(begin, p.cols, p.cols, j0) * sizeof(T);
  const size_t out_step = forth * step * p.cols * sizeof(T);
  // inputs may have gaps between their rows
  size_t in_a = row_offset<T, EDGE>(begin, p.ld_a, p.cols, j0) * sizeof(T), in_b = RES ? row_offset<T, EDGE>(begin, p.ld_b, p.cols, j0) * sizeof(T) : 0;
  int next = at.first;
  const int ends = last_rows<T, EDGE>(rows, p.cols);
  auto fetch = [&](uint32_t stage) {
    if (next < rows) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!mask[k]) continue;
        ring_copy(stage + (k * kOps) * kUnit, p.a, in_a + k * kstep, EDGE && actual(next) >= ends, p.rows * p.cols * sizeof(T));
        if (RES) ring_copy(stage + (k * kOps + 1) * kUnit, p.b, in_b + k * kstep, EDGE && actual(next) >= ends, p.rows * p.cols * sizeof(T));
      }
      in_a += forth * step * p.ld_a * sizeof(T);
      if (RES) in_b += forth * step * p.ld_b * sizeof(T);
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
  // every thread brings some granules' parameters, whichever teams they are for
  for (int i = kInRegs ? at.t : static_cast<int>(threadIdx.x); PASS != kStats && i < (kInRegs ? at.t + 1 : K * q.team); i += blockDim.x) {
    const uint32_t m = column_mask<T, EDGE>(at, q, i, p.cols);
    const long long col = static_cast<long long>(at.rank * q.chunk + i) * E - at.m;
    const int k = i / q.team, t = i - k * q.team;
    const uint32_t to = sm100::smem_u32(ring) + q.stages * stride + (t >> 5) * (K * 2 * kParam) + (t & 31) * 16 + 2 * k * kParam;
    load_params<T>(p.w, p.w_f32, p.w_vec && !EDGE, col, m, 1.f, wr);
    load_params<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col, m, 0.f, br);
    if (!kInRegs) {
      param_put<T>(to, wr);
      param_put<T>(to + kParam, br);
    }
  }
  if (!kInRegs) __syncthreads();       // the parameters and the counts
  // Combining the warps' statistics, a lane looks after the warp of its number.  Warps with equal counts,
  // a power of two of them, merge like lanes.  The last CTA of a cluster may hold less than its chunk (16-bit
  // 32760: its last warp is 8 values short) and then merges by its counts.  (Asking the counts themselves gives
  // the same answer, but not one that the compiler knows to be the whole CTA's: bf16 4096 x 16384 64 us against 61.)
  const bool full = PASS != kCluster || static_cast<size_t>(at.rank + 1) * q.chunk * E <= p.cols;
  const bool alike = !EDGE && full && q.chunk == K * q.team && (warps & (warps - 1)) == 0;
  const float part_count = q.team > 32 && lane < warps ? counts[at.group * warps + lane] : 0.f;
  const float part_inv = part_count > 0.f ? 1.f / part_count : 0.f, part_total = q.team > 32 ? warp_sum(part_count) : 0.f;
  const float part_each = part_total > 0.f ? 1.f / part_total : 0.f;

  uint32_t stage = slots;
  int row = at.first, buf = 0;
  const int spare = at.spare(q);
  float mean_next[R], rstd_next[R];
  auto given = [&](int first) {        // the statistics of the rows from `first` on
    if constexpr (PASS == kApply) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (first + r * step < rows) {
          mean_next[r] = __ldcg(p.mean + actual(first + r * step));      // written by the kernel before
          rstd_next[r] = __ldcg(p.rstd + actual(first + r * step));
        }
    }
  };
  given(row);
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
    if constexpr (PASS != kApply) {
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
    if constexpr (PASS == kStats) {      // every warp leaves its own: no barrier
      if (lane == 0 && row < rows) {
        float* to = partial + ((static_cast<size_t>(row) * q.cluster + at.rank) * warps + (threadIdx.x >> 5)) * 3;
        to[0] = s[0];
        to[1] = m2[0];
        to[2] = count;
      }
    } else if (q.team > 32) {
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
        if (PASS == kCluster) {
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
    }
    if constexpr (PASS != kStats) {
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if constexpr (PASS == kApply) {
        mean[r] = mean_next[r];
        rstd[r] = rstd_next[r];
      } else {
        rstd[r] = 1.f / sqrtf(m2[r] * inv_n + p.eps);
        if (at.t == 0 && at.rank == 0 && row + r * step < rows) {
          p.mean[row + r * step] = mean[r];
          p.rstd[row + r * step] = rstd[r];
        }
      }
    }
    given(row + R * step);
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
    }
    out += R * out_step;
  }
  if (PASS == kCluster) cluster_barrier();      // no CTA leaves while a peer may still write into it
}

// The statistics of a long row from those of its `parts`: a CTA a row.
__global__ void __launch_bounds__(kBlock) ln_fwd_combine(const float* partial, int parts, LnArgs p) {
  __shared__ float red[kBlock / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const size_t row = blockIdx.x;
  const float* f = partial + row * parts * 3;
  const float inv_n = 1.f / static_cast<float>(p.cols);
  float s = 0.f, q = 0.f;
  for (int i = threadIdx.x; i < parts; i += kBlock) s += f[3 * i];
  const float mean = block_sum(s, red) * inv_n;
  for (int i = threadIdx.x; i < parts; i += kBlock) {
    const float n = f[3 * i + 2], d = n > 0.f ? f[3 * i] / n - mean : 0.f;
    q += fmaf(n * d, d, f[3 * i + 1]);
  }
  q = block_sum(q, red);
  if (threadIdx.x == 0) {
    p.mean[row] = mean;
    p.rstd[row] = 1.f / sqrtf(q * inv_n + p.eps);
  }
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


template <typename T, int K, bool RES, bool EDGE, int PASS>
int launch_fwd(const LnArgs& p, RowPlan q, float* partial, cudaStream_t st) {
  static std::atomic<int> cache[64];
  auto kernel = ln_fwd_rows<T, K, fwd_rows_between_barriers(K), RES, EDGE, PASS>;
  int regs = 0;
  if (int rc = prepare("layer_norm_fwd", kernel, cache, &regs)) return rc;
  size_grid(p.rows, resident(q.groups * q.team, regs, q.smem), &q);
  if (PASS == kCluster && !fit_clusters(kernel, &q)) return kDoesNotFit;
  return launch_rows("layer_norm_fwd", PASS, kernel, q, st, p, q, partial);
}

template <typename T, bool RES, bool EDGE>
int pick_fwd(const LnArgs& p, const RowPlan& q, cudaStream_t st) {
  if (q.cluster > 1) return launch_fwd<T, 32 / kE<T>, RES, EDGE, kCluster>(p, q, nullptr, st);
  switch (q.per_thread) {
    case 1: return launch_fwd<T, 1, RES, EDGE, kWhole>(p, q, nullptr, st);
    case 2: return launch_fwd<T, 2, RES, EDGE, kWhole>(p, q, nullptr, st);
    case 4: return launch_fwd<T, 4, RES, EDGE, kWhole>(p, q, nullptr, st);
    default: return launch_fwd<T, 32 / kE<T>, RES, EDGE, kWhole>(p, q, nullptr, st);
  }
}

template <typename T, bool RES, bool EDGE>
int long_fwd(const LnArgs& p, const RowPlan& q, float* partial, cudaStream_t st) {
  if (int rc = launch_fwd<T, 16 / kE<T>, RES, EDGE, kStats>(p, q, partial, st)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows));
  cfg.blockDim = dim3(kBlock);
  cfg.stream = st;
  launch_dependent(&cfg, ln_fwd_combine, static_cast<const float*>(partial), q.cluster * (q.team / 32), p);
  if (int rc = after_launch("layer_norm_fwd_combine")) return rc;
  return launch_fwd<T, 16 / kE<T>, RES, EDGE, kApply>(p, q, nullptr, st);
}

template <typename T>
int fwd(const LnArgs& p, bool granules, float* ws, cudaStream_t st) {
  RowPlan q;
  const int ops = p.b ? 2 : 1;
  const bool edge = p.cols % kE<T> != 0;
  int rc = kDoesNotFit;
  if (granules && plan_fwd_rows(p.rows, p.cols, sizeof(T), ops, &q)) {
    if (p.b) rc = edge ? pick_fwd<T, true, true>(p, q, st) : pick_fwd<T, true, false>(p, q, st);
    else rc = edge ? pick_fwd<T, false, true>(p, q, st) : pick_fwd<T, false, false>(p, q, st);
  }
  if (rc == kDoesNotFit && granules && plan_long(p.rows, p.cols, sizeof(T), ops, 2, &q)) {
    if (p.b) rc = edge ? long_fwd<T, true, true>(p, q, ws, st) : long_fwd<T, true, false>(p, q, ws, st);
    else rc = edge ? long_fwd<T, false, true>(p, q, ws, st) : long_fwd<T, false, false>(p, q, ws, st);
  }
  if (rc != kDoesNotFit) return rc;
  ln_fwd_any<T><<<grid_for(p.rows, 1, 8), kBlock, 0, st>>>(p);
  return after_launch("layer_norm_fwd");
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_layer_norm_fwd_workspace_bytes(const mb_ln_desc* d) {
  if (!d || d->cols == 0 || d->cols > 0x7fffffffULL || d->rows == 0 || !dtype_bytes(d->dtype)) return 0;
  size_t floats = 0;
  for (int ops = 1; ops <= 2; ++ops) {      // three values a warp, for rows that one team or cluster does not hold
    RowPlan q;
    if (plan_fwd_rows(d->rows, d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, &q) && q.cluster == 1) continue;
    if (!plan_long(d->rows, d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, 2, &q)) continue;
    const size_t n = d->rows * q.cluster * (q.team / 32) * 3;
    if (n > floats) floats = n;
  }
  return floats * sizeof(float);
}

int mb_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* y,
                      void* sum, float* mean, float* rstd, const mb_ln_desc* d, const mb_dropout_desc* drop,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "mb_layer_norm_fwd";
  if (int rc = check_desc(who, d)) return rc;
  LnArgs p{x, residual, nullptr, weight, bias, y, sum, mean, rstd, d->rows, d->cols, d->ld_a, d->ld_b, 0, d->param_dtype == MB_F32, aligned(weight, 16) && aligned(bias, 16), d->eps, {}};
  if (int rc = make_drop(who, drop, &p.drop)) return rc;
  if (d->rows == 0) return MB_OK;
  if (!x || !y || !mean || !rstd) return fail(MB_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (y == sum) return fail(MB_ERR_INVALID_ARGUMENT, "%s: y and sum must not be the same buffer", who);
  if (((y == x || sum == x) && d->ld_a != d->cols) || (residual && (y == residual || sum == residual) && d->ld_b != d->cols))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: only dense rows can be overwritten", who);
  if (drop && !residual) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout needs a residual", who);
  if (!natural(d, x) || !natural(d, residual) || !natural(d, y) || !natural(d, sum) || !natural_param(d, weight) ||
      !natural_param(d, bias) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  const size_t need = mb_layer_norm_fwd_workspace_bytes(d);
  if (need && (!workspace || !aligned(workspace, 4) || workspace_bytes < need))
    return fail(MB_ERR_WORKSPACE, "%s: workspace too small or misaligned", who);
  cudaStream_t st = as_stream(stream);
  float* ws = static_cast<float*>(workspace);
  const bool granules = on_granules(d, {{x, d->ld_a}, {residual, d->ld_b}, {y, d->cols}, {sum, d->cols}});
  if (d->dtype == MB_F32) return fwd<float>(p, granules, ws, st);
  if (d->dtype == MB_BF16) return fwd<__nv_bfloat16>(p, granules, ws, st);
  return fwd<__half>(p, granules, ws, st);
}

}  // extern "C"
