// Layer norm backward: kernels and their choice (layernorm.cuh).  Each element type is compiled by a file
// of its own, layernorm_bwd_*.cu.
#pragma once
#include "layernorm.cuh"

namespace mb {
namespace {

// Backward.  partial[CTA of a row][0][col] = sum of dy xhat, [1][col] = sum of dy over the CTA's rows.
//
// R rows are handled between two barriers: their sums are formed from a first reading of the
// ring, then the rows are read a second time to form dv.  Reading twice costs shared-memory loads but
// no registers, which the column sums need; the parameters lie in shared memory for the same reason
// (in registers where a thread has one granule).  Several teams share an SM, so that one computes while
// another waits for its barrier.  (bf16 16384 x 4096: 155 us with everything in registers and one or two
// teams, 83 with the second reading and packed pairs, 70 with four teams of 32 values a thread.)
//
// Long rows (PASS): kStats writes the two sums of each chunk's warps, sums_of_rows[row][chunk][warp][2]; kApply finds
// the rows' sums there, [row][2], and forms dv and the column sums in one reading.
//
// With t = v - mean or y - b:  sum g xhat = rstd sum (dy t) w  or  sum dy t  (the weight cancels), and
// dw = sum over rows of (dy t) rstd  or  (sum dy t) / w, so xhat itself is never formed.
template <typename T, int K, int R, bool FROM_Y, bool DSUM, bool DROP, bool EDGE, int PASS>
__global__ void __launch_bounds__(K * kE<T> >= 32 ? kMaxThreadsWide : kMaxThreads) ln_bwd_rows(LnArgs p, RowPlan q, float* partial, float* sums_of_rows) {
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ float red[2][kMaxThreads / 32][2 * R];      // double-buffered by row: one barrier a row
  __shared__ float peer[2][kMaxCluster][2 * R];
  if (PASS == kCluster) cluster_barrier();      // every CTA has started before one writes into another
  if (PASS == kApply) asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int E = kE<T>, P = kPairs<T>, kOps = DSUM && PASS != kStats ? 3 : 2, kSlots = K * kOps, kKinds = FROM_Y ? 2 : 1;
  constexpr int kParam = kParamUnits<T> * kUnit;
  constexpr bool kInRegs = K == 1;
  // the result's pass walks the rows backwards: the last ones are still in L2
  const RowWalk at(q, p.cols, E, PASS == kApply ? static_cast<int>(p.rows) - 1 : -1);
  const float inv_n = 1.f / static_cast<float>(p.cols);
  const int j0 = at.rank * q.chunk + at.t;           // the thread's granules: j0 + k * team
  const int rows = static_cast<int>(p.rows), step = at.step;
  const uint32_t stride = (blockDim.x >> 5) * (kSlots * kUnit);      // a stage
  const uint32_t slots = sm100::smem_u32(ring) + (threadIdx.x >> 5) * (kSlots * kUnit) + (threadIdx.x & 31) * 16;
  const uint32_t params = sm100::smem_u32(ring) + q.stages * stride + (at.t >> 5) * (K * kKinds * kParam) + (at.t & 31) * 16;
  const uint32_t kstep = q.team * 16;

  uint32_t mask[K];
  float2 aw[K][P], ab[K][P];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    mask[k] = column_mask<T, EDGE>(at, q, at.t + k * q.team, p.cols);
#pragma unroll
    for (int i = 0; i < P; ++i) aw[k][i] = ab[k][i] = both(0.f);
  }

  // byte offset of the thread's first granule in the first of the rows at hand (all tensors are dense)
  auto actual = [&](int i) { return PASS == kApply ? rows - 1 - i : i; };
  size_t out = row_offset<T, EDGE>(at.first < rows ? actual(at.first) : 0, p.cols, p.cols, j0) * sizeof(T);
  const size_t out_step = (PASS == kApply ? ~size_t(0) : 1) * step * p.cols * sizeof(T);
  const int ends = last_rows<T, EDGE>(rows, p.cols);
  auto fetch = [&](uint32_t stage, int i, size_t off) {
#pragma unroll
    for (int o = 0; o < kOps; ++o)
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (mask[k]) ring_copy(stage + (k * kOps + o) * kUnit, o == 0 ? p.a : o == 1 ? p.b : p.c, off + k * kstep, EDGE && actual(i) >= ends, p.rows * p.cols * sizeof(T));
  };

  float2 wr[P], nbr[P];                // kInRegs: the weight; with FROM_Y minus the bias
  auto weight = [&](int k, float2 v[P]) {
    if constexpr (kInRegs) copy_pairs(wr, v); else param_get<T>(params + (k * kKinds) * kParam, v);
  };
  auto minus_bias = [&](int k, float2 v[P]) {
    if constexpr (kInRegs) copy_pairs(nbr, v); else param_get<T>(params + (k * kKinds + 1) * kParam, v);
  };
  // t and dy of one granule; zero outside the row
  auto read = [&](uint32_t stage, int k, float mean, float2 (&t)[P], float2 (&dy)[P]) {
    ring_get<T>(stage + (k * kOps + 1) * kUnit, t);
    if (FROM_Y) minus_bias(k, dy);
#pragma unroll
    for (int i = 0; i < P; ++i) t[i] = add2(t[i], FROM_Y ? dy[i] : both(-mean));
    ring_get<T>(stage + (k * kOps) * kUnit, dy);
    if (EDGE && mask[k] != (1u << E) - 1) {
      zero_outside(t, mask[k]);
      zero_outside(dy, mask[k]);
    }
  };

  auto column_sums = [&](int k, int i, float2 u, float2 dy, float rstd) {      // u = dy t
    ab[k][i] = add2(ab[k][i], dy);
    aw[k][i] = FROM_Y ? add2(aw[k][i], u) : fma2(u, both(rstd), aw[k][i]);
  };
  // slots that are never fetched hold zeros, so that the sums need not ask
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (!mask[k])
      for (int s = 0; s < q.stages; ++s)
#pragma unroll
        for (int o = 0; o < kOps; ++o) smem_put(slots + s * stride + (k * kOps + o) * kUnit, make_uint4(0, 0, 0, 0));
  for (int s = 0; s < q.stages; s += R) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (at.first + (s + r) * step < rows) fetch(slots + (s + r) * stride, at.first + (s + r) * step, out + (s + r) * out_step);
    cp_async_commit();
  }
  // every thread brings some granules' parameters, whichever teams they are for
  for (int i = kInRegs ? at.t : static_cast<int>(threadIdx.x); i < (kInRegs ? at.t + 1 : K * q.team); i += blockDim.x) {
    const uint32_t m = column_mask<T, EDGE>(at, q, i, p.cols);
    const long long col = static_cast<long long>(at.rank * q.chunk + i) * E - at.m;
    const int k = i / q.team, t = i - k * q.team;
    const uint32_t to = sm100::smem_u32(ring) + q.stages * stride + (t >> 5) * (K * kKinds * kParam) + (t & 31) * 16 + k * kKinds * kParam;
    float2 v[P];
    load_params<T>(p.w, p.w_f32, p.w_vec && !EDGE, col, m, 1.f, v);
    if constexpr (kInRegs) copy_pairs(v, wr); else param_put<T>(to, v);
    if (FROM_Y) {
      load_params<T>(p.bias, p.w_f32, p.w_vec && !EDGE, col, m, 0.f, v);
#pragma unroll
      for (int j = 0; j < P; ++j) v[j] = make_float2(-v[j].x, -v[j].y);
      if constexpr (kInRegs) copy_pairs(v, nbr); else param_put<T>(to + kParam, v);
    }
  }
  if (!kInRegs) __syncthreads();
  // With FROM_Y: whether `reciprocal` reaches all of the thread's weights, as it nearly always does.  The rows are
  // then finished by code without a choice in it (bf16 60000 x 512: 44 us; a choice for each granule 50,
  // `quotient` for every value 47).
  bool ordinary = true;
  if (FROM_Y && PASS != kStats) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 w[P];
      weight(k, w);
#pragma unroll
      for (int i = 0; i < P; ++i) ordinary = ordinary && has_reciprocal(w[i].x) && has_reciprocal(w[i].y);
    }
  }

  int row = at.first;
  const int spare = at.spare(q);
  float mean[R], rstd[R];
  auto statistics = [&](int first, float (&m)[R], float (&s)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = first + r * step;
      m[r] = !FROM_Y && i < rows ? __ldg(p.mean + actual(i)) : 0.f;
      s[r] = i < rows ? __ldg(p.rstd + actual(i)) : 0.f;
    }
  };
  statistics(row, mean, rstd);
  uint32_t stage = slots;
  int buf = 0;
  for (; row - spare < rows; row += R * step, buf ^= 1) {
    float mean_next[R], rstd_next[R];
    statistics(row + R * step, mean_next, rstd_next);
    cp_async_wait(q.stages / R - 1);
    float s[2 * R];                      // sum dy w and sum g t of each row
    if constexpr (PASS != kApply) {
    float2 t1[R], t2[R];
#pragma unroll
    for (int r = 0; r < R; ++r) t1[r] = t2[r] = both(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 w[P];
      weight(k, w);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row + r * step >= rows) continue;
        float2 t[P], dy[P];
        read(stage + r * stride, k, mean[r], t, dy);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 u = mul2(dy[i], t[i]);
          t1[r] = fma2(dy[i], w[i], t1[r]);
          t2[r] = FROM_Y ? add2(t2[r], u) : fma2(u, w[i], t2[r]);
          if (PASS != kStats) column_sums(k, i, u, dy[i], rstd[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = t1[r].x + t1[r].y;
      s[2 * r + 1] = t2[r].x + t2[r].y;
    }
    if constexpr (PASS == kStats) {      // every warp leaves its own: no barrier
      const float x = warp_sums(s);
      if ((threadIdx.x & (16 / R - 1)) == 0 && row < rows)
        sums_of_rows[((static_cast<size_t>(row) * q.cluster + at.rank) * (q.team >> 5) + (threadIdx.x >> 5)) * 2 + (threadIdx.x & 31) / (16 / R)] = x;
    } else if (q.team <= 32) {
      lanes_sums(s, q.team);
    } else {
      const float x = warp_sums(s);
      if ((threadIdx.x & (16 / R - 1)) == 0) red[buf][threadIdx.x >> 5][(threadIdx.x & 31) / (16 / R)] = x;
      team_barrier(at.group, q.team);
      gather(red[buf][at.group * (q.team >> 5)], q.team >> 5, s);
      if (PASS == kCluster) {
        if (threadIdx.x < q.cluster)
#pragma unroll
          for (int i = 0; i < 2 * R; ++i) put_remote(&peer[buf][at.rank][i], threadIdx.x, s[i]);
        cluster_barrier();
        gather(peer[buf][0], q.cluster, s);
      }
    }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = row + r * step;
        s[2 * r] = i < rows ? __ldcg(sums_of_rows + 2 * static_cast<size_t>(actual(i))) : 0.f;
        s[2 * r + 1] = i < rows ? __ldcg(sums_of_rows + 2 * static_cast<size_t>(actual(i)) + 1) : 0.f;
      }
    }
    if constexpr (PASS != kStats) {
    uint32_t gone[R][K];                 // what dropout drops, the pairs' sign bits folded into a word
    if (DROP) {
      const unsigned long long key = __ldg(p.drop.seed);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        size_t g[K];
        Signs<T> s8[K];
#pragma unroll
        for (int k = 0; k < K; ++k) g[k] = (out + r * out_step + k * kstep) / 16;
        granule_signs<T, K>(p.drop, key, g, s8);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          gone[r][k] = 0;
#pragma unroll
          for (int i = 0; i < P; ++i) gone[r][k] |= (s8[k].d[i] & 0x80008000u) >> i;
        }
      }
    }
    auto result = [&](auto ordinary_weights) {
    constexpr bool kOrdinary = decltype(ordinary_weights)::value;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 w[P];
      weight(k, w);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row + r * step >= rows) continue;
        // rstd (g - mean(g) - xhat mean(g xhat))
        const float2 c1 = both(-s[2 * r] * inv_n), c2 = both(FROM_Y ? -s[2 * r + 1] * inv_n : -s[2 * r + 1] * inv_n * rstd[r] * rstd[r]);
        float2 t[P], d[P];
        read(stage + r * stride, k, mean[r], t, d);
        if (PASS == kApply)
#pragma unroll
          for (int i = 0; i < P; ++i) column_sums(k, i, mul2(d[i], t[i]), d[i], rstd[r]);
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = fma2(d[i], w[i], c1);
        if (FROM_Y) {
#pragma unroll
          for (int i = 0; i < P; ++i)
            t[i] = kOrdinary ? mul2(t[i], make_float2(reciprocal(w[i].x), reciprocal(w[i].y)))
                             : make_float2(quotient(t[i].x, w[i].x), quotient(t[i].y, w[i].y));
        }
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = fma2(t[i], c2, d[i]);
        if (DSUM) {
          ring_get<T>(stage + r * stride + (k * kOps + 2) * kUnit, t);
#pragma unroll
          for (int i = 0; i < P; ++i) d[i] = fma2(d[i], both(rstd[r]), t[i]);
        } else {
#pragma unroll
          for (int i = 0; i < P; ++i) d[i] = mul2(d[i], both(rstd[r]));
        }
        const size_t e = out + r * out_step + k * kstep;
        if (mask[k]) store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out) + e), d, mask[k]);
        if (DROP) {
          Signs<T> s8;
#pragma unroll
          for (int i = 0; i < P; ++i) s8.d[i] = gone[r][k] << i;
          apply_signs<T>(d, s8, p.drop.scale);
          if (mask[k]) store_granule<T, EDGE>(reinterpret_cast<T*>(static_cast<char*>(p.out2) + e), d, mask[k]);
        }
      }
    }
    };
    if (!FROM_Y || __builtin_expect(ordinary, 1)) result(std::true_type{});
    else result(std::false_type{});
    }
    // the next rows into the slots just read for the last time
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + (q.stages + r) * step < rows) fetch(stage + r * stride, row + (q.stages + r) * step, out + (q.stages + r) * out_step);
    cp_async_commit();
    stage += R * stride;
    if (stage >= slots + q.stages * stride) stage = slots;
    out += R * out_step;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = mean_next[r];
      rstd[r] = rstd_next[r];
    }
  }
  if (PASS == kCluster) cluster_barrier();      // no CTA leaves while a peer may still write into it
  if (PASS == kStats || !partial) return;
  if (FROM_Y) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float2 w[P];
      weight(k, w);
#pragma unroll
      for (int i = 0; i < P; ++i) aw[k][i] = make_float2(aw[k][i].x / w[i].x, aw[k][i].y / w[i].y);
    }
  }
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
        for (int i = 0; i < P; ++i) {
          to[(k * 2 * P + i) * pitch] = aw[k][i];
          to[(k * 2 * P + P + i) * pitch] = ab[k][i];
        }
    }
    __syncthreads();
    if (at.group < n - low) {
      const float2* have = sums + at.group * q.team + at.t;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          aw[k][i] = add2(aw[k][i], have[(k * 2 * P + i) * pitch]);
          ab[k][i] = add2(ab[k][i], have[(k * 2 * P + P + i) * pitch]);
        }
    }
    n = low;
  }
  if (at.group == 0) {
    float* to = partial + static_cast<size_t>(blockIdx.x / q.cluster) * 2 * p.cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const long long col = static_cast<long long>(j0 + k * q.team) * E - at.m;
#pragma unroll
      for (int h = 0; h < E / 4; ++h) {
        if (mask[k] && !EDGE) {
          *reinterpret_cast<uint4*>(to + col + 4 * h) = pack<float>(aw[k] + 2 * h);
          *reinterpret_cast<uint4*>(to + p.cols + col + 4 * h) = pack<float>(ab[k] + 2 * h);
        }
      }
      if (EDGE) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if ((mask[k] >> i) & 1u) {
            to[col + i] = element(aw[k], i);
            to[p.cols + col + i] = element(ab[k], i);
          }
      }
    }
  }
}

// The sums of a long row from those of its `parts`: a CTA a row, into [row][2].
__global__ void __launch_bounds__(kBlock) ln_bwd_combine(const float* part_sums, int parts, float* row_sums) {
  __shared__ float red[kBlock / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const size_t row = blockIdx.x;
  const float2* f = reinterpret_cast<const float2*>(part_sums) + row * parts;
  float a = 0.f, b = 0.f;
  for (int i = threadIdx.x; i < parts; i += kBlock) {
    a += f[i].x;
    b += f[i].y;
  }
  a = block_sum(a, red);
  b = block_sum(b, red);
  if (threadIdx.x == 0) {
    row_sums[2 * row] = a;
    row_sums[2 * row + 1] = b;
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
  launch_dependent(&cfg, ln_bwd_finish<T>, partial, parts, cols, dw, db, w_f32);
  return after_launch("layer_norm_bwd_finish");
}

// Scratch: the partial column sums; for long rows also the chunks' and the rows' sums.
template <typename T, int K, bool FROM_Y, bool DSUM, bool DROP, bool EDGE, int PASS>
int launch_bwd(const LnArgs& p, RowPlan q, const Grads& g, cudaStream_t st, float* sums_of_rows = nullptr) {
  static std::atomic<int> cache[64];
  auto kernel = ln_bwd_rows<T, K, bwd_rows_between_barriers(K), FROM_Y, DSUM, DROP, EDGE, PASS>;
  int regs = 0;
  if (int rc = prepare("layer_norm_bwd", kernel, cache, &regs)) return rc;
  if (PASS == kCluster && !fit_clusters(kernel, &q)) return kDoesNotFit;
  const bool sums = PASS != kStats && (g.dw || g.db);
  if (int rc = launch_rows("layer_norm_bwd", PASS, kernel, q, st, p, q, sums ? g.ws : nullptr, sums_of_rows)) return rc;
  return sums ? finish<T>(g.ws, q.grid / q.cluster, p.cols, g.dw, g.db, p.w_f32, st) : MB_OK;
}

template <typename T, bool FROM_Y, bool DSUM, bool DROP, bool EDGE>
int pick_bwd(const LnArgs& p, const RowPlan& q, const Grads& g, cudaStream_t st) {
  constexpr int most = 32 / kE<T>;
  if (q.cluster > 1) return launch_bwd<T, most, FROM_Y, DSUM, DROP, EDGE, kCluster>(p, q, g, st);
  switch (q.per_thread) {
    case 1: return launch_bwd<T, 1, FROM_Y, DSUM, DROP, EDGE, kWhole>(p, q, g, st);
    case 2: return launch_bwd<T, 2, FROM_Y, DSUM, DROP, EDGE, kWhole>(p, q, g, st);
    case 4: return launch_bwd<T, 4, FROM_Y, DSUM, DROP, EDGE, kWhole>(p, q, g, st);
    default: return launch_bwd<T, most, FROM_Y, DSUM, DROP, EDGE, kWhole>(p, q, g, st);
  }
}

template <typename T, bool FROM_Y, bool DSUM, bool DROP, bool EDGE>
int long_bwd(const LnArgs& p, const RowPlan& q, const Grads& g, cudaStream_t st) {
  constexpr int K = 16 / kE<T>;
  float* row_sums = g.ws + static_cast<size_t>(q.grid / q.cluster) * 2 * p.cols;
  float* chunk_sums = row_sums + 2 * p.rows;      // (8-byte aligned, as cols * 2 and rows * 2 are even)
  if (int rc = launch_bwd<T, K, FROM_Y, false, false, EDGE, kStats>(p, q, g, st, chunk_sums)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows));
  cfg.blockDim = dim3(kBlock);
  cfg.stream = st;
  launch_dependent(&cfg, ln_bwd_combine, static_cast<const float*>(chunk_sums), q.cluster * (q.team / 32), row_sums);
  if (int rc = after_launch("layer_norm_bwd_combine")) return rc;
  return launch_bwd<T, K, FROM_Y, DSUM, DROP, EDGE, kApply>(p, q, g, st, row_sums);
}

template <typename T, bool FROM_Y, bool DSUM, bool DROP>
int pick_edge(const LnArgs& p, const RowPlan& q, bool is_long, const Grads& g, cudaStream_t st) {
  if (is_long) return p.cols % kE<T> ? long_bwd<T, FROM_Y, DSUM, DROP, true>(p, q, g, st) : long_bwd<T, FROM_Y, DSUM, DROP, false>(p, q, g, st);
  return p.cols % kE<T> ? pick_bwd<T, FROM_Y, DSUM, DROP, true>(p, q, g, st) : pick_bwd<T, FROM_Y, DSUM, DROP, false>(p, q, g, st);
}

template <typename T, bool FROM_Y>
int bwd(const LnArgs& p, const mb_ln_desc* d, bool granules, const Grads& g, cudaStream_t st) {
  // (a dx that equals dv because nothing is dropped is rare enough for the element-wise kernels)
  for (int is_long = 0; is_long <= 1 && granules && (p.drop.on || !p.out2); ++is_long) {
    RowPlan q;
    if (is_long ? !plan_bwd_long(d, p.c ? 3 : 2, FROM_Y, &q) : !plan_bwd(d, p.c ? 3 : 2, FROM_Y, &q)) continue;
    int rc;
    if (p.drop.on) rc = p.c ? pick_edge<T, FROM_Y, true, true>(p, q, is_long, g, st) : pick_edge<T, FROM_Y, false, true>(p, q, is_long, g, st);
    else rc = p.c ? pick_edge<T, FROM_Y, true, false>(p, q, is_long, g, st) : pick_edge<T, FROM_Y, false, false>(p, q, is_long, g, st);
    if (rc != kDoesNotFit) return rc;
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
