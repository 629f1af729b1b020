// Walking the rows of a dense tensor 16 bytes ("a granule") at a time, fetched ahead by asynchronous
// copies.
//
// Granules lie at multiples of 16 bytes of the TENSOR, not of the row, so every access is aligned
// whatever the row length: a row that starts m elements into a granule owns only part of its first
// and last one.  Rows r and r + period have the same m when period * cols is a multiple of the
// granule's elements (period 1, 2, 4 or 8), and a team of threads is given rows of one residue only:
// its threads keep the same columns from row to row, and the parameters and column sums of those
// columns stay with them.
//
// Each thread copies the granules it will itself read (cp.async into shared memory, some rows
// ahead), so the ring needs no barrier: waiting for one's own copies is enough.  A warp's part of a
// stage is a block of units of 512 bytes, 16 a lane, one unit for each (granule, operand): a thread
// reaches all of its slots by constant offsets from one address, and neighbouring lanes always touch
// neighbouring 16 bytes (32 bytes a lane in two copies fetched every sector twice: 63 us instead of
// 42 for the 144256 x 128 fp32 backward).
#pragma once
#include <type_traits>
#include "philox.cuh"
#include "sm100.cuh"
#include "types.cuh"

namespace mb {

// Threads of a CTA: what the registers of an SM hold at 80 a thread, or 128 where a thread has 32 values.
constexpr int kMaxThreads = 768, kMaxThreadsWide = 512;
constexpr int kMaxTeam = 512;     // threads of a CTA that share a row (a CTA of a cluster: all of them)
constexpr int kMaxCluster = 4;    // 4 CTAs of 200 KB still fill 132 of 148 SMs, 8 only 120, 16 only 112
constexpr int kUnit = 512;
template <typename T> constexpr int kE = 16 / static_cast<int>(sizeof(T));    // elements of a granule
template <typename T> constexpr int kPairs = kE<T> / 2;

// How a kernel goes about a row: all of it by one team; by a cluster of CTAs; or, when it is long, a
// chunk per CTA in two kernels, one for the row's statistics and one for the result.
enum Pass { kWhole, kCluster, kStats, kApply };

struct RowPlan {
  int team;        // threads of a CTA that share a row: a power of two up to 32, or a multiple of 32
  int groups;      // teams per CTA
  int per_thread;  // granules per thread (K of the kernel)
  int cluster;     // CTAs that share a row (then groups == 1): a cluster, or the chunks of a long row
  int chunk;       // granules of a row per CTA
  int stages;      // rows in flight per team
  int period;
  int grid;        // CTAs, a multiple of cluster * period
  size_t smem;     // bytes of shared memory
};

// Where a thread stands: its team, its rows (first, first + step, ...) and its granules.
struct RowWalk {
  int group, t, rank, m, first, step;
  // With `last` >= 0 the walk counts rows from that one backwards.
  __device__ __forceinline__ RowWalk(const RowPlan& q, size_t cols, int elems, int last = -1) {
    group = threadIdx.x / q.team;
    t = threadIdx.x - group * q.team;
    const int cta = blockIdx.x / q.cluster;
    rank = blockIdx.x - cta * q.cluster;
    const int residue = cta % q.period;
    m = static_cast<int>((static_cast<unsigned>(last >= 0 ? last - residue : residue) * static_cast<unsigned>(cols)) & (elems - 1));
    step = static_cast<int>(gridDim.x / q.cluster / q.period) * q.groups * q.period;
    first = residue + q.period * (cta / q.period * q.groups + group);
  }
  // Teams that share a warp shuffle together, so they leave a loop over rows together: how far the
  // warp's first team is behind this one.
  __device__ __forceinline__ int spare(const RowPlan& q) const {
    return q.team < 32 ? (group - static_cast<int>(threadIdx.x & ~31u) / q.team) * q.period : 0;
  }
};

// Which elements of granule `jl` of the CTA's chunk belong to the row (0: none).
template <typename T, bool EDGE>
__device__ __forceinline__ uint32_t column_mask(const RowWalk& at, const RowPlan& q, int jl, size_t cols) {
  constexpr int E = kE<T>;
  constexpr uint32_t all = (1u << E) - 1;
  const int j = at.rank * q.chunk + jl, granules = static_cast<int>((at.m + cols + E - 1) / E);
  if (jl >= q.chunk || j >= granules) return 0;
  uint32_t mask = all;
  if (EDGE) {
    const long long col = static_cast<long long>(j) * E - at.m, n = static_cast<long long>(cols);
    if (col < 0) mask &= all << -col;
    if (col + E > n) mask &= all >> (col + E - n);
  }
  return mask;
}

// Element offset of granule `j` of a row.
template <typename T, bool EDGE>
__device__ __forceinline__ size_t row_offset(size_t row, size_t ld, size_t cols, int j) {
  return (EDGE ? (row * cols) & ~size_t(kE<T> - 1) : row * ld) + static_cast<size_t>(j) * kE<T>;
}

// ---- asynchronous copies -------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `n` of this thread's newest copy groups are in flight.
__device__ __forceinline__ void cp_async_wait(int n) {
  switch (n) {      // uniform
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
  }
}
// The granule at byte `off` of a tensor; with `last`, one that may reach behind the tensor's end, where
// it is filled with zeros.
__device__ __forceinline__ void ring_copy(uint32_t dst, const void* base, size_t off, bool last, size_t bytes) {
  const char* src = static_cast<const char*>(base) + off;
  if (last) cp_async16(dst, src, bytes - off >= 16 ? 16 : static_cast<int>(bytes - off));
  else cp_async16(dst, src, 16);
}
// Rows from this one on have granules that may reach behind the tensor's end.
template <typename T, bool EDGE>
__device__ __forceinline__ int last_rows(int rows, size_t cols) {
  return EDGE ? rows - 1 - (cols < kE<T> ? kE<T> : 0) : rows;
}

// ---- pairs of fp32 -------------------------------------------------------------------------
// Two fp32 operations in one instruction (each half rounds as the scalar operation does).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 w, x, y;\n mov.b64 {%0, %1}, w;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 w, x, y;\n mov.b64 {%0, %1}, w;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 1 / v for 2^-126 <= |v| <= 2^126, off by one unit in the last place at most.  (Outside that range v or 1 / v
// is subnormal, which the instruction takes for zero, or 1 / v overflows.)
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ bool has_reciprocal(float v) { return __float_as_uint(fabsf(v)) - 0x00800000u <= 0x7e000000u; }
// a / v for any v: at the ends of the range both are moved away from them by a power of two.
__device__ __forceinline__ float quotient(float a, float v) {
  const float f = fabsf(v) < 0x1p-60f ? 0x1p64f : fabsf(v) > 0x1p60f ? 0x1p-64f : 1.f;
  return a * f * reciprocal(v * f);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ---- granules as pairs ---------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void unpack(const uint4& a, float2 v[kPairs<T>]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
  if constexpr (sizeof(T) == 4) {
    v[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    v[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float2 v[kPairs<T>]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    w[0] = __float_as_uint(v[0].x); w[1] = __float_as_uint(v[0].y);
    w[2] = __float_as_uint(v[1].x); w[3] = __float_as_uint(v[1].y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __float22half2_rn(v[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float element(const float2* v, int i) { return i & 1 ? v[i >> 1].y : v[i >> 1].x; }

// Stores the elements of `mask` at p, which is aligned to 16 bytes; with EDGE a row may share the
// granule with its neighbour, and then only its own elements are written.
template <typename T, bool EDGE>
__device__ __forceinline__ void store_granule(T* p, const float2 v[kPairs<T>], uint32_t mask) {
  if (!EDGE || mask == (1u << kE<T>) - 1) {
    *reinterpret_cast<uint4*>(p) = pack<T>(v);
  } else {
#pragma unroll
    for (int i = 0; i < kE<T>; ++i)
      if ((mask >> i) & 1u) p[i] = from_f32<T>(element(v, i));
  }
}

__device__ __forceinline__ uint4 smem_get(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void smem_put(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <typename T> __device__ __forceinline__ void ring_get(uint32_t a, float2 v[kPairs<T>]) { unpack<T>(smem_get(a), v); }

// The fp32 parameters of a granule: one unit for fp32 tensors, two for 16-bit ones.
template <typename T> constexpr int kParamUnits = kE<T> / 4;
template <typename T> __device__ __forceinline__ void param_put(uint32_t a, const float2 v[kPairs<T>]) {
#pragma unroll
  for (int h = 0; h < kParamUnits<T>; ++h) smem_put(a + h * kUnit, pack<float>(v + 2 * h));
}
template <typename T> __device__ __forceinline__ void param_get(uint32_t a, float2 v[kPairs<T>]) {
#pragma unroll
  for (int h = 0; h < kParamUnits<T>; ++h) unpack<float>(smem_get(a + h * kUnit), v + 2 * h);
}
template <int N> __device__ __forceinline__ void copy_pairs(const float2 (&a)[N], float2* b) {
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = a[i];
}
// A granule's parameters from column `col` on; those outside `mask` read as `other`.
template <typename T>
__device__ __forceinline__ void load_params(const void* p, bool is_f32, bool vec, long long col, uint32_t mask, float other, float2 v[kPairs<T>]) {
  constexpr int E = kE<T>;
  if (!p || mask == 0) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) v[i] = both(other);
  } else if (vec && mask == (1u << E) - 1) {
    if (is_f32) {
#pragma unroll
      for (int h = 0; h < E / 4; ++h) unpack<float>(__ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + col) + h), v + 2 * h);
    } else {
      unpack<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p) + col)), v);
    }
  } else {
    float f[E];
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = (mask >> i) & 1u ? param<T>(p, is_f32, static_cast<size_t>(col + i)) : other;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
  }
}

// What dropout does to N granules of the tensor (numbers g): sign bits as in Dropped, one word for
// each pair of elements.
template <typename T> struct Signs { uint32_t d[kPairs<T>]; };
template <typename T, int N>
__device__ __forceinline__ void granule_signs(const Drop& p, unsigned long long key, const size_t (&g)[N], Signs<T> (&out)[N]) {
  unsigned long long block[N];
  Dropped f[N];
#pragma unroll
  for (int n = 0; n < N; ++n) block[n] = kE<T> == 8 ? g[n] : g[n] >> 1;
  dropped<N>(p, key, block, f);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) out[n].d[i] = kE<T> == 8 || !(g[n] & 1) ? f[n].d[i] : f[n].d[i + 4 - kPairs<T>];
}
template <typename T, int P>
__device__ __forceinline__ void apply_signs(float2 (&v)[P], const Signs<T>& s, float scale) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    v[i] = mul2(v[i], both(scale));
    v[i].x = zero_if(v[i].x, sign_low(s.d[i]));
    v[i].y = zero_if(v[i].y, sign_high(s.d[i]));
  }
}
template <int N>
__device__ __forceinline__ void zero_outside(float2 (&v)[N], uint32_t mask) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!((mask >> (2 * i)) & 1u)) v[i].x = 0.f;
    if (!((mask >> (2 * i)) & 2u)) v[i].y = 0.f;
  }
}

// ---- sums over a team ----------------------------------------------------------------------
// N sums over a warp for the price of little more than one: lanes hand over the values they do not
// keep.  Sum i ends in the lanes [i * 32 / N, (i + 1) * 32 / N).
__device__ __forceinline__ float warp_sums(const float (&s)[1]) { return warp_sum(s[0]); }
__device__ __forceinline__ float warp_sums(const float (&s)[2]) {
  const bool up = threadIdx.x & 16;
  float x = (up ? s[1] : s[0]) + __shfl_xor_sync(0xffffffffu, up ? s[0] : s[1], 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float warp_sums(const float (&s)[4]) {
  const bool up = threadIdx.x & 16, odd = threadIdx.x & 8;
  float x = (up ? s[2] : s[0]) + __shfl_xor_sync(0xffffffffu, up ? s[0] : s[2], 16);
  const float y = (up ? s[3] : s[1]) + __shfl_xor_sync(0xffffffffu, up ? s[1] : s[3], 16);
  x = (odd ? y : x) + __shfl_xor_sync(0xffffffffu, odd ? x : y, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// (sum, squared deviations from the own mean) of `n` values each in N sets of a team's lanes (a power of
// two up to 32), merged: for equal counts n the deviations grow by (sum a - sum b)^2 / 2n.  One pass
// over the lanes instead of one for the mean and another for the deviations.
template <int N>
__device__ __forceinline__ void merge_lanes(float (&s)[N], float (&m2)[N], int lanes, float n) {
  float f = 0.5f / n;
  for (int o = 1; o < lanes; o <<= 1, f *= 0.5f)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float t = __shfl_xor_sync(0xffffffffu, s[i], o), d = s[i] - t;
      m2[i] = fmaf(d * f, d, m2[i] + __shfl_xor_sync(0xffffffffu, m2[i], o));
      s[i] += t;
    }
}
// The N values of a row of `n` rows of N floats (64 at most) in shared memory summed over the rows, by every lane.
template <int N>
__device__ __forceinline__ void gather(const float* f, int n, float (&s)[N]) {
  if (n <= 8) {        // few: every lane reads them all, without a chain of shuffles
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = f[i];
    for (int w = 1; w < n; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += f[w * N + i];
    return;
  }
  const int lane = threadIdx.x & 31;
  float x = lane < N * n ? f[lane] : 0.f;
  if (N * n > 32) x += lane + 32 < N * n ? f[lane + 32] : 0.f;
#pragma unroll
  for (int o = N; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = N == 1 ? x : __shfl_sync(0xffffffffu, x, i);
}
// Over aligned groups of `lanes` (a power of two up to 32).
template <int N>
__device__ __forceinline__ void lanes_sums(float (&s)[N], int lanes) {
  if (lanes == 32) {
    const float x = warp_sums(s);
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = N == 1 ? x : __shfl_sync(0xffffffffu, x, i * (32 / N));
    return;
  }
  for (int o = lanes >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
}

__device__ __forceinline__ void team_barrier(int group, int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(team) : "memory");
}

// ---- cluster ---------------------------------------------------------------------------------
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_remote(const void* smem, int rank, float v) {   // into CTA `rank`'s copy of `smem`
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(smem)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

}  // namespace mb
