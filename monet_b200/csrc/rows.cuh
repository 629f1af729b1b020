// Walking the rows of a dense tensor eight values ("a granule": 16 bytes of a 16-bit type, 32 of
// fp32) at a time, fetched ahead by asynchronous copies.
//
// Granules lie at multiples of eight elements of the TENSOR, not of the row, so every access is
// aligned whatever the row length: a row that starts m elements into a granule owns only part of
// its first and last one.  Rows r and r + period have the same m when period * cols % 8 == 0
// (period 1, 2, 4 or 8), and a team of threads is given rows of one residue only: its threads keep
// the same columns from row to row, and the parameters and column sums of those columns stay in
// registers.  A granule is also one block of the dropout generator.
//
// Each thread copies the granules it will itself read (cp.async into shared memory, `stages` rows
// ahead), so the ring needs no barrier: waiting for one's own copies is enough.
#pragma once
#include "philox.cuh"
#include "sm100.cuh"
#include "types.cuh"

namespace mb {

constexpr int kMaxThreads = 768;  // a CTA
constexpr int kMaxTeam = 512;     // threads of a CTA that share a row
constexpr int kRows = 2;          // rows a team handles between two barriers

struct RowPlan {
  int team;        // threads of a CTA that share a row: a power of two up to 32, or a multiple of 32
  int groups;      // teams per CTA
  int per_thread;  // granules per thread (K of the kernel)
  int cluster;     // CTAs that share a row (then groups == 1)
  int chunk;       // granules of a row per CTA
  int stages;      // rows in flight per team
  int period;
  int grid;        // CTAs, a multiple of cluster * period
  size_t smem;     // bytes of the ring
};

// Where a thread stands: its team, its rows and its granules.
struct RowWalk {
  int group, t, rank, m;
  size_t first, step;
  __device__ __forceinline__ RowWalk(const RowPlan& q, int cols) {
    group = threadIdx.x / q.team;
    t = threadIdx.x - group * q.team;
    const int lane_cta = blockIdx.x / q.cluster;
    rank = blockIdx.x - lane_cta * q.cluster;
    const int cls = lane_cta % q.period;
    m = static_cast<int>((static_cast<unsigned>(cls) * static_cast<unsigned>(cols)) & 7u);
    step = static_cast<size_t>(gridDim.x / q.cluster / q.period) * q.groups * q.period;
    first = cls + static_cast<size_t>(q.period) * (static_cast<size_t>(lane_cta / q.period) * q.groups + group);
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `n` of this thread's newest copy groups are in flight.
__device__ __forceinline__ void cp_async_wait(int n) {
  switch (n) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    case 7: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 8;" ::: "memory"); break;
  }
}

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
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ void unpack8(const uint4& a, float v[8], __nv_bfloat16) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const uint4& a, float v[8], __half) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float v[8], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack8(const float v[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One granule in global memory.  `p` is aligned to the granule.
template <typename T> __device__ __forceinline__ void load8(const T* p, float v[8]) {
  unpack8(*reinterpret_cast<const uint4*>(p), v, T{});
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float v[8]) {
  const f8 r = ld8(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = r.v[i];
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float v[8]) {
  *reinterpret_cast<uint4*>(p) = pack8(v, T{});
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float v[8]) {
  f8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = v[i];
  st8(p, r);
}
// The elements of `mask` only: a granule that a row shares with its neighbour.
template <typename T> __device__ __forceinline__ void store8_masked(T* p, const float v[8], uint32_t mask) {
  if (mask == 0xffu) {
    store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((mask >> i) & 1u) p[i] = from_f32<T>(v[i]);
  }
}

// A granule of the ring: `pitch` granules per 16-byte plane (fp32 has two planes, so that
// neighbouring threads stay 16 bytes apart).
template <typename T> constexpr int kPlanes = static_cast<int>(sizeof(T) / 2);

template <typename T>
__device__ __forceinline__ void ring_fetch(uint32_t dst, int pitch, const T* src, size_t avail) {
  // `avail` elements from src on belong to the tensor; the rest of the granule is zero-filled
#pragma unroll
  for (int h = 0; h < kPlanes<T>; ++h) {
    constexpr int per = 16 / static_cast<int>(sizeof(T));
    const size_t left = avail > static_cast<size_t>(h * per) ? avail - h * per : 0;
    const int bytes = left >= static_cast<size_t>(per) ? 16 : static_cast<int>(left * sizeof(T));
    cp_async16(dst + h * pitch * 16, bytes ? src + h * per : src, bytes);
  }
}
template <typename T>
__device__ __forceinline__ void ring_fetch(uint32_t dst, int pitch, const T* src) {
#pragma unroll
  for (int h = 0; h < kPlanes<T>; ++h) cp_async16(dst + h * pitch * 16, src + h * (16 / sizeof(T)), 16);
}
template <typename T> __device__ __forceinline__ void ring_read(const uint4* src, int, float v[8]) { unpack8(*src, v, T{}); }
template <> __device__ __forceinline__ void ring_read<float>(const uint4* src, int pitch, float v[8]) {
  const uint4 a = src[0], b = src[pitch];
  v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
  v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
}

template <bool EDGE, typename T>
__device__ __forceinline__ void store8_row(T* p, const float v[8], uint32_t mask) {
  if (EDGE) store8_masked(p, v, mask);
  else store8(p, v);
}

// Which elements of the thread's k-th granule belong to its row (0: none).
template <bool EDGE>
__device__ __forceinline__ uint32_t column_mask(const RowWalk& at, const RowPlan& q, int granules, int cols, int k) {
  const int jl = at.t + k * q.team, j = at.rank * q.chunk + jl;
  if (jl >= q.chunk || j >= granules) return 0;
  uint32_t mask = 0xffu;
  if (EDGE) {
    const long long col = static_cast<long long>(j) * 8 - at.m;
    if (col < 0) mask &= 0xffu << -col;
    if (col + 8 > cols) mask &= 0xffu >> (col + 8 - cols);
  }
  return mask;
}

// The thread's granules of one row of a tensor into the ring.
template <typename T, int K, bool EDGE>
__device__ __forceinline__ void fetch_row(const T* from, size_t ld, size_t row, size_t rows, size_t cols, int j0, int team,
                                          const uint32_t (&mask)[K], uint32_t dst, int plane) {
  const size_t e = (EDGE ? ((row * cols) >> 3) * 8 : row * ld) + static_cast<size_t>(j0) * 8;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!mask[k]) continue;
    const size_t at = e + static_cast<size_t>(k * team) * 8;
    if (EDGE) ring_fetch<T>(dst + k * team * 16, plane, from + at, rows * cols - at);
    else ring_fetch<T>(dst + k * team * 16, plane, from + at);
  }
}

// Eight fp32 values in shared memory as two planes of float4, `pitch` apart.
__device__ __forceinline__ void put8(float4* p, int pitch, const float v[8]) {
  p[0] = make_float4(v[0], v[1], v[2], v[3]);
  p[pitch] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void get8(const float4* p, int pitch, float v[8]) {
  const float4 a = p[0], b = p[pitch];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// The same on four pairs.
__device__ __forceinline__ void get8(const float4* p, int pitch, float2 v[4]) {
  const float4 a = p[0], b = p[pitch];
  v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
}
template <typename T> __device__ __forceinline__ void ring_read(const uint4* src, int pitch, float2 v[4]) {
  float f[8];
  ring_read<T>(src, pitch, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float2 v[4]) {
  const float f[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
  store8(p, f);
}
template <bool EDGE, typename T>
__device__ __forceinline__ void store8_row(T* p, const float2 v[4], uint32_t mask) {
  const float f[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
  store8_row<EDGE>(p, f, mask);
}

// Eight parameters from column `col` on; those outside `mask` read as `other`.
template <typename T>
__device__ __forceinline__ void param8(const void* p, bool is_f32, bool vec, long long col, uint32_t mask, float other, float v[8]) {
  if (!p || mask == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = other;
  } else if (vec && mask == 0xffu) {
    if (is_f32) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + col));
      const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + col) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else if (sizeof(T) == 2) {
      load8(static_cast<const T*>(p) + col, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (mask >> i) & 1u ? param<T>(p, is_f32, static_cast<size_t>(col + i)) : other;
  }
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {   // over aligned groups of `lanes` (a power of two)
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Four sums over a warp for the price of little more than one: lanes hand over the values they do not
// keep.  Lane l ends with sum l / 8.
__device__ __forceinline__ float warp_sum4(float a, float b, float c, float d) {
  const int lane = threadIdx.x & 31;
  const bool up = lane & 16;
  float x = (up ? c : a) + __shfl_xor_sync(0xffffffffu, up ? a : c, 16);
  float y = (up ? d : b) + __shfl_xor_sync(0xffffffffu, up ? b : d, 16);
  const bool odd = lane & 8;
  x = (odd ? y : x) + __shfl_xor_sync(0xffffffffu, odd ? x : y, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ float4 f4_add(const float4& a, const float4& b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// The sum of `n` <= 16 float4 in shared memory, by every lane of the warp.
__device__ __forceinline__ float4 gather4(const float4* v, int n) {
  const int lane = threadIdx.x & 31;
  const float* f = reinterpret_cast<const float*>(v);
  float s = lane < 4 * n ? f[lane] : 0.f;
  if (n > 8) s += lane + 32 < 4 * n ? f[lane + 32] : 0.f;
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return make_float4(__shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, s, 1), __shfl_sync(0xffffffffu, s, 2),
                     __shfl_sync(0xffffffffu, s, 3));
}

__device__ __forceinline__ void team_barrier(int group, int team) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(team) : "memory");
}

// ---- cluster ---------------------------------------------------------------------------------
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_remote(const void* smem, int rank, float4 v) {   // into CTA `rank`'s copy of `smem`
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sm100::smem_u32(smem)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

}  // namespace mb
