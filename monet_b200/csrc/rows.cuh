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

constexpr int kMaxThreads = 512;

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
    default: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
  }
}

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
