// Layer norm over the last `cols` values of each row, plain or fused with the dropout and the
// residual add before it, forward and backward (from the normalised tensor or from the output).
//
//   forward    v = x | residual + dropout(x);  mean, rstd of the row;  y = (v - mean) rstd w + b
//   backward   xhat = (v - mean) rstd | (y - b) / w,  g = dy w,
//              dv = rstd (g - mean(g) - xhat mean(g xhat)) (+ dsum),  dx = dropout(dv),
//              dw = sum_rows dy xhat,  db = sum_rows dy
//
// Everything is computed in fp32; outputs are rounded once.  Sums over rows are made in a fixed
// order: per-CTA partials in the workspace, then one reduction.
#pragma once
#include <atomic>
#include <initializer_list>
#include <utility>
#include "rows.cuh"

namespace mb {
namespace {

struct LnArgs {
  const void *a, *b, *c;       // forward: x, residual; backward: dy, kept, dsum
  const void *w, *bias;
  void *out, *out2;            // forward: y, sum; backward: dv, dx
  float *mean, *rstd;          // written by the forward, read by the backward
  size_t rows, cols, ld_a, ld_b, ld_c;
  bool w_f32;                  // parameters are fp32 (else the activations' type)
  bool w_vec;                  // ... and lie on 16-byte boundaries
  float eps;
  Drop drop;
};

// ---- rows in registers ---------------------------------------------------------------------
// A team of threads (part of a warp up to a cluster of CTAs) holds a row in registers: it is read
// once, its statistics are formed from the registers, and the result is written.  Rows to come are
// fetched by asynchronous copies meanwhile (rows.cuh).

struct WarpSums { float4 v[2][kMaxThreads / 32]; };   // double-buffered by row: one barrier a row

// ---- any shape, any stride, any alignment ----------------------------------------------------
// One CTA per row, element-wise accesses; a row is read again for each of its three uses, from L2
// when it is long.
constexpr int kBlock = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();               // `red` may still be read from the sum before
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kBlock / 32; ++i) s += red[i];
  return s;
}

// ---- which kernel ------------------------------------------------------------------------------
// A row stays in registers when it fits kMaxTeam * K granules per CTA and eight CTAs, K being at
// most 4 (8 in a cluster) forward and 2 backward, where each value also has two column sums and a
// weight; longer rows, and tensors whose rows do not lie on granule boundaries in the same way, take
// the element-wise kernels.
constexpr int kRingLimit = 216 * 1024;

inline int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

inline bool plan_rows(size_t rows, size_t cols, int elem, int ops, bool backward, bool from_y, RowPlan* q) {
  if (rows >> 30) return false;                              // row numbers are 32-bit, and some steps ahead
  int g = 8;
  while (cols % g) g /= 2;                                   // gcd(cols, 8)
  q->period = 8 / g;
  const size_t most = (cols + (8 - g) + 7) / 8;              // granules a row can touch
  const int k_max = backward ? 2 : 4, k_cluster = backward ? 2 : 8;
  if (most > static_cast<size_t>(kMaxTeam) * 8 * k_cluster) return false;
  for (q->cluster = 1; q->cluster <= 8; q->cluster *= 2) {
    q->chunk = ceil_div(static_cast<long long>(most), q->cluster);
    if (q->chunk > kMaxTeam * (q->cluster == 8 ? k_cluster : k_max)) continue;
    if (q->chunk <= 32) {
      q->team = 1;
      while (q->team < q->chunk) q->team *= 2;
      q->per_thread = 1;
    } else {
      const int wish = backward ? 256 : 128;
      int k = 1;
      while (k < k_max && ceil_div(q->chunk, 32 * k) * 32 > wish) k *= 2;
      while (ceil_div(q->chunk, 32 * k) * 32 > kMaxTeam) k *= 2;
      q->per_thread = k;
      q->team = ceil_div(q->chunk, 32 * k) * 32;
    }
    const int threads = !backward ? 256 : q->per_thread == 1 ? 512 : 768;
    q->groups = q->cluster > 1 || q->team >= threads ? 1 : threads / q->team;
    if (q->team > 32 && q->groups > 15) q->groups = 15;      // named barriers
    const size_t stage = static_cast<size_t>(q->groups) * q->chunk * 8 * elem * ops;
    if (backward) {
      // two CTAs per SM of one granule a thread; fp32 weight (and its inverse and the bias) beside the ring
      const size_t params = static_cast<size_t>(q->chunk) * 32 * (from_y ? 3 : 1);
      const size_t budget = (q->per_thread == 1 ? 104 : 208) * 1024;
      const int deep = budget > params ? static_cast<int>((budget - params) / stage) : 0;
      q->stages = deep > 8 ? 8 : deep < kRows ? kRows : deep;
      q->smem = stage * q->stages + params;
      const size_t fold = q->groups > 1 ? static_cast<size_t>((q->groups + 1) / 2) * q->team * q->per_thread * 16 * sizeof(float) : 0;
      if (fold > q->smem) q->smem = fold;                    // the teams' column sums are folded there
    } else {
      const int deep = static_cast<int>(64 * 1024 / stage);
      q->stages = deep > 6 ? 6 : deep < 2 ? 2 : deep;
      q->smem = stage * q->stages;
    }
    if (q->smem <= kRingLimit) return true;
  }
  return false;
}

// CTAs: `per_sm` on every SM, no more than there are rows, a whole number of clusters of each residue.
inline void size_grid(size_t rows, int per_sm, RowPlan* q) {
  const long long unit = static_cast<long long>(q->cluster) * q->period;
  long long want = static_cast<long long>(num_sms()) * per_sm / unit;
  const size_t need = ((rows + q->period - 1) / q->period + q->groups - 1) / q->groups;
  if (static_cast<size_t>(want) > need) want = static_cast<long long>(need);
  if (want < 1) want = 1;
  q->grid = static_cast<int>(want * unit);
}


// The launches of one kernel: its register count (which bounds the CTAs per SM) and the device-side
// shared-memory limit are looked up once per device.
template <typename Kernel>
int prepare(const char* who, Kernel kernel, std::atomic<int>* cache, int* regs) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return fail(MB_ERR_LAUNCH, "%s: no current device", who);
  int r = cache[dev].load(std::memory_order_relaxed);
  if (r == 0) {
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingLimit);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, kernel);
    if (e != cudaSuccess) return fail(MB_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(cudaGetLastError()));
    r = a.numRegs + 1;
    cache[dev].store(r, std::memory_order_relaxed);
  }
  *regs = r - 1;
  return MB_OK;
}

// CTAs of `threads` threads that fit on an SM.
inline int resident(int threads, int regs, size_t smem) {
  const int by_regs = 65536 / ((regs + 7) / 8 * 8 * threads), by_threads = 2048 / threads;
  const int by_smem = static_cast<int>(size_t(227 * 1024) / (smem + 4096));
  const int n = by_regs < by_threads ? by_regs : by_threads;
  const int k = n < by_smem ? n : by_smem;
  return k < 1 ? 1 : k > 16 ? 16 : k;
}

template <typename... KArgs, typename... Args>
int launch_rows(const char* who, void (*kernel)(KArgs...), const RowPlan& q, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(q.grid);
  cfg.blockDim = dim3(q.groups * q.team);
  cfg.dynamicSmemBytes = q.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = q.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = q.cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  return after_launch(who);
}

// A cluster's CTAs run together: a grid of more clusters than fit at once would end in a second,
// nearly empty round.
template <typename Kernel>
void fit_clusters(Kernel kernel, RowPlan* q) {
  if (q->cluster == 1) return;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(q->grid);
  cfg.blockDim = dim3(q->groups * q->team);
  cfg.dynamicSmemBytes = q->smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = q->cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return;
  }
  n -= n % q->period;
  if (n >= q->period && q->grid > n * q->cluster) q->grid = n * q->cluster;
}

int check_desc(const char* who, const mb_ln_desc* d) {
  if (!d) return fail(MB_ERR_INVALID_ARGUMENT, "%s: null descriptor", who);
  if (!dtype_bytes(d->dtype)) return fail(MB_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", who, d->dtype);
  if (d->param_dtype != MB_F32 && d->param_dtype != d->dtype)
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: parameters must be fp32 or of the activations' type", who);
  if (d->cols == 0 || d->cols > 0x7fffffffULL) return fail(MB_ERR_UNSUPPORTED, "%s: cols must lie in [1, 2^31)", who);
  if (!(d->eps >= 0.f)) return fail(MB_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", who);
  return MB_OK;
}

bool natural(const mb_ln_desc* d, const void* p) { return aligned(p, dtype_bytes(d->dtype)); }
bool natural_param(const mb_ln_desc* d, const void* p) { return aligned(p, dtype_bytes(d->param_dtype)); }


// Whether every tensor's rows lie on granule boundaries in the same way.
inline bool on_granules(const mb_ln_desc* d, std::initializer_list<std::pair<const void*, size_t>> tensors) {
  for (const auto& t : tensors) {
    if (!t.first) continue;
    if (!aligned(t.first, 8 * dtype_bytes(d->dtype))) return false;
    if (d->cols % 8 ? t.second != d->cols : t.second % 8 != 0) return false;
  }
  return true;
}

}  // namespace
}  // namespace mb
