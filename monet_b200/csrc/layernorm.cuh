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
// Rows whose tensors lie on granule boundaries in the same way are walked in granules (rows.cuh), one
// thread holding up to 16 values (32 forward, where there are no column sums) and a team up to
// kMaxTeam threads.  Longer rows: forward stays in the shared memory of up to eight CTAs, backward in
// the registers of up to eight.  Everything else takes the element-wise kernels.
constexpr size_t kSmemLimit = 216 * 1024;

inline int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }
// Rows between two barriers of the backward kernel with k granules a thread.
constexpr int bwd_rows_between_barriers(int k) { return k == 1 ? 2 : 1; }
constexpr int fwd_rows_between_barriers(int k, int elems) { return k * elems <= 16 ? 2 : 1; }

// The period of the rows' alignment, and the granules that a row can touch.
inline size_t row_granules(size_t cols, int elems, int* period) {
  int g = elems;
  while (cols % g) g /= 2;
  *period = elems / g;
  return (cols + (elems - g) + elems - 1) / elems;
}

// Threads for `chunk` granules of up to `most` a thread; false if they do not fit a team.
inline bool plan_team(int chunk, int most, RowPlan* q) {
  q->chunk = chunk;
  q->per_thread = 1;
  if (chunk <= 32) {                   // several rows a warp, or one
    for (q->team = 1; q->team < chunk;) q->team *= 2;
    return true;
  }
  while (q->per_thread < most && chunk > 32 * q->per_thread) q->per_thread *= 2;    // one warp if possible: no barrier
  q->team = ceil_div(chunk, 32 * q->per_thread) * 32;
  return q->team <= kMaxTeam;
}

// Teams per CTA: as many as `threads` hold, fewer where the rows would not reach every SM.
inline void plan_groups(size_t rows, int threads, RowPlan* q) {
  q->groups = q->cluster > 1 ? 1 : threads / q->team;
  if (q->team > 32 && q->groups > 15) q->groups = 15;        // named barriers
  const size_t spread = (rows + num_sms() - 1) / num_sms();
  if (static_cast<size_t>(q->groups) > spread) q->groups = static_cast<int>(spread);
  if (q->groups < 1) q->groups = 1;
  if (q->team < 32) q->groups = (q->groups + 32 / q->team - 1) / (32 / q->team) * (32 / q->team);    // whole warps
}

inline bool plan_bwd_rows(size_t rows, size_t cols, int elem, int ops, bool from_y, RowPlan* q) {
  if (rows >> 30) return false;                              // row numbers are 32-bit, and some steps ahead
  const int elems = 16 / elem;
  const size_t most = row_granules(cols, elems, &q->period);
  if (most > static_cast<size_t>(kMaxTeam) * 8 * (16 / elems)) return false;
  for (q->cluster = 1; q->cluster <= 8; q->cluster *= 2) {
    if (!plan_team(ceil_div(most, q->cluster), 16 / elems, q)) continue;
    if (q->cluster > 1) {                                    // the cluster's kernel has 16 values a thread
      q->per_thread = 16 / elems;
      q->team = ceil_div(q->chunk, 32 * q->per_thread) * 32;
    }
    plan_groups(rows, kMaxThreads, q);
    // one CTA per SM; the fp32 weight (with from_y its inverse and the bias) beside the ring
    const int r = bwd_rows_between_barriers(q->per_thread);
    const size_t stage = static_cast<size_t>(q->groups * q->team / 32) * q->per_thread * ops * kUnit;
    const size_t params = q->per_thread == 1 ? 0 : static_cast<size_t>(q->team) * q->per_thread * elems * 4 * (from_y ? 3 : 1);
    const size_t deep = (kSmemLimit - params) / (r * stage);
    if (deep < 2) continue;
    q->stages = r * static_cast<int>(deep > 8 / r ? 8 / r : deep);
    q->smem = stage * q->stages + params;
    const size_t fold = q->groups > 1 ? static_cast<size_t>((q->groups + 1) / 2) * q->team * q->per_thread * elems * 2 * sizeof(float) : 0;
    if (fold > q->smem) q->smem = fold;                      // the teams' column sums are folded there
    return q->smem <= kSmemLimit;
  }
  return false;
}

inline bool plan_fwd_rows(size_t rows, size_t cols, int elem, int ops, RowPlan* q) {
  if (rows >> 30) return false;
  const int elems = 16 / elem;
  const size_t most = row_granules(cols, elems, &q->period);
  q->cluster = 1;
  if (most > static_cast<size_t>(kMaxTeam) * (32 / elems)) return false;
  if (!plan_team(static_cast<int>(most), 16 / elems, q)) {
    q->per_thread = 32 / elems;
    q->team = ceil_div(static_cast<int>(most), 32 * q->per_thread) * 32;
  }
  plan_groups(rows, kMaxThreads, q);
  const int r = fwd_rows_between_barriers(q->per_thread, elems);
  const size_t stage = static_cast<size_t>(q->groups * q->team / 32) * q->per_thread * ops * kUnit;
  const size_t params = q->per_thread == 1 ? 0 : static_cast<size_t>(q->team) * q->per_thread * elems * 8;
  const size_t budget = (q->groups * q->team > kMaxThreads / 2 ? kSmemLimit : 100 * 1024) - params;
  const size_t deep = budget / (r * stage);
  if (deep < 1) return false;
  q->stages = r * static_cast<int>(deep > 8 / r ? 8 / r : deep);
  q->smem = stage * q->stages + params;
  return true;
}

// One row in the shared memory of 1 to 8 CTAs, of which two share an SM if they are small enough.
inline bool plan_fwd_long(size_t rows, size_t cols, int elem, int ops, RowPlan* q) {
  if (rows >> 30) return false;
  const size_t most = row_granules(cols, 16 / elem, &q->period);
  for (size_t limit = 106 * 1024; limit <= kSmemLimit; limit += kSmemLimit - 106 * 1024)
    for (q->cluster = 1; q->cluster <= 8; q->cluster *= 2) {
      const size_t chunk = (most + q->cluster - 1) / q->cluster;
      if (chunk > 65536) continue;
      q->chunk = static_cast<int>(chunk);
      q->team = kMaxTeam;
      q->groups = 1;
      q->stages = 1;
      q->per_thread = ceil_div(q->chunk, q->team);
      q->smem = static_cast<size_t>(q->team) / 32 * q->per_thread * ops * kUnit;
      if (q->smem <= limit) return true;
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
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemLimit));
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


// Whether every tensor's rows (address, row stride) lie on granule boundaries in the same way.
inline bool on_granules(const mb_ln_desc* d, std::initializer_list<std::pair<const void*, size_t>> tensors) {
  for (const auto& t : tensors) {
    if (!t.first) continue;
    const size_t elems = 16 / dtype_bytes(d->dtype);
    if (!aligned(t.first, 16)) return false;
    if (d->cols % elems ? t.second != d->cols : t.second % elems != 0) return false;
  }
  return true;
}

}  // namespace
}  // namespace mb
