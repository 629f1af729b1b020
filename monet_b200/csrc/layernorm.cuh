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
//
// Bound by HBM for large tensors: forward reads and writes each element once, backward reads two or
// three tensors and writes one or two.  Measured against a copy at 6569 GB/s: forward bf16 16384 x 8192
// 89 us (0.92), 16384 x 4096 50 us (0.82); backward bf16 16384 x 4096 70 us (0.88), fp32 144256 x 128 from
// the output 42 us (0.80); with dropout, add and sum bf16 8192 x 2048 forward 32 us (0.64), backward 46 us
// (0.56), where latency is what is left: the generator stands in series with a row's reductions, and
// issue is active half of the time.
// Small calls (a few microseconds) are bound by their launches.
#pragma once
#include <atomic>
#include <initializer_list>
#include <utility>
#include "rows.cuh"

namespace mb {

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
// Where the backward's sums over rows go, and its workspace.
struct Grads { void *dw, *db; float* ws; };

namespace {

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
// Rows whose tensors lie on granule boundaries in the same way are walked in granules (rows.cuh): a
// thread holds 4 to 32 values, a team up to kMaxTeam threads, a cluster up to four of these.  Longer rows
// are walked twice, for the sums and for the result.  Everything else takes the element-wise kernels.
constexpr size_t kSmemLimit = 225 * 1024;

inline int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }
// Rows between two barriers of the backward kernel with k granules a thread.
constexpr int bwd_rows_between_barriers(int k) { return k == 1 ? 2 : 1; }
constexpr int fwd_rows_between_barriers(int k) { return k == 1 ? 2 : 1; }
// Threads of a forward CTA: 32 values a thread fit 80 registers in the plain form alone (768 threads
// instead of 512: bf16 16384 x 8192 107 -> 89 us).
constexpr int fwd_threads(int k, int elems, bool residual) {
  return k * elems >= 32 && residual ? kMaxThreadsWide : kMaxThreads;
}

// The period of the rows' alignment, and the granules that a row can touch.
inline size_t row_granules(size_t cols, int elems, int* period) {
  int g = elems;
  while (cols % g) g /= 2;
  *period = elems / g;
  return (cols + (elems - g) + elems - 1) / elems;
}

// A team for `chunk` granules with `values` values a thread.
inline void plan_team(int chunk, int elems, int values, RowPlan* q) {
  q->chunk = chunk;
  if (chunk <= 32) {                   // several rows a warp, or one
    q->per_thread = 1;
    for (q->team = 1; q->team < chunk;) q->team *= 2;
    return;
  }
  q->per_thread = values / elems;
  q->team = ceil_div(chunk, 32 * q->per_thread) * 32;
}
// Rows of up to 1024 values take one warp each, which needs no barrier: the fewest values a thread
// then, or 0.  (30000 x 1001 bf16 backward: 46 us against 60 with two warps a row.)  The choice goes by
// the length of a row alone, not by the number of rows, so that a row's result does not depend on how
// many others there are; a few rows are served a little slower for it (2051 x 1000 fp32, fused forward
// and backward: 39 us against 34 with two warps).
inline int one_warp_values(int chunk, int elems) {
  int v = 2 * elems;
  while (v < 32 && chunk * elems > 32 * v) v *= 2;
  return chunk * elems <= 32 * v ? v : 0;
}
// 32 values a thread, or 16 where whole warps of 32 would leave a quarter more of their slots empty (1023
// 16-bit values that start inside a granule touch 129: one more than a warp's).
inline int wide_values(int chunk, int elems) {
  const int wide = ceil_div(chunk, 1024 / elems) * (1024 / elems), narrow = ceil_div(chunk, 512 / elems) * (512 / elems);
  return wide * 4 > narrow * 5 && narrow / (16 / elems) <= kMaxTeam ? 16 : 32;
}
inline int cta_threads(const RowPlan& q, int elems) { return q.per_thread * elems >= 32 ? kMaxThreadsWide : kMaxThreads; }

// Teams per CTA: at most `most`, or as few as give no team more rows than that would.
inline void plan_groups(size_t rows, int most, RowPlan* q) {
  q->groups = q->cluster > 1 || most < 1 ? 1 : most;
  if (q->team > 32 && q->groups > 15) q->groups = 15;        // named barriers
  const size_t sms = num_sms(), each = (rows + sms * q->groups - 1) / (sms * q->groups);
  q->groups = static_cast<int>((rows + sms * each - 1) / (sms * each));
  if (q->groups < 1) q->groups = 1;
  if (q->team < 32) q->groups = (q->groups + 32 / q->team - 1) / (32 / q->team) * (32 / q->team);    // whole warps
}

// The ring beside `params` bytes: as many rows ahead as fit, up to eight; false if not even `least`
// times the r rows between two barriers do.
inline bool plan_ring(size_t rows, int r, int ops, int least, size_t params, RowPlan* q) {
  const size_t stage = static_cast<size_t>(ceil_div(q->groups * q->team, 32)) * q->per_thread * ops * kUnit;
  if (params >= kSmemLimit) return false;
  const size_t deep = (kSmemLimit - params) / (r * stage);
  if (deep < static_cast<size_t>(least)) return false;
  const size_t teams = static_cast<size_t>(num_sms() / q->cluster > 0 ? num_sms() / q->cluster : 1) * q->groups;
  const size_t of_use = ((rows + teams - 1) / teams + r - 1) / r;      // no more than a team has rows, if every SM has a CTA
  int n = 8 / r;
  if (deep < static_cast<size_t>(n)) n = static_cast<int>(deep);
  if (of_use < static_cast<size_t>(n) && q->period == 1) n = static_cast<int>(of_use);
  q->stages = r * n;
  q->smem = stage * q->stages + params;
  return true;
}

inline bool plan_bwd_rows(size_t rows, size_t cols, int elem, int ops, bool from_y, RowPlan* q) {
  if (rows >> 30) return false;                              // row numbers are 32-bit, and some steps ahead
  const int elems = 16 / elem;
  const size_t most = row_granules(cols, elems, &q->period);
  if (most > static_cast<size_t>(kMaxTeam) * kMaxCluster * (32 / elems)) return false;
  for (q->cluster = 1; q->cluster <= kMaxCluster; q->cluster *= 2) {
    const int chunk = ceil_div(static_cast<long long>(most), q->cluster);
    // the fp32 weight (with from_y also minus the bias) lies beside the ring
    const size_t params_row = static_cast<size_t>(chunk) * elems * 4 * (from_y ? 2 : 1), row = static_cast<size_t>(chunk) * 16 * ops;
    const size_t deep = params_row < kSmemLimit ? (kSmemLimit - params_row) / row : 0;
    // What bounds these kernels is the bytes on their way: three rows a team where shared memory holds
    // six, so one is at work and two arrive, and as many values a thread as leave the CTA 512 threads
    // (fp32 8192 x 4096 with dsum: 129 us with one team of 512, 166 with two of 256; bf16 16384 x 4096:
    // 70 us with four teams of 128, 74 with three of 256).
    int teams = deep >= 6 ? static_cast<int>(deep / 3) : deep >= 5 ? 2 : 1, values = q->cluster > 1 ? 32 : one_warp_values(chunk, elems);
    if (!values) {
      values = wide_values(chunk, elems);
      while (values > 8 && values > 2 * elems && static_cast<long long>(chunk) * elems / values * teams < 512 &&
             static_cast<long long>(chunk) * elems * 2 / values <= kMaxTeam)
        values /= 2;
    }
    plan_team(chunk, elems, values, q);
    if (q->team > kMaxTeam) continue;
    const int r = bwd_rows_between_barriers(q->per_thread), fit = cta_threads(*q, elems) / q->team;
    const size_t params = q->per_thread == 1 ? 0 : static_cast<size_t>(q->team) * q->per_thread * elems * 4 * (from_y ? 2 : 1);
    for (teams = q->team <= 32 || teams > fit ? fit : teams; teams >= 1; --teams) {
      plan_groups(rows, teams, q);
      const size_t fold = q->groups > 1 ? static_cast<size_t>((q->groups + 1) / 2) * q->team * q->per_thread * elems * 2 * sizeof(float) : 0;
      if (fold <= kSmemLimit && plan_ring(rows, r, ops, 2, params, q)) {
        if (fold > q->smem) q->smem = fold;                  // the teams' column sums are folded there
        return true;
      }
    }
  }
  return false;
}

inline bool plan_fwd_rows(size_t rows, size_t cols, int elem, int ops, RowPlan* q) {
  if (rows >> 30) return false;
  const int elems = 16 / elem;
  const size_t most = row_granules(cols, elems, &q->period);
  if (most > static_cast<size_t>(kMaxTeam) * kMaxCluster * (32 / elems)) return false;
  for (q->cluster = 1; q->cluster <= kMaxCluster; q->cluster *= 2) {
    const int chunk = ceil_div(static_cast<long long>(most), q->cluster);
    int values = q->cluster > 1 ? 32 : one_warp_values(chunk, elems);
    if (!values) values = wide_values(chunk, elems);      // (16384 x 8192 bf16: 107 us with 32 against 154 with 16)
    plan_team(chunk, elems, values, q);
    if (q->team > kMaxTeam) continue;
    const int r = fwd_rows_between_barriers(q->per_thread);
    const size_t params = q->per_thread == 1 ? 0 : static_cast<size_t>(q->team) * q->per_thread * elems * 8;
    for (int teams = fwd_threads(q->per_thread, elems, ops == 2) / q->team; teams >= 1; --teams) {
      plan_groups(rows, teams, q);
      if (plan_ring(rows, r, ops, 2, params, q)) return true;
    }
  }
  return false;
}

// Long rows: `cluster` chunks of up to kMaxThreads threads with 16 values each, as many as use the SMs
// best.  `params` fp32 values of each column lie beside the ring.
inline bool plan_long(size_t rows, size_t cols, int elem, int ops, int params, RowPlan* q) {
  if (rows >> 30) return false;
  const int elems = 16 / elem, sms = num_sms();
  const size_t most = row_granules(cols, elems, &q->period);
  q->per_thread = 16 / elems;
  q->groups = 1;
  const int least = ceil_div(static_cast<long long>(most), static_cast<long long>(kMaxThreads) * q->per_thread);
  double best = 0.0;
  for (int n = least; n <= 2 * least; ++n) {
    const int unit = n * q->period, rounds = ceil_div(unit, sms);
    const double use = unit <= sms ? static_cast<double>(sms / unit * unit) / sms : static_cast<double>(unit) / (rounds * sms);
    if (use > best + 0.02) {
      best = use;
      q->cluster = n;
    }
  }
  q->chunk = ceil_div(static_cast<long long>(most), q->cluster);
  q->team = ceil_div(q->chunk, 32 * q->per_thread) * 32;
  if (q->team < 64) q->team = 64;                            // (a long row has far more)
  return plan_ring(rows, 1, ops, 1, static_cast<size_t>(q->team) * q->per_thread * elems * 4 * params, q);
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


inline int column_parts(const mb_ln_desc* d) {
  const size_t tiles = (d->cols + 31) / 32, groups = (d->rows + 7) / 8;
  size_t want = (static_cast<size_t>(num_sms()) * 8 + tiles - 1) / tiles;
  if (want > groups) want = groups;
  return static_cast<int>(want < 1 ? 1 : want > 1024 ? 1024 : want);
}


// Plan of the row kernel; one CTA per SM, so that there are few partial sums.
inline bool plan_bwd(const mb_ln_desc* d, int ops, bool from_y, RowPlan* q) {
  if (!plan_bwd_rows(d->rows, d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, from_y, q)) return false;
  size_grid(d->rows, 1, q);
  return true;
}

inline bool plan_bwd_long(const mb_ln_desc* d, int ops, bool from_y, RowPlan* q) {
  if (!plan_long(d->rows, d->cols, static_cast<int>(dtype_bytes(d->dtype)), ops, from_y ? 2 : 1, q)) return false;
  size_grid(d->rows, 1, q);
  return true;
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

// Launched while the kernel before it in the stream still runs; it waits for that one's end by itself
// (griddepcontrol.wait) before it touches memory.
template <typename... KArgs, typename... Args>
void launch_dependent(cudaLaunchConfig_t* cfg, void (*kernel)(KArgs...), Args... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attr;
  cfg->numAttrs = 1;
  cudaLaunchKernelEx(cfg, kernel, static_cast<KArgs>(args)...);
}

template <typename... KArgs, typename... Args>
int launch_rows(const char* who, int pass, void (*kernel)(KArgs...), const RowPlan& q, cudaStream_t st, Args... args) {
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
  cfg.numAttrs = pass == kCluster ? 1 : 0;
  if (pass == kApply) launch_dependent(&cfg, kernel, args...);
  else cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  return after_launch(who);
}

// A cluster's CTAs run together: a grid of more clusters than fit at once would end in a second,
// nearly empty round.  False if not even one fits this device.
template <typename Kernel>
bool fit_clusters(Kernel kernel, RowPlan* q) {
  if (q->cluster == 1) return true;
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
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) cudaGetLastError();
  if (n < 1) return false;
  n -= n % q->period;
  if (n >= q->period && q->grid > n * q->cluster) q->grid = n * q->cluster;
  return true;
}
constexpr int kDoesNotFit = -1;      // not a status: the caller takes another kernel

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
