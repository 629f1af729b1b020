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
#include "philox.cuh"
#include "types.cuh"

namespace mb {
namespace {

struct LnArgs {
  const void *a, *b, *c;       // forward: x, residual; backward: dy, kept, dsum
  const void *w, *bias;
  void *out, *out2;            // forward: y, sum; backward: dv, dx
  float *mean, *rstd;          // written by the forward, read by the backward
  size_t rows, cols, ld_a, ld_b, ld_c;
  bool w_f32;                  // parameters are fp32 (else the activations' type)
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

// dw, db from `parts` partials per column.
template <typename T>
__global__ void __launch_bounds__(256) ln_bwd_finish(const float* partial, int parts, size_t cols, void* dw, void* db, bool w_f32) {
  __shared__ float sw[8][33], sb[8][33];
  const size_t col = static_cast<size_t>(blockIdx.x) * 32 + threadIdx.x;
  float aw = 0.f, ab = 0.f;
  if (col < cols)
    for (int k = threadIdx.y; k < parts; k += 8) {
      aw += partial[(static_cast<size_t>(k) * 2) * cols + col];
      ab += partial[(static_cast<size_t>(k) * 2 + 1) * cols + col];
    }
  sw[threadIdx.y][threadIdx.x] = aw;
  sb[threadIdx.y][threadIdx.x] = ab;
  __syncthreads();
  if (threadIdx.y == 0 && col < cols) {
    for (int k = 1; k < 8; ++k) {
      aw += sw[k][threadIdx.x];
      ab += sb[k][threadIdx.x];
    }
    if (dw) put_param<T>(dw, w_f32, col, aw);
    if (db) put_param<T>(db, w_f32, col, ab);
  }
}

int column_parts(const mb_ln_desc* d) {
  const size_t tiles = (d->cols + 31) / 32, groups = (d->rows + 7) / 8;
  size_t want = (static_cast<size_t>(num_sms()) * 8 + tiles - 1) / tiles;
  if (want > groups) want = groups;
  return static_cast<int>(want < 1 ? 1 : want > 1024 ? 1024 : want);
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

template <typename T>
int fwd(const LnArgs& p, cudaStream_t st) {
  ln_fwd_any<T><<<grid_for(p.rows, 1, 8), kBlock, 0, st>>>(p);
  return after_launch("layer_norm_fwd");
}

template <typename T, bool FROM_Y>
int bwd(const LnArgs& p, void* dw, void* db, float* ws, int parts, cudaStream_t st) {
  const int tiles = static_cast<int>((p.cols + 31) / 32);
  if (dw || db) {      // before the outputs, which may lie over the inputs
    ln_bwd_columns_any<T, FROM_Y><<<dim3(tiles, parts), dim3(32, 8), 0, st>>>(p, ws);
    if (int rc = after_launch("layer_norm_bwd_columns")) return rc;
    ln_bwd_finish<T><<<tiles, dim3(32, 8), 0, st>>>(ws, parts, p.cols, dw, db, p.w_f32);
    if (int rc = after_launch("layer_norm_bwd_finish")) return rc;
  }
  ln_bwd_any<T, FROM_Y><<<grid_for(p.rows, 1, 8), kBlock, 0, st>>>(p);
  return after_launch("layer_norm_bwd");
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
  LnArgs p{x, residual, nullptr, weight, bias, y, sum, mean, rstd, d->rows, d->cols, d->ld_a, d->ld_b, 0, d->param_dtype == MB_F32, d->eps, {}};
  if (int rc = make_drop(who, drop, &p.drop)) return rc;
  if (d->rows == 0) return MB_OK;
  if (!x || !y || !mean || !rstd) return fail(MB_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (drop && !residual) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout needs a residual", who);
  if (!natural(d, x) || !natural(d, residual) || !natural(d, y) || !natural(d, sum) || !natural_param(d, weight) ||
      !natural_param(d, bias) || !aligned(mean, 4) || !aligned(rstd, 4))
    return fail(MB_ERR_INVALID_ARGUMENT, "%s: misaligned pointer", who);
  cudaStream_t st = as_stream(stream);
  if (d->dtype == MB_F32) return fwd<float>(p, st);
  if (d->dtype == MB_BF16) return fwd<__nv_bfloat16>(p, st);
  return fwd<__half>(p, st);
}

size_t mb_layer_norm_workspace_bytes(const mb_ln_desc* d) {
  if (!d || d->cols == 0 || d->rows == 0) return 0;
  return static_cast<size_t>(column_parts(d)) * 2 * d->cols * sizeof(float);
}

int mb_layer_norm_bwd(const void* dy, const void* kept, int kept_is_output, const void* dsum, const void* weight,
                      const void* bias, const float* mean, const float* rstd, void* dv, void* dx, void* dweight,
                      void* dbias, const mb_ln_desc* d, const mb_dropout_desc* drop, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const char* who = "mb_layer_norm_bwd";
  if (int rc = check_desc(who, d)) return rc;
  LnArgs p{dy, kept, dsum, weight, bias, dv, dx, const_cast<float*>(mean), const_cast<float*>(rstd),
           d->rows, d->cols, d->ld_a, d->ld_b, d->ld_c, d->param_dtype == MB_F32, d->eps, {}};
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
  const int parts = column_parts(d);
  if ((dweight || dbias) && (!workspace || !aligned(workspace, 16) || workspace_bytes < mb_layer_norm_workspace_bytes(d)))
    return fail(MB_ERR_WORKSPACE, "%s: workspace too small or misaligned", who);
  float* ws = static_cast<float*>(workspace);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return kept_is_output ? bwd<T, true>(p, dweight, dbias, ws, parts, st) : bwd<T, false>(p, dweight, dbias, ws, parts, st);
  };
  if (d->dtype == MB_F32) return go(0.f);
  if (d->dtype == MB_BF16) return go(__nv_bfloat16{});
  return go(__half{});
}

}  // extern "C"
