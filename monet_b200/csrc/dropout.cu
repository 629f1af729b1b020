// Dropout from the counter-based generator (philox.cuh).  The backward is the same map applied to
// the gradient.  Bound by HBM: it reads and writes each element once.
#include "philox.cuh"
#include "types.cuh"

namespace mb {
namespace {

constexpr int kBlock = 256;

// One thread per block of eight elements; any alignment.
template <typename T>
__global__ void __launch_bounds__(kBlock) dropout_any(const T* x, T* y, size_t n, Drop d) {
  const unsigned long long key = d.on ? __ldg(d.seed) : 0;
  const size_t blocks = (n + 7) / 8;
  for (size_t b = static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x; b < blocks; b += static_cast<size_t>(gridDim.x) * kBlock) {
    const uint32_t keep = d.on ? keep8(key, b, d.stream, d.last) : 0xffu;
    const size_t i0 = b * 8;
    const int m = n - i0 < 8 ? static_cast<int>(n - i0) : 8;
    for (int j = 0; j < m; ++j) y[i0 + j] = from_f32<T>((keep >> j) & 1u ? to_f32(x[i0 + j]) * d.scale : 0.f);
  }
}

template <typename T>
int run(const void* x, void* y, size_t n, const Drop& d, cudaStream_t st) {
  const int grid = grid_for((n + 7) / 8, kBlock, 8);
  dropout_any<T><<<grid, kBlock, 0, st>>>(static_cast<const T*>(x), static_cast<T*>(y), n, d);
  return after_launch("dropout");
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" int mb_dropout(const void* x, void* y, size_t n, int dtype, const mb_dropout_desc* desc, void* stream) {
  const size_t e = dtype_bytes(dtype);
  if (!e) return fail(MB_ERR_INVALID_ARGUMENT, "mb_dropout: unknown dtype %d", dtype);
  if (!desc) return fail(MB_ERR_INVALID_ARGUMENT, "mb_dropout: null descriptor");
  Drop d;
  if (int rc = make_drop("mb_dropout", desc, &d)) return rc;
  if (n == 0) return MB_OK;
  if (!x || !y) return fail(MB_ERR_INVALID_ARGUMENT, "mb_dropout: null pointer");
  if (!aligned(x, e) || !aligned(y, e)) return fail(MB_ERR_INVALID_ARGUMENT, "mb_dropout: misaligned pointer");
  cudaStream_t st = as_stream(stream);
  if (dtype == MB_F32) return run<float>(x, y, n, d, st);
  if (dtype == MB_BF16) return run<__nv_bfloat16>(x, y, n, d, st);
  return run<__half>(x, y, n, d, st);
}
