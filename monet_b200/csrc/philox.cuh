// Counter-based dropout: which elements are dropped is a function of (seed, stream number,
// element index) alone, so a mask is never stored and a recomputed forward draws the same one.
//
// Element i belongs to block i / 8.  Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) keyed by the 64-bit seed turns the counter (block low,
// block high, stream, h) into four words = eight 16-bit halves, low half first.  Half i % 8 of
// h = 0 is the upper half of the element's 32-bit number u, that of h = 1 the lower half.  The
// element is dropped when u < round(p 2^32).  The upper halves decide nearly always, so the second
// evaluation (h = 1) runs on a tie only: the cost is ten rounds per eight elements, the resolution
// of p is 2^-32.
#pragma once
#include "common.cuh"

namespace mb {

struct Drop {
  const unsigned long long* seed;   // device
  uint32_t stream;
  uint32_t last;                    // dropped when u <= last (last = round(p 2^32) - 1)
  float scale;                      // 1 / (1 - p); 0 for p = 1
  int on;                           // 0: nothing is dropped
};

// Fills `out` from the caller's descriptor (null: no dropout); an MB_* status.
inline int make_drop(const char* who, const mb_dropout_desc* d, Drop* out) {
  *out = Drop{nullptr, 0u, 0u, 1.f, 0};
  if (!d) return MB_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return fail(MB_ERR_INVALID_ARGUMENT, "%s: dropout probability must lie in [0, 1]", who);
  const unsigned long long t = static_cast<unsigned long long>(d->p * 4294967296.0 + 0.5);
  if (t == 0) return MB_OK;
  if (!d->seed || !aligned(d->seed, 8)) return fail(MB_ERR_INVALID_ARGUMENT, "%s: the dropout seed must be an 8-byte aligned device pointer", who);
  out->seed = reinterpret_cast<const unsigned long long*>(d->seed);
  out->stream = d->offset;
  out->last = static_cast<uint32_t>(t - 1);
  out->scale = d->p < 1.0 ? static_cast<float>(1.0 / (1.0 - d->p)) : 0.f;
  out->on = 1;
  return MB_OK;
}

// The words of N blocks.  The rounds of the blocks are interleaved: they share the key schedule and
// fill each other's latency.
template <int N>
__device__ __forceinline__ void philox(unsigned long long key, const unsigned long long (&block)[N], uint32_t stream, uint32_t h,
                                       uint32_t (&w)[N][4]) {
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    w[n][0] = static_cast<uint32_t>(block[n]);
    w[n][1] = static_cast<uint32_t>(block[n] >> 32);
    w[n][2] = stream;
    w[n][3] = h;
  }
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const unsigned long long a = static_cast<unsigned long long>(0xD2511F53u) * w[n][0];
      const unsigned long long b = static_cast<unsigned long long>(0xCD9E8D57u) * w[n][2];
      w[n][0] = static_cast<uint32_t>(b >> 32) ^ w[n][1] ^ k0;
      w[n][1] = static_cast<uint32_t>(b);
      w[n][2] = static_cast<uint32_t>(a >> 32) ^ w[n][3] ^ k1;
      w[n][3] = static_cast<uint32_t>(a);
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Which of a block's elements are dropped, as sign bits: bit 15 of d[j] for element 2j, bit 31 for
// element 2j + 1 (the other bits mean nothing).
//
// The upper 15 bits of two numbers are compared with the limit's by one subtraction, whose borrow
// bits are the answer unless a number ties; the most negative half, 0x8000, is the tie, so a running
// minimum finds whether there is one.  Then (one block in 4096) the whole numbers are compared.
struct Dropped { uint32_t d[4]; };

static __device__ __noinline__ uint4 dropped_by_whole_numbers(unsigned long long key, unsigned long long block, uint32_t stream,
                                                              uint32_t last, uint4 q) {
  uint32_t low[1][4];
  const unsigned long long one[1] = {block};
  philox<1>(key, one, stream, 1, low);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t d[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t even = w[j] << 16 | (low[0][j] & 0xffffu), odd = (w[j] & 0xffff0000u) | low[0][j] >> 16;
    d[j] = (even <= last ? 0x8000u : 0u) | (odd <= last ? 0x80000000u : 0u);
  }
  return make_uint4(d[0], d[1], d[2], d[3]);
}

template <int N>
__device__ __forceinline__ void dropped(const Drop& p, unsigned long long key, const unsigned long long (&block)[N], Dropped (&out)[N]) {
  uint32_t w[N][4];
  philox<N>(key, block, p.stream, 0, w);
  const uint32_t limit = (p.last >> 17) * 0x10001u | 0x80008000u;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t least = 0x7fff7fffu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[n].d[j] = limit - ((w[n][j] >> 1) & 0x7fff7fffu);
      least = __vmins2(least, out[n].d[j]);
    }
    const uint32_t tie = least ^ 0x80008000u;      // a half that is zero
    if (((tie - 0x10001u) & ~tie & 0x80008000u) && (p.last & 0x1ffffu) != 0x1ffffu) {
      const uint4 d = dropped_by_whole_numbers(key, block[n], p.stream, p.last, make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]));
      out[n].d[0] = d.x; out[n].d[1] = d.y; out[n].d[2] = d.z; out[n].d[3] = d.w;
    }
  }
}

// All ones where element 0 / 1 of a pair is dropped, else zero.
template <uint32_t SELECT>     // bytes 1 and 3 of d, their sign bits spread over bytes
__device__ __forceinline__ uint32_t spread_signs(uint32_t d) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(d), "n"(SELECT));
  return r;
}
__device__ __forceinline__ uint32_t sign_low(uint32_t d) { return spread_signs<0x9999>(d); }
__device__ __forceinline__ uint32_t sign_high(uint32_t d) { return spread_signs<0xbbbb>(d); }
__device__ __forceinline__ uint32_t sign_halves(uint32_t d) { return spread_signs<0xbb99>(d); }
__device__ __forceinline__ float zero_if(float v, uint32_t mask) { return __uint_as_float(__float_as_uint(v) & ~mask); }

// The sign bits of a block in one word, and back: unfold(x, j) stands for d[j].
__device__ __forceinline__ uint32_t fold(const Dropped& f) {
  return (f.d[0] & 0x80008000u) | (f.d[1] & 0x80008000u) >> 1 | (f.d[2] & 0x80008000u) >> 2 | (f.d[3] & 0x80008000u) >> 3;
}
__device__ __forceinline__ uint32_t unfold(uint32_t x, int j) { return x << j; }

// One element at a time.
__device__ __forceinline__ bool kept(const Drop& p, unsigned long long key, unsigned long long i) {
  const unsigned long long one[1] = {i >> 3};
  Dropped f[1];
  dropped<1>(p, key, one, f);
  return !(fold(f[0]) << ((i & 7) >> 1) & (i & 1 ? 0x80000000u : 0x8000u));
}

}  // namespace mb
