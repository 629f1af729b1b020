// Counter-based dropout: which elements are dropped is a function of (seed, stream number,
// element index) alone, so a mask is never stored and a recomputed forward draws the same one.
//
// Element i belongs to block i / 8.  Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) keyed by the 64-bit seed turns the counter (block low,
// block high, stream, h) into four words = eight 16-bit halves, low half first.  Half i % 8 of
// h = 0 is the upper half of the element's 32-bit number u, that of h = 1 the lower half.  The
// element is dropped when u < round(p 2^32).  Comparing the upper halves decides all but one
// element in 65536, so the second evaluation (h = 1) runs on a tie only: the cost is ten rounds
// per eight elements, the resolution of p is 2^-32.
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

__device__ __forceinline__ uint4 philox(unsigned long long key, unsigned long long block, uint32_t stream, uint32_t h) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32), c2 = stream, c3 = h;
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = static_cast<unsigned long long>(0xD2511F53u) * c0;
    const unsigned long long b = static_cast<unsigned long long>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The ties of a block, decided by the lower halves: one block in 8192, so it is kept out of line.
static __device__ __noinline__ uint32_t keep8_ties(unsigned long long key, unsigned long long block, uint32_t stream, uint32_t last,
                                            uint4 q) {
  const uint4 s = philox(key, block, stream, 1);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w}, v[4] = {s.x, s.y, s.z, s.w};
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t hi = (w[j >> 1] >> (16 * (j & 1))) & 0xffffu, lo = (v[j >> 1] >> (16 * (j & 1))) & 0xffffu;
    if (hi == (last >> 16) && lo > (last & 0xffffu)) keep |= 1u << j;
  }
  return keep;
}

// Bit j of the result: element 8 * block + j is kept.
__device__ __forceinline__ uint32_t keep8(unsigned long long key, unsigned long long block, uint32_t stream, uint32_t last) {
  const uint4 q = philox(key, block, stream, 0);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  const uint32_t top = last | 0xffffu;          // upper half above last's upper half <=> word > top
  const uint32_t both = (last >> 16) * 0x10001u;
  uint32_t keep = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    keep |= ((w[j] << 16) > top ? 1u : 0u) << (2 * j);
    keep |= (w[j] > top ? 2u : 0u) << (2 * j);
    const uint32_t x = w[j] ^ both;             // a half that ties is zero here
    tie |= (x - 0x10001u) & ~x & 0x80008000u;
  }
  // `tie` is non-zero exactly when one of the eight halves ties
  if (tie && (last & 0xffffu) != 0xffffu) keep |= keep8_ties(key, block, stream, last, q);
  return keep;
}

__device__ __forceinline__ bool kept(const Drop& d, unsigned long long key, unsigned long long i) {
  return (keep8(key, i >> 3, d.stream, d.last) >> (i & 7)) & 1u;
}

}  // namespace mb
