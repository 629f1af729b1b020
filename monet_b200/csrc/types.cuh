// Element types of the operators that take 32- and 16-bit activations: conversion to and from the
// fp32 in which everything is computed.  A result is rounded once, to nearest even, when stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace mb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// A parameter (weight, bias) of either type it may have: fp32 or the activations'.
template <typename T>
__device__ __forceinline__ float param(const void* p, bool is_f32, size_t i) {
  return is_f32 ? __ldg(static_cast<const float*>(p) + i) : to_f32(static_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void put_param(void* p, bool is_f32, size_t i, float v) {
  if (is_f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = from_f32<T>(v);
}

inline size_t dtype_bytes(int dtype) { return dtype == MB_F32 ? 4 : (dtype == MB_BF16 || dtype == MB_F16) ? 2 : 0; }

}  // namespace mb
