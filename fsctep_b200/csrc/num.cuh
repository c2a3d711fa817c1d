// Element types of the routed-expert operators: conversion, 16-byte vectors, packed 8-bit rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fsc {

struct e4m3 {
  uint8_t b;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as one access: 16 bytes (N = 16 / sizeof(T)) or one element (N = 1).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// Two floats to packed e4m3 (round to nearest even, finite values beyond the range saturate to
// +-448, NaN stays NaN); `a` in the low byte.
__device__ __forceinline__ uint16_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// Lets a kernel have up to `most` bytes of dynamic shared memory; false if it cannot.  The limit belongs to the kernel
// and not to a launch, and another thread may set it in between: `most` is the same constant in every call, whatever
// the launch takes of it.
template <typename K>
bool allow_shared(K kernel, size_t most) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) == cudaSuccess;
}

}  // namespace fsc
