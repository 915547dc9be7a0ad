// bt_values.cuh -- the element types of the sampling and expert kernels as arithmetic values.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace btv {

template <class V>
struct Elem;

template <>
struct Elem<__half> {
  using T = __half;
  static __device__ __forceinline__ float to_float(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from_float(float v) { return __float2half_rn(v); }
};

template <>
struct Elem<__nv_bfloat16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to_float(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from_float(float v) { return __float2bfloat16_rn(v); }
};

template <>
struct Elem<float> {
  using T = float;
  static __device__ __forceinline__ float to_float(T v) { return v; }
  static __device__ __forceinline__ T from_float(float v) { return v; }
};

}  // namespace btv
