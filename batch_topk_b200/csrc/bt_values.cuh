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
  // values q and q + 1 (q even) of a word
  static __device__ __forceinline__ void to_floats(const void* w, int q, float& a, float& b) {
    const float2 f = __half22float2(static_cast<const __half2*>(w)[q / 2]);
    a = f.x;
    b = f.y;
  }
  static __device__ __forceinline__ void from_floats(void* w, int q, float a, float b) {
    static_cast<__half2*>(w)[q / 2] = __floats2half2_rn(a, b);
  }
};

template <>
struct Elem<__nv_bfloat16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to_float(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from_float(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void to_floats(const void* w, int q, float& a, float& b) {
    const unsigned u = static_cast<const unsigned*>(w)[q / 2];
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xFFFF0000u);
  }
  static __device__ __forceinline__ void from_floats(void* w, int q, float a, float b) {
    static_cast<__nv_bfloat162*>(w)[q / 2] = __floats2bfloat162_rn(a, b);
  }
};

template <>
struct Elem<float> {
  using T = float;
  static __device__ __forceinline__ float to_float(T v) { return v; }
  static __device__ __forceinline__ T from_float(float v) { return v; }
  static __device__ __forceinline__ void to_floats(const void* w, int q, float& a, float& b) {
    a = static_cast<const float*>(w)[q];
    b = static_cast<const float*>(w)[q + 1];
  }
  static __device__ __forceinline__ void from_floats(void* w, int q, float a, float b) {
    static_cast<float*>(w)[q] = a;
    static_cast<float*>(w)[q + 1] = b;
  }
};

}  // namespace btv
