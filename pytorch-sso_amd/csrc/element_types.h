// Tensors of float32, bfloat16 or float16 elements, worked on in float32.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace kfac {

enum { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };      // `type` of the entry points
inline size_t type_size(int type) { return type == TYPE_F32 ? 4 : 2; }

template <class V> struct Element;
template <> struct Element<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Element<__hip_bfloat16> {
  static __device__ __forceinline__ float get(__hip_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __hip_bfloat16 put(float v) { return __float2bfloat16(v); }
};
template <> struct Element<_Float16> {
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};

// N elements in one access
template <class V, int N>
struct alignas(sizeof(V) * N) Pack {
  V v[N];
};

}  // namespace kfac
