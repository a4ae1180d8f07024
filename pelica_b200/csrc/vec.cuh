// vec.cuh - V values of f32, f16 or bf16 memory as f32 registers: the streams of the row and norm operators. V values are one
// 16-byte access (the form for rows that start on 16 bytes) or one value (V = 1: every other width, stride and start).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

template <typename E> struct VecOf {
  static constexpr int N = 16 / sizeof(E);  // values of one 16-byte access
};

__device__ __forceinline__ float pm_to_f32(float v) { return v; }
__device__ __forceinline__ float pm_to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float pm_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename E> __device__ __forceinline__ E pm_from_f32(float v);
template <> __device__ __forceinline__ float pm_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half pm_from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 pm_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V values as they lie in memory
template <typename E, int V> struct alignas(V * sizeof(E) < 16 ? V * sizeof(E) : 16) Raw {
  E v[V];
};

template <typename E, int V> __device__ __forceinline__ Raw<E, V> pm_load(const E *p) {
  Raw<E, V> r;
  if constexpr (V * sizeof(E) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(E) / 16); i++) ((uint4 *)&r)[i] = ((const uint4 *)p)[i];
  } else {
    static_assert(V == 1, "one value or whole 16-byte words");
    r.v[0] = *p;
  }
  return r;
}
template <typename E, int V> __device__ __forceinline__ void pm_store(E *p, const Raw<E, V> &r) {
  if constexpr (V * sizeof(E) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(E) / 16); i++) ((uint4 *)p)[i] = ((const uint4 *)&r)[i];
  } else {
    *p = r.v[0];
  }
}
template <typename E, int V> __device__ __forceinline__ void pm_widen(const Raw<E, V> &r, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i++) f[i] = pm_to_f32(r.v[i]);
}
// to the stream's type: the one rounding of a result, to nearest
template <typename E, int V> __device__ __forceinline__ Raw<E, V> pm_narrow(const float (&f)[V]) {
  Raw<E, V> r;
#pragma unroll
  for (int i = 0; i < V; i++) r.v[i] = pm_from_f32<E>(f[i]);
  return r;
}
