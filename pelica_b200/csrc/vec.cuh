// vec.cuh - V values of f32, f16 or bf16 memory as f32 registers: the streams of the row and norm operators. V values are one
// 16-byte access (the form for rows that start on 16 bytes) or one value (V = 1: every other width, stride and start).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

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
// two neighbouring values as one f32x2 register pair, and back with the one rounding of a result (to nearest)
__device__ __forceinline__ uint64_t pm_widen2(const float *v) { return pm_pack2(v[0], v[1]); }
__device__ __forceinline__ uint64_t pm_widen2(const __half *v) {
  const float2 f = __half22float2(*(const __half2 *)v);
  return pm_pack2(f.x, f.y);
}
__device__ __forceinline__ uint64_t pm_widen2(const __nv_bfloat16 *v) {  // the upper half of an f32 each
  const uint32_t w = *(const uint32_t *)v;
  return pm_pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void pm_narrow2(float *o, float a, float b) { o[0] = a, o[1] = b; }
__device__ __forceinline__ void pm_narrow2(__half *o, float a, float b) { *(__half2 *)o = __floats2half2_rn(a, b); }
__device__ __forceinline__ void pm_narrow2(__nv_bfloat16 *o, float a, float b) { *(__nv_bfloat162 *)o = __floats2bfloat162_rn(a, b); }

template <typename E, int V> __device__ __forceinline__ Raw<E, V> pm_narrow(const float (&f)[V]) {
  Raw<E, V> r;
  if constexpr (V == 1) {
    r.v[0] = pm_from_f32<E>(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pm_narrow2(&r.v[i], f[i], f[i + 1]);
  }
  return r;
}

// one instruction works on a pair (each value rounded as by the scalar one)
__device__ __forceinline__ uint64_t pm_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pm_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// V f32 values, in pairs where there are any
template <int V> struct VecF {
  uint64_t p[V / 2];
};
template <> struct VecF<1> {
  float p[1];
};
template <typename E, int V> __device__ __forceinline__ VecF<V> vf_widen(const Raw<E, V> &r) {
  VecF<V> f;
  if constexpr (V == 1) f.p[0] = pm_to_f32(r.v[0]);
  else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) f.p[i] = pm_widen2(&r.v[2 * i]);
  }
  return f;
}
template <typename E, int V> __device__ __forceinline__ Raw<E, V> vf_narrow(const VecF<V> &f) {
  Raw<E, V> r;
  if constexpr (V == 1) r.v[0] = pm_from_f32<E>(f.p[0]);
  else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
      float a, b;
      pm_unpack2(f.p[i], a, b);
      pm_narrow2(&r.v[2 * i], a, b);
    }
  }
  return r;
}
template <int V> __device__ __forceinline__ VecF<V> vf_zero() {
  VecF<V> f;
#pragma unroll
  for (int i = 0; i < (V == 1 ? 1 : V / 2); i++) f.p[i] = 0;
  return f;
}
template <int V> __device__ __forceinline__ VecF<V> vf_mul(const VecF<V> &a, float s) {
  VecF<V> f;
  if constexpr (V == 1) f.p[0] = __fmul_rn(a.p[0], s);
  else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) f.p[i] = pm_mul2(a.p[i], pm_pack2(s, s));
  }
  return f;
}
template <int V> __device__ __forceinline__ void vf_add(VecF<V> &acc, const VecF<V> &a, float s) {
  if constexpr (V == 1) acc.p[0] = __fmaf_rn(a.p[0], s, acc.p[0]);
  else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) acc.p[i] = pm_fma2(a.p[i], pm_pack2(s, s), acc.p[i]);
  }
}
// running sums of a b: two, or one where V is one
template <int V> struct DotT { using T = uint64_t; };
template <> struct DotT<1> { using T = float; };
template <int V> using DotOf = typename DotT<V>::T;
template <int V> __device__ __forceinline__ void vf_dot_add(DotOf<V> &acc, const VecF<V> &a, const VecF<V> &b) {
  if constexpr (V == 1) acc = __fmaf_rn(a.p[0], b.p[0], acc);
  else {
#pragma unroll
    for (int i = 0; i < V / 2; i++) acc = pm_fma2(a.p[i], b.p[i], acc);
  }
}
__device__ __forceinline__ float vf_sum(float v) { return v; }
__device__ __forceinline__ float vf_sum(uint64_t v) {
  float a, b;
  pm_unpack2(v, a, b);
  return __fadd_rn(a, b);
}
// the arithmetic of whole vectors (pairs)
template <int N> __device__ __forceinline__ VecF<N> vf_all(float v) {
  VecF<N> f;
#pragma unroll
  for (int i = 0; i < N / 2; i++) f.p[i] = pm_pack2(v, v);
  return f;
}
template <int N> __device__ __forceinline__ VecF<N> operator*(const VecF<N> &a, const VecF<N> &b) {
  VecF<N> f;
#pragma unroll
  for (int i = 0; i < N / 2; i++) f.p[i] = pm_mul2(a.p[i], b.p[i]);
  return f;
}
template <int N> __device__ __forceinline__ VecF<N> operator*(const VecF<N> &a, float s) { return vf_mul<N>(a, s); }
template <int N> __device__ __forceinline__ VecF<N> operator+(const VecF<N> &a, const VecF<N> &b) {
  VecF<N> f;
#pragma unroll
  for (int i = 0; i < N / 2; i++) f.p[i] = pm_add2(a.p[i], b.p[i]);
  return f;
}
template <int N> __device__ __forceinline__ VecF<N> vf_fma(const VecF<N> &a, const VecF<N> &b, const VecF<N> &c) {
  VecF<N> f;
#pragma unroll
  for (int i = 0; i < N / 2; i++) f.p[i] = pm_fma2(a.p[i], b.p[i], c.p[i]);
  return f;
}
template <int N> __device__ __forceinline__ VecF<N> vf_fma(const VecF<N> &a, float s, const VecF<N> &c) { return vf_fma(a, vf_all<N>(s), c); }
template <int N> __device__ __forceinline__ float vf_dot(const VecF<N> &a, const VecF<N> &b) {
  uint64_t s = pm_mul2(a.p[0], b.p[0]);
#pragma unroll
  for (int i = 1; i < N / 2; i++) s = pm_fma2(a.p[i], b.p[i], s);
  return vf_sum(s);
}
