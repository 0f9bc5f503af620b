// Short vectors of neighbouring channels: as they lie in memory, and in 32 bits.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace d3d {
namespace {

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// The channels of a thread in 32 bits; two at a time are worked on by packed instructions.
template <int V> struct alignas(V % 4 == 0 ? 16 : V % 2 == 0 ? 8 : 4) Vec { float v[V]; };
template <int V> __device__ __forceinline__ Vec<V> all(float x) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = x;
  return r;
}
template <int V> __device__ __forceinline__ float2 pair(const Vec<V>& a, int e) { return make_float2(a.v[e], a.v[e + 1]); }
template <int V> __device__ __forceinline__ Vec<V> fma(const Vec<V>& a, const Vec<V>& b, const Vec<V>& c) {
  Vec<V> r;
  if constexpr (V > 1)
#pragma unroll
    for (int e = 0; e < V / 2 * 2; e += 2) {
      const float2 t = __ffma2_rn(pair(a, e), pair(b, e), pair(c, e));
      r.v[e] = t.x, r.v[e + 1] = t.y;
    }
  if constexpr (V % 2) r.v[V - 1] = fmaf(a.v[V - 1], b.v[V - 1], c.v[V - 1]);
  return r;
}
template <int V> __device__ __forceinline__ Vec<V> mul(const Vec<V>& a, const Vec<V>& b) {
  Vec<V> r;
  if constexpr (V > 1)
#pragma unroll
    for (int e = 0; e < V / 2 * 2; e += 2) {
      const float2 t = __fmul2_rn(pair(a, e), pair(b, e));
      r.v[e] = t.x, r.v[e + 1] = t.y;
    }
  if constexpr (V % 2) r.v[V - 1] = a.v[V - 1] * b.v[V - 1];
  return r;
}
template <int V> __device__ __forceinline__ Vec<V> add(const Vec<V>& a, const Vec<V>& b) {
  Vec<V> r;
  if constexpr (V > 1)
#pragma unroll
    for (int e = 0; e < V / 2 * 2; e += 2) {
      const float2 t = __fadd2_rn(pair(a, e), pair(b, e));
      r.v[e] = t.x, r.v[e + 1] = t.y;
    }
  if constexpr (V % 2) r.v[V - 1] = a.v[V - 1] + b.v[V - 1];
  return r;
}
template <class T, int V> __device__ __forceinline__ Vec<V> widen(const Pack<T, V>& p) {
  Vec<V> r;
  if constexpr (V > 1 && sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[e / 2];
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        r.v[e] = __uint_as_float(w << 16), r.v[e + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        const float2 t = __half22float2(reinterpret_cast<const __half2&>(w));
        r.v[e] = t.x, r.v[e + 1] = t.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = to_f32(p.v[e]);
  }
  return r;
}
template <class T, int V> __device__ __forceinline__ Pack<T, V> narrow(const Vec<V>& x) {
  Pack<T, V> r;
  if constexpr (V > 1 && sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 t = pair(x, e);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) reinterpret_cast<__nv_bfloat162*>(&r)[e / 2] = __float22bfloat162_rn(t);
      else reinterpret_cast<__half2*>(&r)[e / 2] = __float22half2_rn(t);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = from_f32<T>(x.v[e]);
  }
  return r;
}

}  // namespace
}  // namespace d3d
