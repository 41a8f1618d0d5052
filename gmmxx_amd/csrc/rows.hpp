// Shared helpers of the sparsely gated layer's kernels (layer_norm.hip, route.hip,
// grouped.hip, combine.hip): element types, 16-byte row access at any alignment and
// sums over groups of lanes.
#pragma once

#include "common.hpp"

namespace gx {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }

// Elements of one 16-byte load.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// V consecutive elements as fp32; elements at or past `valid` read as 0.  Whole
// vectors are one 16-byte load whatever the row's alignment; the last, partial one
// of an odd row is read element by element.
template <typename T>
__device__ __forceinline__ void load_row(const T* p, int valid, float (&v)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if (valid >= V) {
    union { uint4 u; T t[V]; } r;
    r.u = ld16_any(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(r.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < valid ? to_f32(p[i]) : 0.f;
  }
}

// The reverse of load_row: rounds to T (nearest even) and stores the first `valid`.
template <typename T>
__device__ __forceinline__ void store_row(T* p, int valid, const float (&v)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if (valid >= V) {
    union { u32x4_any u; T t[V]; } r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.t[i] = (T)v[i];
    *reinterpret_cast<u32x4_any*>(p) = r.u;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}

// Sum over aligned groups of G consecutive lanes (G a power of two up to 64), the
// same value and the same order of additions in every lane.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int off = G / 2; off >= 1; off /= 2) v += __shfl_xor(v, off);
  return v;
}

// Sum over groups of G threads: lanes_sum within a wave, `red` (two slots of 16
// floats, used in turn so that one barrier separates writers from readers) above it.
template <int G>
__device__ __forceinline__ float group_sum(float v, float (*red)[16], int& turn) {
  if constexpr (G <= 64) {
    return lanes_sum<G>(v);
  } else {
    v = lanes_sum<64>(v);
    float* slot = red[turn & 1];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) s += slot[w];
    return s;
  }
}

}  // namespace gx
