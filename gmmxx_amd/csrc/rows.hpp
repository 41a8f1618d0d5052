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

// The same as raw bytes; elements at or past `valid` are zeros.
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p, int valid) {
  constexpr int V = kVec<T>;
  union { uint4 u; T t[V]; } r;
  if (valid >= V) return ld16_any(p);
#pragma unroll
  for (int i = 0; i < V; ++i) r.t[i] = i < valid ? p[i] : (T)0.f;
  return r.u;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, int valid, uint4 v) {
  constexpr int V = kVec<T>;
  union { uint4 u; u32x4_any w; T t[V]; } r;
  r.u = v;
  if (valid >= V) {
    *reinterpret_cast<u32x4_any*>(p) = r.w;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = r.t[i];
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

// op(v, the value at distance D) within aligned groups of 2 D lanes whose halves each hold one value: the other
// half's value in every lane.  D up to 8 in one instruction with the operation (mirrored lanes), 16 and 32 by
// exchanging rows.
template <int D, typename F>
__device__ __forceinline__ float with_other(float v, F&& op) {
  if constexpr (D <= 8) {
    constexpr int kCtrl = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x140;   // quad_perm, half mirror, mirror
    const int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xF, 0xF, false);
    return op(v, __int_as_float(o));
  } else {
    const unsigned u = __float_as_uint(v);
    const auto r = D == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                           : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
}

// op over aligned groups of G consecutive lanes (G a power of two up to 64): the same value, by the same order
// of operations, in every lane of the group.  All 64 lanes take part.
template <int G, typename F>
__device__ __forceinline__ float lanes_reduce(float v, F&& op) {
  if constexpr (G > 1) v = with_other<1>(v, op);
  if constexpr (G > 2) v = with_other<2>(v, op);
  if constexpr (G > 4) v = with_other<4>(v, op);
  if constexpr (G > 8) v = with_other<8>(v, op);
  if constexpr (G > 16) v = with_other<16>(v, op);
  if constexpr (G > 32) v = with_other<32>(v, op);
  return v;
}
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_reduce<G>(v, [](float a, float b) { return a + b; });
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
