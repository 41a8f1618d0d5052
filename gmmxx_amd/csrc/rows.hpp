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

// 16 bytes of a row of n elements, of which `valid` are left from p on, whatever the row's alignment: one load
// without a branch, so that several are in flight together.  Near the row's end it takes the row's last 16
// bytes instead, which keep16 moves to their place.  SHORT: n is less than a vector; element by element.
template <bool SHORT, typename T>
__device__ __forceinline__ uint4 fetch16(const T* p, int valid) {
  constexpr int V = kVec<T>;
  if constexpr (!SHORT) return ld16_any(valid >= V ? p : p + (valid - V));
  union { uint4 u; T t[V]; } r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.t[i] = i < valid ? p[i] : (T)0.f;
  return r.u;
}

// What fetch16 loaded, with zeros at elements at or past `valid`.
template <bool SHORT, typename T>
__device__ __forceinline__ uint4 keep16(uint4 u, int valid, int n) {
  constexpr int V = kVec<T>;
  if constexpr (SHORT) return valid > 0 ? u : make_uint4(0, 0, 0, 0);
  if (n % V == 0) return valid > 0 ? u : make_uint4(0, 0, 0, 0);
  if (valid >= V) return u;
  const int bytes = valid > 0 ? (V - valid) * (int)sizeof(T) : 16, words = bytes >> 2;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t t[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    t[i] = 0;
#pragma unroll
    for (int s = 0; s + i < 4; ++s) t[i] = words == s ? w[s + i] : t[i];
  }
  if constexpr (sizeof(T) == 2) {
    const int bits = (bytes & 2) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __builtin_amdgcn_alignbit(t[i + 1], t[i], bits);
  }
  return make_uint4(t[0], t[1], t[2], t[3]);
}

// The elements of 16 bytes as fp32.
template <typename T>
__device__ __forceinline__ void unpack16(uint4 u, float (&v)[kVec<T>]) {
  union { uint4 u; T t[kVec<T>]; } r;
  r.u = u;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) v[i] = to_f32(r.t[i]);
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

// Rounds to T (nearest even) and stores the first `valid`.
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
// of operations, in every lane of the group.  A group's lanes take part together; no exchange crosses a group, so
// other groups of the wave may have left.
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

// Sums of N values over groups of G threads: lanes_sum within a wave, `red` (two slots of 16 waves' values, used
// in turn so that one barrier separates writers from readers) above it, of which each lane reads one wave's.
template <int G, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float (*red)[16][N], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(G < 64 ? G : 64)>(v[i]);
  if constexpr (G > 64) {
    float(*slot)[N] = red[turn & 1];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[threadIdx.x >> 6][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<G / 64>(slot[threadIdx.x % (G / 64)][i]);
  }
}

}  // namespace gx
