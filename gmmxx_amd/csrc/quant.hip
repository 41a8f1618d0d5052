// Rows in 8-bit integers with a scale each, and products of such rows.
//
//   a = max |x|,  r = 127 / a,  q = round(x r) (ties to even),  scale = a / 127
//   out[n][f] = (Σ_d qx[n][d] qw[f][d]) xs[n] ws[f] + bias[f]
//
// All in fp32, the sum in exact 32-bit integers (D <= 2^17).  A row of zeros has scale 0; a
// row that holds a NaN or an infinity has scale NaN, so its products are NaN.  Where a is so
// small that 127 / a would pass fp32, both are taken times 2^100 first, which is exact.

#include <math.h>

#include "grouped_tiles.hpp"
#include "tokens.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 20;

// --- quantisation ----------------------------------------------------------------

__device__ __forceinline__ float larger_bits(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// A row by G threads, which keep its elements: NV vectors each.  0: any row, read twice.
template <typename T, int G, int NV, bool SHORT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(QuantArgs a) {
  constexpr int V = kVec<T>, R = kThreads / G, KEEP = NV ? NV : 1;
  __shared__ float red[kThreads / 64];
  const int lane = threadIdx.x % G;
  const int padded = (a.D + 15) / 16 * 16;
  for (int64_t n0 = (int64_t)blockIdx.x * R; n0 < a.N; n0 += (int64_t)gridDim.x * R) {
    const int64_t n = n0 + threadIdx.x / G;
    const bool there = n < a.N;
    const T* row = static_cast<const T*>(a.x) + (there ? n : a.N - 1) * a.ldx;
    uint32_t most = 0;       // (bits: a NaN is the largest, then an infinity)
    // vector c's elements, zeros past the row
    const auto fetch = [&](int c) { return fetch16<SHORT>(row + (c < a.D ? c : 0), c < a.D ? a.D - c : a.D); };
    const auto unpack = [&](uint4 u, int c, float (&v)[V]) { unpack16<T>(keep16<SHORT, T>(u, a.D - c, a.D), v); };
    uint4 kept[KEEP];
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) kept[i] = fetch((i * G + lane) * V);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float v[V];
        unpack(kept[i], (i * G + lane) * V, v);
#pragma unroll
        for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
      }
    } else {
      for (int c = lane * V; c < a.D; c += G * V) {
        float v[V];
        unpack(fetch(c), c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
      }
    }
    most = __float_as_uint(lanes_reduce<(G < 64 ? G : 64)>(__uint_as_float(most), larger_bits));
    if constexpr (G > 64) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __uint_as_float(most);
      __syncthreads();
      for (int w = 0; w < G / 64; ++w) most = max(most, __float_as_uint(red[w]));
    }
    const bool finite = most < 0x7f800000u;
    const float top = __uint_as_float(most), lift = top < 0x1p-100f ? 0x1p100f : 1.f;
    const float by = finite && most ? 127.f / (top * lift) : 0.f;
    if (!there) continue;
    if (lane == 0) a.scales[n] = finite ? top / 127.f : __uint_as_float(0x7fc00000u);
    int8_t* out = a.values + n * a.ldv;
    const auto store = [&](uint4 u, int c) {
      float v[V];
      unpack(u, c, v);
      union { uint64_t u; uint32_t w; int8_t b[8]; } o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.b[i] = i < V && finite ? (int8_t)(int)rintf(v[i % V] * lift * by) : 0;
      if constexpr (V == 8) *reinterpret_cast<uint64_t*>(out + c) = o.u;
      else *reinterpret_cast<uint32_t*>(out + c) = o.w;
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((i * G + lane) * V < padded) store(kept[i], (i * G + lane) * V);
    } else {
      for (int c = lane * V; c < padded; c += G * V) store(fetch(c), c);
    }
  }
}

template <typename T, int G, int NV, bool SHORT = false>
void quantize_shaped(const QuantArgs& a, hipStream_t s) {
  const int64_t need = (a.N + kThreads / G - 1) / (kThreads / G);
  quantize_kernel<T, G, NV, SHORT><<<(unsigned)(need < kMaxBlocks ? need : kMaxBlocks), kThreads, 0, s>>>(a);
}

template <typename T>
void quantize_typed(const QuantArgs& a, hipStream_t s) {
  const int nvec = (a.D + kVec<T> - 1) / kVec<T>;
  if (a.D < kVec<T>) quantize_shaped<T, 16, 1, true>(a, s);
  else if (nvec <= 32) quantize_shaped<T, 16, 2>(a, s);
  else if (nvec <= 128) quantize_shaped<T, 64, 2>(a, s);
  else if (nvec <= 256) quantize_shaped<T, 64, 4>(a, s);
  else if (nvec <= 512) quantize_shaped<T, 64, 8>(a, s);
  else if (nvec <= 2048) quantize_shaped<T, 256, 8>(a, s);
  else quantize_shaped<T, 256, 0>(a, s);
}

// --- products: tiles -------------------------------------------------------------

struct q8 { int8_t v; };
typedef int i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 multiply_add(q8, i32x4 a, i32x4 b, f32x16 c) {
  return __builtin_bit_cast(
      f32x16, __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, __builtin_bit_cast(i32x16, c), 0, 0, 0));
}

// A wave's results, 64 columns by 32 TQ rows, as store_tile: of integers, with the rows' and the columns' scales.
template <typename O, int TQ, typename S>
__device__ __forceinline__ void store_products(uint8_t* piece, const f32x16 (&acc)[2][TQ], int lane, const QuantMatmulArgs& a,
                                               int64_t row0, int rows, int64_t col0, S&& scale_of_row) {
  constexpr int Bytes = 64 * sizeof(O), Chunks = Bytes / 16;
  constexpr int Rows = 64 / Chunks;
  constexpr int Group = sizeof(O) == 2 || TQ == 1 ? TQ : TQ / 2;
  const int cols = (int)(a.F - col0 < 64 ? a.F - col0 : 64);
  float sw[2][16], b[2][16];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int n = 32 * i + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
      const int64_t f = col0 + (n < cols ? n : 0);
      sw[i][v] = cols > 0 ? a.ws[f] : 0.f;
      b[i][v] = cols > 0 && a.bias ? to_f32(static_cast<const O*>(a.bias)[f]) : 0.f;
    }
#pragma unroll
  for (int j0 = 0; j0 < TQ; j0 += Group) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = 32 * i + 8 * v + 4 * (lane >> 5);
#pragma unroll
        for (int j = 0; j < Group; ++j) {
          typedef O vec __attribute__((ext_vector_type(4)));
          const float sx = scale_of_row(j0 + j);
          vec o;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            o[c] = (O)((float)__float_as_int(acc[i][j0 + j][4 * v + c]) * (sx * sw[i][4 * v + c]) + b[i][4 * v + c]);
          const int r = 32 * j + (lane & 31), byte = n * (int)sizeof(O);
          *reinterpret_cast<vec*>(piece + r * Bytes + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15)) = o;
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int c = lane % Chunks, n = c * (16 / (int)sizeof(O));
    if (n < cols) {
#pragma unroll 4
      for (int r = lane / Chunks; r < 32 * Group; r += Rows) {
        const uint4 v = *reinterpret_cast<const uint4*>(piece + r * Bytes + ((c ^ (r & 7)) << 4));
        if (32 * j0 + r < rows) store16(static_cast<O*>(a.out) + (row0 + 32 * j0 + r) * a.F + col0 + n, cols - n, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <typename O, int B, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void quant_tiles_kernel(QuantMatmulArgs a, int ntiles, int total) {
  typedef Core<q8, true, true, B, B, WP, WQ> C;
  typedef typename C::P P;
  typedef typename C::Q Q;
  const int id = block_id();
  if (id >= total) return;
  const int tile = xcd_tile(id, total);
  const int64_t q0 = (int64_t)(tile / ntiles) * B, p0 = (int64_t)(tile % ntiles) * B;
  const int rows = (int)(a.N - q0 < B ? a.N - q0 : B), cols = (int)(a.F - p0 < B ? a.F - p0 : B);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wp = (wave % WP) * (B / WP), wq = (wave / WP) * (B / WQ);
  const int K = a.D, last = (K + 15) / 16 * 16 - 16;
  const int pc = P::column(), qc = Q::column();
  const uint8_t* w = reinterpret_cast<const uint8_t*>(a.w) + p0 * a.ldw;
  const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x) + q0 * a.ldx;
  // (256 rows of up to 2^17 bytes, and their strides: 32 bits where the host has checked)
  uint32_t poff[P::Loads], qoff[Q::Loads];
#pragma unroll
  for (int i = 0; i < P::Loads; ++i) poff[i] = (uint32_t)min(P::row(i), cols - 1) * (uint32_t)a.ldw;
#pragma unroll
  for (int i = 0; i < Q::Loads; ++i) qoff[i] = (uint32_t)min(Q::row(i), rows - 1) * (uint32_t)a.ldx;
  f32x16 acc[C::TP][C::TQ] = {};
  auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
    dp += wave * 1024;
    dq += wave * 1024;
    const uint32_t kp = (uint32_t)min(s * C::BK + pc, last), kq = (uint32_t)min(s * C::BK + qc, last);
#pragma unroll
    for (int i = 0; i < P::Loads; ++i) fetch_direct(w, poff[i] + kp, dp + i * (C::Threads * 16));
#pragma unroll
    for (int i = 0; i < Q::Loads; ++i) fetch_direct(x, qoff[i] + kq, dq + i * (C::Threads * 16));
  };
  auto store = [&](uint8_t* piece) {
    store_products<O>(piece, acc, lane, a, q0 + wq, rows - wq, p0 + wp,
                      [&](int j) { return a.xs[q0 + min(wq + 32 * j + (lane & 31), rows - 1)]; });
  };
  C::run(K, fill, wave, lane, acc, store);
}

template <typename O, int B, int WP, int WQ>
void tiled(const QuantMatmulArgs& a, hipStream_t s) {
  const int64_t ntiles = (a.F + B - 1) / B, total = ntiles * ((a.N + B - 1) / B);
  quant_tiles_kernel<O, B, WP, WQ><<<grid_of(total, 64 * WP * WQ), 64 * WP * WQ, 0, s>>>(a, (int)ntiles, (int)total);
}

// --- products: few rows ------------------------------------------------------------

// 16 columns a workgroup, by 16 x 16 x 64 MFMA with the matrix's rows first; its four waves take every fourth 64 of
// the reduction, MT tiles of 16 rows of x at a time.
constexpr int kFewRows = 64;
template <typename O, int MT>
__global__ __launch_bounds__(kThreads) void quant_few_kernel(QuantMatmulArgs a) {
  constexpr int W = kThreads / 64, U = 4;
  typedef int i32x4v __attribute__((ext_vector_type(4)));
  __shared__ i32x4v sums[W][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f0 = (int64_t)blockIdx.x * 16;
  const int K = a.D, last = (K + 15) / 16 * 16 - 16;
  const int r = lane & 15, kc = (lane >> 4) * 16;
  const int8_t* w = a.w + (f0 + r < a.F ? f0 + r : a.F - 1) * a.ldw;
  const int8_t* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = a.x + (16 * m + r < a.N ? 16 * m + r : a.N - 1) * a.ldx;
  i32x4v acc[MT] = {};
  for (int k0 = wave * 64; k0 < K; k0 += W * 64 * U) {
    i32x4 p[U], q[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * W * 64 + kc;
      p[u] = *reinterpret_cast<const i32x4*>(w + min(k, last));
#pragma unroll
      for (int m = 0; m < MT; ++m) q[u][m] = *reinterpret_cast<const i32x4*>(x[m] + min(k, last));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int left = K - (k0 + u * W * 64 + kc);        // (the matrix's zeros are enough)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        p[u][d] &= left >= 4 * d + 4 ? -1 : (left > 4 * d ? (1 << 8 * (left - 4 * d)) - 1 : 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[u], q[u][m], acc[m], 0, 0, 0);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) sums[wave][m][lane] = acc[m];
  __syncthreads();
  for (int m = wave; m < MT; m += W) {
    i32x4v t = sums[0][m][lane];
#pragma unroll
    for (int q = 1; q < W; ++q) t += sums[q][m][lane];
    const int64_t n = 16 * m + r;
    if (n >= a.N) continue;
    const float sx = a.xs[n];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t f = f0 + 4 * (lane >> 4) + c;
      if (f >= a.F) break;
      const float b = a.bias ? to_f32(static_cast<const O*>(a.bias)[f]) : 0.f;
      static_cast<O*>(a.out)[n * a.F + f] = (O)((float)t[c] * (sx * a.ws[f]) + b);
    }
  }
}

template <typename O>
void matmul_typed(const QuantMatmulArgs& a, hipStream_t s) {
  if (a.N <= kFewRows) {
    const unsigned grid = (unsigned)((a.F + 15) / 16);
    if (a.N <= 16) quant_few_kernel<O, 1><<<grid, kThreads, 0, s>>>(a);
    else if (a.N <= 32) quant_few_kernel<O, 2><<<grid, kThreads, 0, s>>>(a);
    else quant_few_kernel<O, 4><<<grid, kThreads, 0, s>>>(a);
    return;
  }
  if (((a.N + 255) / 256) * ((a.F + 255) / 256) >= 256) tiled<O, 256, 4, 2>(a, s);
  else tiled<O, 128, 2, 2>(a, s);
}

}  // namespace

void launch_quantize(const QuantArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) quantize_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) quantize_typed<__bf16>(a, s);
  else quantize_typed<_Float16>(a, s);
}

void launch_quant_matmul(const QuantMatmulArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) matmul_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) matmul_typed<__bf16>(a, s);
  else matmul_typed<_Float16>(a, s);
}

}  // namespace gx::layer
