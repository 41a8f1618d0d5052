// Rows in 8-bit integers with a scale each, and products of such rows.
//
//   a = max |x|,  r = 127 (1 / a),  q = round(x r) (ties to even),  scale = a (1 / 127)
//   out[n][f] = (Σ_d qx[n][d] qw[f][d]) xs[n] ws[f] + bias[f]
//
// All in fp32, each operation rounded, the sum in exact 32-bit integers (D <= 2^17; the one sum that passes them, 2^31, is
// told from the others, see kPast).  The scales' product is formed
// first; where it may pass fp32's range on either side (see usual), the result is formed in 64 bits and rounded.  A row of zeros has scale 0; a
// row that holds a NaN or an infinity has scale NaN, so its products are NaN.  Where a is so
// small that r would pass fp32, both are taken times 2^100 first, which is exact.
//
// 16384 x 4096 x 8192: 485 to 585 us a product (1.9 to 2.3 POP/s), the longer the warmer the card.  What the operands are made of sets the
// clock: zeros take 357 us, and matrix instructions alone, from registers, give 4.9 POP/s on zeros and 3.5 on random
// values.  The rows in 8 bits: 35 to 50 us (201 MB).  4 x 4096 x 8192 in one kernel: 10 us (33.7 MB, 3.4 TB/s).

#include <math.h>

#include "grouped_tiles.hpp"
#include "tokens.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;

// --- quantisation ----------------------------------------------------------------

__device__ __forceinline__ float larger_bits(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// A row's factor and scale from the bits of its largest absolute value, and its values.
struct Scale {
  float lift, by, scale;
  bool finite;
  __device__ __forceinline__ explicit Scale(float top) {
    const uint32_t most = __float_as_uint(top);
    finite = most < 0x7f800000u;
    lift = top < 0x1p-100f ? 0x1p100f : 1.f;
    by = finite && most ? 1.f / (top * lift) * 127.f : 0.f;
    scale = finite ? top * (1.f / 127.f) : __uint_as_float(0x7fc00000u);
  }
  // Vector u of a row of n elements, of which `left` are left: zeros past them.
  template <typename T>
  __device__ __forceinline__ void store(int8_t* out, uint4 u, int left, int n) const {
    constexpr int V = kVec<T>;
    float v[V];
    unpack16<T>(n < V ? (left > 0 ? u : make_uint4(0, 0, 0, 0)) : keep16<false, T>(u, left, n), v);
    union { uint64_t u; uint32_t w; int8_t b[8]; } o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.b[i] = i < V && finite ? (int8_t)(int)rintf(v[i % V] * lift * by) : 0;
    if constexpr (V == 8) *reinterpret_cast<uint64_t*>(out) = o.u;
    else *reinterpret_cast<uint32_t*>(out) = o.w;
  }
};

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
    const Scale by(__uint_as_float(most));
    if (!there) continue;
    if (lane == 0) a.scales[n] = by.scale;
    int8_t* out = a.values + n * a.ldv;
    const auto store = [&](uint4 u, int c) { by.template store<T>(out + c, u, a.D - c, a.D); };
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
  // (workgroups that take several rows: 16384 x 4096 bf16 34.8 us, 37.9 with one for each four rows)
  quantize_kernel<T, G, NV, SHORT><<<(unsigned)(need < 2048 ? need : 2048), kThreads, 0, s>>>(a);
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

// --- a sum as a result -------------------------------------------------------------

// Scales of 0, NaN or between 2^-60 and 2^60: the product of two such has fp32's precision, times a whole number too.
// (& and |: without branches, 4 x 4096 x 8192 11.3 us a call, with them 11.5)
__device__ __forceinline__ bool usual(float s) {
  return !(fabsf(s) > 0x1p60f) & !((s != 0.f) & (fabsf(s) < 0x1p-60f));
}

// The 32 bits of -2^31 are a sum of 2^31: of 2^17 products all of (-128)^2; no sum is below -2^17 128 127.
constexpr int kPast = -0x7fffffff - 1;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 added(i32x4 a, i32x4 b) { return (i32x4)((u32x4)a + (u32x4)b); }   // (past 2^31 too)
__device__ __forceinline__ bool may_pass(int D) { return D == kQuantMaxD; }

__device__ __forceinline__ float scaled(int sum, float x, float w, float b) { return (float)sum * (x * w) + b; }
__device__ __forceinline__ float scaled_any(int sum, float x, float w, float b) {
  if (!usual(x) || !usual(w)) return (float)((sum == kPast ? 0x1p31 : (double)sum) * ((double)x * (double)w) + (double)b);
  return sum == kPast ? 0x1p31f * (x * w) + b : scaled(sum, x, w, b);
}

// --- products: tiles -------------------------------------------------------------

// A workgroup of WP x WQ waves forms a tile out[q][p], q over BQ rows of x and p over BP of w, by 32 x 32 x 32 MFMA with
// w first, so that a lane holds one row and four adjacent columns of the result at a time.  Both operands go
// straight into LDS in stages of DEEP bytes of the reduction, kStages of them in turn: the loads of three stages are in
// flight while one is multiplied.  Row r of a stage holds its 16-byte chunk c at c ^ place(r): the loads fill
// LDS in lane order, so each lane fetches the chunk that belongs at its place, and 16 lanes that read one chunk of
// consecutive rows take all 64 banks.
//
// Past the end of the reduction the last chunk is read again; the last stage's fragments are masked.  Rows and columns
// past the matrices are read from the last ones and not stored.
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kStages = 4;

template <int BP, int BQ, int WP, int WQ, int DEEP>
struct Tile {
  static constexpr int Waves = WP * WQ, Threads = 64 * Waves;
  static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;               // 32 x 32 tiles of a wave
  static constexpr int Chunks = DEEP / 16, Rows = 64 / Chunks;             // of a row; rows of a wave's load
  static constexpr int LP = BP / (Rows * Waves), LQ = BQ / (Rows * Waves); // loads of a lane and stage
  static constexpr int KK = DEEP / 32;                                     // products deep
  static constexpr int Bytes = (BP + BQ) * DEEP;                           // of a stage: w's rows, then x's
  static_assert(kStages == 4 && LP >= 1 && LQ >= 1 && KK % 2 == 0 && (DEEP == 64 || DEEP == 128), "");
  static_assert(Rows * Waves % 16 == 0, "a lane's rows agree in their places");
  __device__ static __forceinline__ int place(int r) { return DEEP == 64 ? r >> 2 & 3 : r >> 1 & 7; }

  struct Frags {
    i32x4 p[TP], q[TQ];
    // Part kk of a stage: 16 bytes of row lane % 32 of each 32, chunk 2 kk + lane / 32.
    __device__ __forceinline__ void read(const uint8_t* stage, int p0, int q0, int lane, int kk) {
      const int at = (lane & 31) * DEEP + (((2 * kk + (lane >> 5)) ^ place(lane)) << 4);
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] = *reinterpret_cast<const i32x4*>(stage + at + (p0 + 32 * i) * DEEP);
#pragma unroll
      for (int j = 0; j < TQ; ++j) q[j] = *reinterpret_cast<const i32x4*>(stage + at + (BP + q0 + 32 * j) * DEEP);
    }
    // Zeros past the first `left` of this lane's 16 (w's are enough).
    __device__ __forceinline__ void mask(int left) {
      i32x4 m;
#pragma unroll
      for (int d = 0; d < 4; ++d) m[d] = left >= 4 * d + 4 ? -1 : (left > 4 * d ? (1 << 8 * (left - 4 * d)) - 1 : 0);
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] &= m;
    }
    // between(n) is called after the n-th product.
    template <typename F>
    __device__ __forceinline__ void multiply(i32x16 (&acc)[TP][TQ], F&& between) const {
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(p[i], q[j], acc[i][j], 0, 0, 0);
          between(i * TQ + j);
        }
    }
  };
  // Loads spread over the products of a part of a stage: `of` of them from `first` on, by load(n).
  template <typename F>
  __device__ static __forceinline__ void spread(int product, int first, int of, F&& load) {
    constexpr int M = TP * TQ;
#pragma unroll
    for (int n = 0; n < of; ++n)
      if (product == (2 * n + 1) * M / (2 * of)) {
        __builtin_amdgcn_sched_barrier(0);
        load(first + n);
        __builtin_amdgcn_sched_barrier(0);
      }
  }

  // This wave's loads of the oldest of the three stages in flight are in LDS, its reads of the stage before it done;
  // then every wave's.
  __device__ static __forceinline__ void arrive() {
    constexpr int kLeft = 2 * (LP + LQ);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kLeft & 15) | (kLeft >> 4) << 14 | 0x70);      // vmcnt(kLeft) lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
  }

  // Sums over K > 0; load(s, stage, n) starts the n-th of a lane's LP + LQ loads of step s (any step: past the last,
  // anything in bounds).  Then store(piece) with a piece of the stages' LDS for each wave: room for
  // its part of the tile in 16 bits, and for 64 x 32 of it in fp32.
  template <typename F, typename G>
  __device__ static __forceinline__ void run(int K, F&& load, int wave, int lane, i32x16 (&acc)[TP][TQ], G&& store) {
    constexpr int L = LP + LQ;
    const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
    __shared__ __align__(16) uint8_t s0[Bytes], s1[Bytes], s2[Bytes], s3[Bytes];
    const int steps = (K + DEEP - 1) / DEEP;
#pragma unroll
    for (int n = 0; n < L; ++n) load(0, s0, n);
#pragma unroll
    for (int n = 0; n < L; ++n) load(1, s1, n);
#pragma unroll
    for (int n = 0; n < L; ++n) load(2, s2, n);
    Frags f[2];
    // A step: the fragments of its first part are read under the last products of the step before.  The loads of the
    // step after next but one are spread over the products: all at once they would hold up the waves that issue them
    // last (16384 x 4096 x 8192: 552 us so, 535 spread).
    auto step = [&](int s, const uint8_t* now, uint8_t* free, bool first, bool last) {
      arrive();
      f[0].read(now, p0, q0, lane, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const auto loads = [&](int n) { load(s + 3, free, n); };
        const int from = L * kk / KK, of = L * (kk + 1) / KK - from;
        if (kk == 0 && first) {
#pragma unroll
          for (int n = 0; n < L / KK; ++n) loads(n);
        } else {
          if (last && kk > 0) f[(kk + 1) & 1].mask(K - s * DEEP - 32 * (kk - 1) - 16 * (lane >> 5));
          f[(kk + 1) & 1].multiply(acc, [&](int m) { spread(m, from, of, loads); });
        }
        __builtin_amdgcn_sched_barrier(0);
        if (kk + 1 < KK) f[(kk + 1) & 1].read(now, p0, q0, lane, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    step(0, s0, s3, true, steps == 1);
    int s = 1;
    for (; s + 4 < steps; s += 4) {
      step(s, s1, s0, false, false);
      step(s + 1, s2, s1, false, false);
      step(s + 2, s3, s2, false, false);
      step(s + 3, s0, s3, false, false);
    }
    if (s < steps) step(s, s1, s0, false, s + 1 == steps);
    if (s + 1 < steps) step(s + 1, s2, s1, false, s + 2 == steps);
    if (s + 2 < steps) step(s + 2, s3, s2, false, s + 3 == steps);
    if (s + 3 < steps) step(s + 3, s0, s3, false, true);
    f[1].mask(K - (steps - 1) * DEEP - 32 * (KK - 1) - 16 * (lane >> 5));
    f[1].multiply(acc, [](int) {});
    // (loads past the last step may still be on their way into the stages)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70);
    __syncthreads();
    constexpr int Piece = 2 * BP * BQ / Waves > 8192 ? 2 * BP * BQ / Waves : 8192, PerStage = Bytes / Piece;
    static_assert(PerStage >= 1 && PerStage * kStages >= Waves, "every wave has room for its results");
    const int in = wave / PerStage;
    store((in == 0 ? s0 : in == 1 ? s1 : in == 2 ? s2 : s3) + wave % PerStage * Piece);
  }
};

// A wave's results, 64 columns by 32 TQ rows, times the rows' and the columns' scales, as whole 128-byte lines: through the
// wave's piece of LDS, from which 8 (16 for fp32) lanes take a row's 64 columns.  sw, bias and sx are the
// columns' and rows' own, in LDS; `cols` and `rows` of them exist.  ANY: scales and sums of any size.
template <bool ANY, typename O, int TQ>
__device__ __forceinline__ void store_products(uint8_t* piece, const i32x16 (&acc)[2][TQ], int lane, const float* sw,
                                               const float* bias, const float* sx, O* out, int64_t ld, int rows, int cols) {
  constexpr int Bytes = 64 * sizeof(O), Chunks = Bytes / 16;
  constexpr int Rows = 64 / Chunks;
  constexpr int Group = sizeof(O) == 2 || TQ == 1 ? TQ : TQ / 2;
#pragma unroll
  for (int j0 = 0; j0 < TQ; j0 += Group) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = 32 * i + 8 * v + 4 * (lane >> 5);
        const f32x4 w = *reinterpret_cast<const f32x4*>(sw + n), b = *reinterpret_cast<const f32x4*>(bias + n);
#pragma unroll
        for (int j = 0; j < Group; ++j) {
          typedef O vec __attribute__((ext_vector_type(4)));
          const float x = sx[32 * (j0 + j) + (lane & 31)];
          vec o;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int sum = acc[i][j0 + j][4 * v + c];
            o[c] = (O)(ANY ? scaled_any(sum, x, w[c], b[c]) : scaled(sum, x, w[c], b[c]));
          }
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
        if (32 * j0 + r < rows) store16(out + (32 * j0 + r) * ld + n, cols - n, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

constexpr int kBand = 4;      // (16384 x 4096 x 8192: 586 us, 603 by rows of tiles, 593 and 605 by 8 and 16)

template <typename O, int BP, int BQ, int WP, int WQ, int DEEP>
__global__ __launch_bounds__(64 * WP * WQ) void quant_tiles_kernel(QuantMatmulArgs a, int ntiles, int total) {
  typedef Tile<BP, BQ, WP, WQ, DEEP> C;
  const int id = block_id();
  if (id >= total) return;
  // An XCD's run of tiles goes through bands of kBand rows of tiles, column by column, so that the tiles at work
  // share rows and columns.
  const int tile = xcd_tile(id, total), mtiles = total / ntiles;
  const int band = tile / (kBand * ntiles), high = min(kBand, mtiles - band * kBand), in = tile - band * kBand * ntiles;
  const int64_t q0 = (int64_t)(band * kBand + in % high) * BQ, p0 = (int64_t)(in / high) * BP;
  const int rows = (int)(a.N - q0 < BQ ? a.N - q0 : BQ), cols = (int)(a.F - p0 < BP ? a.F - p0 : BP);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wp = (wave % WP) * (BP / WP), wq = (wave / WP) * (BQ / WQ);
  const int K = a.D, last = (K + 15) / 16 * 16 - 16;
  const uint8_t* w = reinterpret_cast<const uint8_t*>(a.w) + p0 * a.ldw;
  const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x) + q0 * a.ldx;
  // (a tile's rows lie at most 2^23 bytes apart: 32 bits hold their offsets)
  constexpr int Step = C::Rows * C::Waves;
  const int r = wave * C::Rows + lane / C::Chunks, chunk = (lane % C::Chunks ^ C::place(r)) * 16;
  uint32_t poff[C::LP], qoff[C::LQ];
#pragma unroll
  for (int i = 0; i < C::LP; ++i) poff[i] = (uint32_t)min(r + i * Step, cols - 1) * (uint32_t)a.ldw;
#pragma unroll
  for (int i = 0; i < C::LQ; ++i) qoff[i] = (uint32_t)min(r + i * Step, rows - 1) * (uint32_t)a.ldx;
  // The tile's scales and bias, in flight before everything else.
  __shared__ __align__(16) float sw[BP], sx[BQ], bias[BP];
  for (int i = threadIdx.x; i < BQ; i += C::Threads) sx[i] = a.xs[q0 + min(i, rows - 1)];
  for (int i = threadIdx.x; i < BP; i += C::Threads) {
    sw[i] = a.ws[p0 + min(i, cols - 1)];
    bias[i] = a.bias ? to_f32(static_cast<const O*>(a.bias)[p0 + min(i, cols - 1)]) : 0.f;
  }
  i32x16 acc[C::TP][C::TQ] = {};
  auto load = [&](int s, uint8_t* stage, int n) {
    const uint32_t k = (uint32_t)min(s * DEEP + chunk, last);
    stage += wave * 1024;
    if (n < C::LP) fetch_direct(w, poff[n] + k, stage + n * (C::Waves * 1024));
    else fetch_direct(x, qoff[n - C::LP] + k, stage + BP * DEEP + (n - C::LP) * (C::Waves * 1024));
  };
  auto store = [&](uint8_t* piece) {
    O* out = static_cast<O*>(a.out) + (q0 + wq) * a.F + p0 + wp;
    bool odd = may_pass(K) | !usual(sw[wp + lane]);     // (64 columns and BQ / WQ rows are this wave's)
    for (int r = lane; r < BQ / WQ; r += 64) odd |= !usual(sx[wq + r]);
    if (__builtin_expect(__any(odd), 0)) store_products<true>(piece, acc, lane, sw + wp, bias + wp, sx + wq, out, a.F, rows - wq, cols - wp);
    else store_products<false>(piece, acc, lane, sw + wp, bias + wp, sx + wq, out, a.F, rows - wq, cols - wp);
  };
  C::run(K, load, wave, lane, acc, store);
}

template <typename O, int BP, int BQ, int WP, int WQ, int DEEP>
void tiled(const QuantMatmulArgs& a, hipStream_t s) {
  const int64_t ntiles = (a.F + BP - 1) / BP, total = ntiles * ((a.N + BQ - 1) / BQ);
  quant_tiles_kernel<O, BP, BQ, WP, WQ, DEEP>
      <<<grid_of(total, 64 * WP * WQ), 64 * WP * WQ, 0, s>>>(a, (int)ntiles, (int)total);
}

// --- products: few rows ------------------------------------------------------------

// 16 NT columns a workgroup, by 16 x 16 x 64 MFMA with the matrix's rows first; its four waves take every fourth 64 of
// the reduction, for MT tiles of 16 rows of x (and the next 16 MT along y).
constexpr int kFewRows = 32;

// 16 bytes of the matrix's rows at reduction element k, zeros from K on.
__device__ __forceinline__ void mask_past(i32x4& p, int left) {
#pragma unroll
  for (int d = 0; d < 4; ++d) p[d] &= left >= 4 * d + 4 ? -1 : (left > 4 * d ? (1 << 8 * (left - 4 * d)) - 1 : 0);
}

// What a lane's four results of tile i (row n, columns f0 .. f0 + 3) are multiplied with, loaded ahead.
template <typename O>
struct Factors {
  float ws[4], b[4];
  __device__ __forceinline__ Factors(const QuantMatmulArgs& a, int64_t f0) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t f = f0 + c < a.F ? f0 + c : a.F - 1;
      ws[c] = a.ws[f];
      b[c] = a.bias ? to_f32(static_cast<const O*>(a.bias)[f]) : 0.f;
    }
  }
  __device__ __forceinline__ void store(const QuantMatmulArgs& a, i32x4 t, float sx, int64_t n, int64_t f0) const {
    if (n >= a.N) return;
    O o[4];
    const bool odd = may_pass(a.D) | !(usual(sx) & usual(ws[0]) & usual(ws[1]) & usual(ws[2]) & usual(ws[3]));
    if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = (O)scaled_any(t[c], sx, ws[c], b[c]);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = (O)scaled(t[c], sx, ws[c], b[c]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (f0 + c < a.F) static_cast<O*>(a.out)[n * a.F + f0 + c] = o[c];
  }
};

template <typename O, int MT, int NT>
__global__ __launch_bounds__(kThreads) void quant_few_kernel(QuantMatmulArgs a) {
  constexpr int W = kThreads / 64, U = 4;
  static_assert(MT * NT <= W, "a wave stores at most one tile");
  __shared__ i32x4 sums[W][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f0 = (int64_t)blockIdx.x * (16 * NT);
  const int K = a.D, last = (K + 15) / 16 * 16 - 16;
  const int r = lane & 15, kc = (lane >> 4) * 16;
  const int64_t n0 = (int64_t)blockIdx.y * (16 * MT);
  const int64_t row = n0 + 16 * (wave % MT) + r, col = f0 + 16 * (wave / MT % NT) + 4 * (lane >> 4);
  const Factors<O> factors(a, col);
  const float sx = a.xs[row < a.N ? row : a.N - 1];
  const int8_t *w[NT], *x[MT];
#pragma unroll
  for (int n = 0; n < NT; ++n) w[n] = a.w + (f0 + 16 * n + r < a.F ? f0 + 16 * n + r : a.F - 1) * a.ldw;
#pragma unroll
  for (int m = 0; m < MT; ++m) x[m] = a.x + (n0 + 16 * m + r < a.N ? n0 + 16 * m + r : a.N - 1) * a.ldx;
  i32x4 acc[NT][MT] = {};
  for (int k0 = wave * 64; k0 < K; k0 += W * 64 * U) {
    i32x4 p[U][NT], q[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(k0 + u * W * 64 + kc, last);
#pragma unroll
      for (int n = 0; n < NT; ++n) p[u][n] = *reinterpret_cast<const i32x4*>(w[n] + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) q[u][m] = *reinterpret_cast<const i32x4*>(x[m] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u * W * 64 + 64 > K) {                     // (the matrix's zeros are enough)
#pragma unroll
        for (int n = 0; n < NT; ++n) mask_past(p[u][n], K - (k0 + u * W * 64 + kc));
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[u][n], q[u][m], acc[n][m], 0, 0, 0);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wave][n * MT + m][lane] = acc[n][m];
  __syncthreads();
  if (wave < NT * MT) {
    i32x4 t = sums[0][wave][lane];
#pragma unroll
    for (int q = 1; q < W; ++q) t = added(t, sums[q][wave][lane]);
    factors.store(a, t, sx, row, col);
  }
}

// The same for up to 8 rows of x that are not in 8 bits yet: every workgroup brings them there itself, into LDS, while its
// first loads of the matrix are in flight.  G threads share a row, NV vectors each.
template <typename T, typename O, int NV>
__global__ __launch_bounds__(kThreads) void quant_few_rows_kernel(QuantArgs x, QuantMatmulArgs a, int G) {
  constexpr int W = kThreads / 64, U = 4, V = kVec<T>;
  extern __shared__ __align__(16) int8_t rows[];          // [N][padded + 16]: the odd 16 spread rows over the banks
  __shared__ i32x4 sums[W][64];
  __shared__ float scale[8], red[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t f0 = (int64_t)blockIdx.x * 16;
  const int K = a.D, last = (K + 15) / 16 * 16 - 16, ld = last + 32;
  const int r = lane & 15, kc = (lane >> 4) * 16;
  const int64_t col = f0 + 4 * (lane >> 4);
  const Factors<O> factors(a, col);
  const int8_t* w = a.w + (f0 + r < a.F ? f0 + r : a.F - 1) * a.ldw;
  i32x4 p[U];
  const auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) p[u] = *reinterpret_cast<const i32x4*>(w + min(k0 + u * W * 64 + kc, last));
  };
  // This thread's part of its row.
  const int n = threadIdx.x / G, l = threadIdx.x % G;
  const bool there = n < a.N;
  const T* src = static_cast<const T*>(x.x) + (there ? n : a.N - 1) * x.ldx;
  uint4 kept[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + l) * V;
    kept[i] = fetch16<false>(src + (c < K ? c : 0), c < K ? K - c : K);
  }
  fetch(wave * 64);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[V];
    unpack16<T>(keep16<false, T>(kept[i], K - (i * G + l) * V, K), v);
#pragma unroll
    for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  float top = __uint_as_float(most);
  if (G == 32) top = lanes_reduce<32>(top, larger_bits);
  else top = lanes_reduce<64>(top, larger_bits);
  if (G > 64) {
    if (lane == 0) red[wave] = top;
    __syncthreads();
    for (int q = 0; q < G / 64; ++q) top = larger_bits(top, red[wave / (G / 64) * (G / 64) + q]);
  }
  const Scale by(top);
  if (there) {
    if (l == 0) scale[n] = by.scale;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + l) * V;
      if (c < last + 16) by.template store<T>(rows + n * ld + c, kept[i], K - c, K);
    }
  }
  __syncthreads();
  const int8_t* q = rows + (r < a.N ? r : (int)a.N - 1) * ld;
  const float sx = scale[r < a.N ? r : (int)a.N - 1];
  i32x4 acc = {};
  for (int k0 = wave * 64; k0 < K; k0 += W * 64 * U) {
    if (k0 >= W * 64) fetch(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * W * 64;
      if (k + 64 > K) mask_past(p[u], K - (k + kc));
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(p[u], *reinterpret_cast<const i32x4*>(q + min(k + kc, last)), acc, 0, 0, 0);
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int i = 1; i < W; ++i) acc = added(acc, sums[i][lane]);
    factors.store(a, acc, sx, r, col);
  }
}

// Threads that share a row of x in it, 0 where rows are too many or too long: 16 vectors a thread.
int few_rows_threads(int64_t N, int D, int elem) {
  if (N > 8) return 0;
  const int V = elem == ELEM_F32 ? 4 : 8, G = N == 1 ? 256 : N == 2 ? 128 : N <= 4 ? 64 : 32;
  return D >= V && D <= 16 * V * G && N * (int64_t)(D + 32) <= 60000 ? G : 0;
}

template <typename T, typename O>
void few_rows_typed(const QuantArgs& x, const QuantMatmulArgs& a, int G, hipStream_t s) {
  const unsigned grid = (unsigned)((a.F + 15) / 16);
  const size_t lds = a.N * ((a.D + 15) / 16 * 16 + 16);
  const int need = ((a.D + kVec<T> - 1) / kVec<T> + G - 1) / G;
  if (need <= 2) quant_few_rows_kernel<T, O, 2><<<grid, kThreads, lds, s>>>(x, a, G);
  else if (need <= 8) quant_few_rows_kernel<T, O, 8><<<grid, kThreads, lds, s>>>(x, a, G);
  else quant_few_rows_kernel<T, O, 16><<<grid, kThreads, lds, s>>>(x, a, G);
}
template <typename T>
void few_rows_out(const QuantArgs& x, const QuantMatmulArgs& a, int G, hipStream_t s) {
  if (a.elem == ELEM_F32) few_rows_typed<T, float>(x, a, G, s);
  else if (a.elem == ELEM_BF16) few_rows_typed<T, __bf16>(x, a, G, s);
  else few_rows_typed<T, _Float16>(x, a, G, s);
}

template <typename O>
void matmul_typed(const QuantMatmulArgs& a, hipStream_t s) {
  // (Of more rows too, by groups of 32, where that gives no more workgroups than the card holds at once: their waves share
  // the reduction, which a tile goes through alone.  64 x 8192 x 2048 14 us against 19 by tiles, 256 x 8000 x 100 14 against
  // 18, 64 x 1024 x 2048 4.5 against 7; 128 x 8192 x 2048, twice as many, 25 against 19.)
  const int64_t groups = (a.F + 15) / 16 * ((a.N + kFewRows - 1) / kFewRows);
  if (a.N <= kFewRows || groups <= 256) {
    // 32 columns a workgroup halve what is read of x where there are enough of them: 32 x 4096 x 8192 11.2 and 14.8 us,
    // 32 x 1024 x 2048 5.2 and 4.5.
    const auto grid = [&](int n) {
      return dim3((unsigned)((a.F + 16 * n - 1) / (16 * n)), (unsigned)((a.N + kFewRows - 1) / kFewRows));
    };
    if (a.N <= 16) quant_few_kernel<O, 1, 1><<<grid(1), kThreads, 0, s>>>(a);
    else if (a.F < 4096) quant_few_kernel<O, 2, 1><<<grid(1), kThreads, 0, s>>>(a);
    else quant_few_kernel<O, 2, 2><<<grid(2), kThreads, 0, s>>>(a);
    return;
  }
  // The tiles that are expected to take least: so many rounds over the card of a start and so much for each 64 of the
  // reduction (us; measured at 16 and 64 of them, the largest tiles on a card that is not full run faster).
  // 2048 x 4096 x 4096: 49, 41 and 52 us by 256 x 256, 128 x 128 and 64 x 128; 3000 x 2048 x 3000: 30, 34, 40;
  // 512 x 4096 x 4096: 41, 20, 16; 5000 x 1000 x 5000: 40, 63, 82.
  const double steps = (a.D + 63) / 64;
  const auto cost = [&](int p, int q, double start, double step, double busy) {
    const double tiles = (double)(((a.F + p - 1) / p) * ((a.N + q - 1) / q));
    return ceil(tiles / 256) * (start + steps * (step + busy * fmin(1.0, tiles / 256)));
  };
  const double large = cost(256, 256, 6.0, 0.53, 0.42), small = cost(128, 64, 4.5, 0.17, 0.0);
  const double medium = cost(128, 128, 4.5, 0.26, 0.0);
  if (large <= medium && large <= small) tiled<O, 256, 256, 4, 2, 64>(a, s);
  else if (medium <= small) tiled<O, 128, 128, 2, 2, 128>(a, s);
  else tiled<O, 128, 64, 2, 2, 128>(a, s);
}

}  // namespace

void launch_quantize(const QuantArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) quantize_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) quantize_typed<__bf16>(a, s);
  else quantize_typed<_Float16>(a, s);
}

bool quant_linear_at_once(int64_t N, int D, int elem) { return few_rows_threads(N, D, elem) > 0; }

void launch_quant_linear(const QuantArgs& x, const QuantMatmulArgs& a, hipStream_t s) {
  if (const int G = few_rows_threads(a.N, a.D, x.elem)) {
    if (x.elem == ELEM_F32) few_rows_out<float>(x, a, G, s);
    else if (x.elem == ELEM_BF16) few_rows_out<__bf16>(x, a, G, s);
    else few_rows_out<_Float16>(x, a, G, s);
    return;
  }
  launch_quantize(x, s);
  launch_quant_matmul(a, s);
}

void launch_quant_matmul(const QuantMatmulArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) matmul_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) matmul_typed<__bf16>(a, s);
  else matmul_typed<_Float16>(a, s);
}

}  // namespace gx::layer
