// Tiles of the grouped products by MFMA (see grouped.hip for the mathematics); one translation unit for each
// element type instantiates them.
//
// A workgroup forms a tile out[q][p], q over BQ rows and p over BP columns, by 32 x 32 MFMA (16 deep for
// 16-bit elements, 2 deep for fp32) with the column operand first, so that a lane holds one row and four
// adjacent columns of the result.  Both operands are staged 128 bytes deep in LDS, two buffers in turn: the
// next steps' loads are in flight while a step's products run.  An operand whose reduction index is adjacent
// in memory lies in LDS as [row][BK] and is read 16 bytes a lane; one whose reduction index is not (a weight
// read along its other dimension, both operands of the weight's gradient) lies as [BK][row] and is read by
// the transposing LDS loads (16 bits) or a word at a time (fp32): no copy of either is ever transposed in
// memory.
//
// DIRECT: operands in whole, aligned 16-byte chunks are loaded straight into LDS.  Such a load fills LDS in
// lane order, so the order of chunks that keeps the reads free of bank conflicts is made by which chunk each
// lane fetches: chunk c of row r sits at c ^ (r & 7), a 32-byte pair u of reduction row k at u ^ (k & 7).
// Any other width, stride or alignment goes through registers, a step further ahead, to the same places.
//
// Ragged ends: rows past a group's end are read from its last row and not stored, columns past the matrix
// likewise; past the end of the reduction its last elements are read again (or zeros) and masked in registers.
#pragma once

#include <math.h>

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// A fragment: the V reduction elements 2 V kk + V (lane / 32) + 0 .. V - 1 of a row, 16 bytes.
template <typename T>
struct Elem16 {
  static constexpr int V = kVec<T>, BK = 128 / (int)sizeof(T), KK = BK / (2 * V);
};

__device__ __forceinline__ f32x16 multiply_add(bf16_t, i32x4 a, i32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply_add(_Float16, i32x4 a, i32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply_add(float, i32x4 a, i32x4 b, f32x16 c) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(f32x4, a)[s], __builtin_bit_cast(f32x4, b)[s], c, 0, 0, 0);
  return c;
}

// 16 bytes a lane from base + off to the wave's 1024 bytes of LDS at `dst`, in lane order.  With a
// 32-bit off and one base for the wave the address takes no vector arithmetic.
template <typename O>
__device__ __forceinline__ void fetch_direct(const uint8_t* base, O off, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(base + off),
                                   (__attribute__((address_space(3))) uint32_t*)dst, 16, 0, 0);
}

// Where a lane reads its fragments of one operand's tile of R rows: N of them, of rows r0 + 32 i + lane % 32.
template <typename T, bool KC, int R, int N>
struct Reader;

template <typename T, int R, int N>
struct Reader<T, true, R, N> {
  static constexpr int KK = Elem16<T>::KK;
  int at[KK];            // of i = 0, for each kk
  __device__ __forceinline__ Reader(int r0, int lane) {
    const int r = r0 + (lane & 31);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) at[kk] = r * 128 + (((2 * kk + (lane >> 5)) ^ (r & 7)) << 4);
  }
  __device__ __forceinline__ i32x4 get(const uint8_t* tile, int i, int kk) const {
    return *reinterpret_cast<const i32x4*>(tile + at[kk] + i * (32 * 128));
  }
};

template <typename T, int R, int N>
struct Reader<T, false, R, N> {
  int lo[N], hi[N];      // of kk = 0, for each i: reduction elements 0..3 and 4..7
  __device__ __forceinline__ Reader(int r0, int lane) {
    // lanes of a 16-lane group: reduction row (lane / 4) % 4, 8-byte piece lane % 4 of its 32 bytes
    const int k = 8 * (lane >> 5) + ((lane >> 2) & 3);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int u = (r0 >> 4) + 2 * i + ((lane >> 4) & 1);
      lo[i] = k * (R * 2) + ((u ^ (k & 7)) << 5) + (lane & 3) * 8;
      hi[i] = (k + 4) * (R * 2) + ((u ^ ((k + 4) & 7)) << 5) + (lane & 3) * 8;
    }
  }
  __device__ __forceinline__ i32x4 get(const uint8_t* tile, int i, int kk) const {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + lo[i] + kk * (16 * R * 2)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + hi[i] + kk * (16 * R * 2)));
    return __builtin_bit_cast(i32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

template <int R, int N>
struct Reader<float, false, R, N> {
  int at;
  __device__ __forceinline__ Reader(int r0, int lane) { at = (lane >> 5) * (4 * R * 4) + (r0 + (lane & 31)) * 4; }
  __device__ __forceinline__ i32x4 get(const uint8_t* tile, int i, int kk) const {
    i32x4 v;
#pragma unroll
    for (int s = 0; s < 4; ++s) v[s] = *reinterpret_cast<const int*>(tile + at + (kk * 8 + s) * (R * 4) + i * 128);
    return v;
  }
};

// A thread's share of the loads of an operand's tile: R rows by BK of the reduction.
template <typename T, bool KC, int R, int THREADS>
struct Share {
  static constexpr int V = kVec<T>;
  static constexpr int Loads = R * 128 / (THREADS * 16);
  static constexpr int PerRow = KC ? 8 : R / V;               // chunks of a row of the tile
  static constexpr int Step = THREADS / PerRow;               // tile rows between a thread's loads
  static_assert(Loads >= 1 && (Step % 8 == 0 || (!KC && sizeof(T) == 4)), "a thread's rows agree modulo 8");
  // Tile row of load i: a row of the operand (KC) or a reduction row.
  __device__ static __forceinline__ int row(int i) { return threadIdx.x / PerRow + i * Step; }
  // First element of the thread's chunk along the tile row.
  __device__ static __forceinline__ int column() {
    const int c = threadIdx.x % PerRow, r = row(0);
    if constexpr (KC) return (c ^ (r & 7)) * V;
    else if constexpr (sizeof(T) == 2) return ((((c >> 1) ^ (r & 7)) << 1) | (c & 1)) * V;
    else return c * V;
  }
};

// Byte offsets from an operand's first element.
template <bool WIDE> struct Offset { typedef uint32_t type; };
template <> struct Offset<true> { typedef int64_t type; };

template <typename T, bool PKC, bool QKC, int BP, int BQ, int WP, int WQ>
struct Core {
  static constexpr int V = Elem16<T>::V, BK = Elem16<T>::BK, KK = Elem16<T>::KK;
  static constexpr int Threads = 64 * WP * WQ;
  static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;    // 32 x 32 tiles of a wave
  typedef Share<T, PKC, BP, Threads> P;
  typedef Share<T, QKC, BQ, Threads> Q;
  typedef Reader<T, PKC, BP, TP> RP;
  typedef Reader<T, QKC, BQ, TQ> RQ;
  struct Frags {
    i32x4 p[TP], q[TQ];
    __device__ __forceinline__ void read(const uint8_t* tp, const uint8_t* tq, const RP& rp, const RQ& rq, int kk) {
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] = rp.get(tp, i, kk);
#pragma unroll
      for (int j = 0; j < TQ; ++j) q[j] = rq.get(tq, j, kk);
    }
    // Zeros at reduction elements past the first `left` of this lane's V.
    __device__ __forceinline__ void mask(int left) {
      i32x4 m;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        m[d] = sizeof(T) == 4 ? (left > d ? -1 : 0) : left >= 2 * d + 2 ? -1 : (left == 2 * d + 1 ? 0xffff : 0);
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] &= m;
#pragma unroll
      for (int j = 0; j < TQ; ++j) q[j] &= m;
    }
    __device__ __forceinline__ void multiply(f32x16 (&acc)[TP][TQ]) const {
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = multiply_add(T(), p[i], q[j], acc[i][j]);
    }
  };

  // Every wave's loads are in LDS and every wave has read its last fragments.
  __device__ static __forceinline__ void arrive() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70);     // vmcnt(0) lgkmcnt(0), in a form that the compiler counts with
    asm volatile("s_barrier" ::: "memory");
  }

  // Sums over `total` > 0 reduction elements in steps of BK; fill(step, p, q) starts the loads of a step,
  // reading past the last element anything that is in bounds.
  //
  // One barrier a step, before the last of its products: by then every fragment of the step is in
  // registers, so its buffer takes the loads of the step after next, and the next step's first fragments
  // are read under those last products.  The last step's fragments are masked.
  // Then store(piece) is called with a piece of the stages' LDS for each wave: room for the wave's part of the
  // tile in 16 bits (256 x 32: in fp32).
  template <typename F, typename G>
  __device__ static __forceinline__ void run(int total, F&& fill, int wave, int lane, f32x16 (&acc)[TP][TQ],
                                             G&& store) {
    const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
    __shared__ __align__(16) uint8_t pa[BP * 128], pb[BP * 128], qa[BQ * 128], qb[BQ * 128];
    const RP rp(p0, lane);
    const RQ rq(q0, lane);
    const int last = (total - 1) / BK;
    Frags f[2];
    fill(0, pa, qa);
    arrive();
    if (last > 0) fill(1, pb, qb);
    f[0].read(pa, qa, rp, rq, 0);
    auto step = [&](int s, uint8_t* p, uint8_t* q, uint8_t* p_next, uint8_t* q_next) {
#pragma unroll
      for (int kk = 0; kk + 1 < KK; ++kk) {
        f[(kk + 1) & 1].read(p, q, rp, rq, kk + 1);
        __builtin_amdgcn_sched_barrier(0);
        f[kk & 1].multiply(acc);
        __builtin_amdgcn_sched_barrier(0);
      }
      arrive();
      if (s + 2 <= last) fill(s + 2, p, q);
      f[0].read(p_next, q_next, rp, rq, 0);
      __builtin_amdgcn_sched_barrier(0);
      f[(KK - 1) & 1].multiply(acc);
      __builtin_amdgcn_sched_barrier(0);
    };
    int s = 0;
    for (; s + 2 <= last; s += 2) {
      step(s, pa, qa, pb, qb);
      step(s + 1, pb, qb, pa, qa);
    }
    if (s < last) step(s, pa, qa, pb, qb);
    const uint8_t* p = last & 1 ? pb : pa;
    const uint8_t* q = last & 1 ? qb : qa;
    const int left = total - last * BK - V * (lane >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if (kk + 1 < KK) f[(kk + 1) & 1].read(p, q, rp, rq, kk + 1);
      __builtin_amdgcn_sched_barrier(0);
      if (total - last * BK > 2 * V * kk) {
        f[kk & 1].mask(left - 2 * V * kk);
        f[kk & 1].multiply(acc);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    if constexpr (BP == BQ) {      // every array holds two waves' results
      store((wave & 4 ? (wave & 2 ? qb : pb) : (wave & 2 ? qa : pa)) + (wave & 1) * (BP * 64));
    } else {
      static_assert(BP == 256 && WP == 4 && WQ == 1 && BQ == 32, "pa holds all waves' results");
      store(pa + wave * (BP * 32));
    }
  }
};

// Writes a wave's results, 64 columns by 32 TQ rows of which a lane holds one row and four adjacent columns
// at a time, as whole 128-byte lines: through the wave's piece of LDS, from which 8 (16 for fp32) lanes take
// a row's 64 columns.  row(r) points to the first of the wave's columns of its row r, or is null; the first
// `cols` columns exist (DIRECT: in whole chunks).
template <bool DIRECT, typename O, int TQ, typename B, typename R>
__device__ __forceinline__ void store_tile(uint8_t* piece, const f32x16 (&acc)[2][TQ], int lane, int cols, B&& bias,
                                           R&& row) {
  constexpr int Bytes = 64 * sizeof(O), Chunks = Bytes / 16;       // of a row
  constexpr int Rows = 64 / Chunks;                                // rows that the wave writes at a time
  constexpr int Group = sizeof(O) == 2 || TQ == 1 ? TQ : TQ / 2;   // 32-row tiles that the piece holds
#pragma unroll
  for (int j0 = 0; j0 < TQ; j0 += Group) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int n = 32 * i + 8 * v + 4 * (lane >> 5);
        float b[4];
        bias(n, b);
#pragma unroll
        for (int j = 0; j < Group; ++j) {
          typedef O vec __attribute__((ext_vector_type(4)));
          vec o;
#pragma unroll
          for (int c = 0; c < 4; ++c) o[c] = (O)(acc[i][j0 + j][4 * v + c] + b[c]);
          const int r = 32 * j + (lane & 31), byte = n * (int)sizeof(O);
          *reinterpret_cast<vec*>(piece + r * Bytes + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15)) = o;
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int c = lane % Chunks, n = c * (16 / (int)sizeof(O));
    if (n < cols) {
#pragma unroll 4
      for (int r = lane / Chunks; r < 32 * Group; r += Rows) {
        O* out = row(32 * j0 + r);
        const uint4 v = *reinterpret_cast<const uint4*>(piece + r * Bytes + ((c ^ (r & 7)) << 4));
        if (!out) continue;
        if constexpr (DIRECT) *reinterpret_cast<uint4*>(out + n) = v;
        else store16(out + n, cols - n, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Zeros in `rows` rows of `cols` columns, ld apart.
template <bool DIRECT, typename O>
__device__ __forceinline__ void store_zeros(O* out, int64_t ld, int rows, int cols, int threads) {
  constexpr int V = kVec<O>;
  const int chunks = (cols + V - 1) / V;
  for (int i = threadIdx.x; i < rows * chunks; i += threads) {
    O* p = out + (i / chunks) * ld + (i % chunks) * V;
    if constexpr (DIRECT) *reinterpret_cast<uint4*>(p) = make_uint4(0, 0, 0, 0);
    else store16(p, cols - (i % chunks) * V, make_uint4(0, 0, 0, 0));
  }
}

// out = x W + b: P is the weight (columns), Q the rows of x.  WIDE: rows of x lie 2^32 bytes or more
// from its first.
template <typename T, bool WKC, bool DIRECT, bool WIDE, int BP, int BQ, int WP, int WQ, bool SHORT>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_rows_kernel(GroupedArgs a, int ntiles) {
  typedef Core<T, WKC, true, BP, BQ, WP, WQ> C;
  typedef typename C::P P;
  typedef typename C::Q Q;
  constexpr int S = sizeof(T), V = C::V, BK = C::BK;
  int group, first, end, ntile;
  if (!find_tile<BQ>(a, block_id(), ntiles, group, first, end, ntile)) return;
  const int n0 = ntile * BP;
  const int rows = end - first < BQ ? end - first : BQ;
  if (group == a.E) {
    const int64_t at = (int64_t)first * a.Nn + n0;
    const int cols = min(a.Nn - n0, BP);
    if (a.out_f32) store_zeros<DIRECT>(static_cast<float*>(a.out) + at, a.Nn, rows, cols, C::Threads);
    else store_zeros<DIRECT>(static_cast<T*>(a.out) + at, a.Nn, rows, cols, C::Threads);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  const int K = a.K, pc = P::column(), qc = Q::column();
  const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.we;
  const T* x = static_cast<const T*>(a.x);
  f32x16 acc[C::TP][C::TQ] = {};
  auto bias = [&](int n, float (&b)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      b[c] = a.bias && n0 + p0 + n + c < a.Nn
                 ? to_f32(static_cast<const T*>(a.bias)[(int64_t)group * a.Nn + n0 + p0 + n + c]) : 0.f;
  };
  auto store = [&](uint8_t* piece) {
    const int cols = a.Nn - n0 - p0;
    const int64_t at = (int64_t)(first + q0) * a.Nn + n0 + p0;
    if (a.out_f32) {
      float* out = static_cast<float*>(a.out) + at;
      store_tile<DIRECT, float>(piece, acc, lane, cols, bias,
                                [&](int r) { return q0 + r < rows ? out + (int64_t)r * a.Nn : nullptr; });
    } else {
      T* out = static_cast<T*>(a.out) + at;
      store_tile<DIRECT, T>(piece, acc, lane, cols, bias,
                            [&](int r) { return q0 + r < rows ? out + (int64_t)r * a.Nn : nullptr; });
    }
  };
  int src[Q::Loads];
  source_rows(a, src, [&](int i) { return first + min(Q::row(i), rows - 1); });
  if constexpr (DIRECT) {
    const uint8_t *wb = reinterpret_cast<const uint8_t*>(w), *xb = reinterpret_cast<const uint8_t*>(x);
    const int64_t ld = a.wk * S;
    typedef typename Offset<WIDE>::type qoff_t;
    uint32_t poff[WKC ? P::Loads : 1];
    qoff_t qoff[Q::Loads];
#pragma unroll
    for (int i = 0; i < Q::Loads; ++i) qoff[i] = (qoff_t)(in_x(a, src[i]) * a.ldx * S);
    if constexpr (WKC) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i) poff[i] = (uint32_t)min(n0 + P::row(i), a.Nn - 1) * (uint32_t)a.wn * S;
    } else {
      poff[0] = min(n0 + pc, a.Nn - V) * S;
    }
    // (past the end of the reduction: its last chunk or row again)
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
      dp += wave * 1024;
      dq += wave * 1024;
      const int k0 = s * BK;
      if constexpr (WKC) {
        const uint32_t k = (uint32_t)min(k0 + pc, K - V) * S;
#pragma unroll
        for (int i = 0; i < P::Loads; ++i) fetch_direct(wb, poff[i] + k, dp + i * (C::Threads * 16));
      } else {
        const uint8_t* ws = wb + k0 * ld;
#pragma unroll
        for (int i = 0; i < P::Loads; ++i)
          fetch_direct(ws, __umul24(min(P::row(i), K - 1 - k0), (uint32_t)ld) + poff[0], dp + i * (C::Threads * 16));
      }
      const uint32_t k = (uint32_t)min(k0 + qc, K - V) * S;
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) fetch_direct(xb, (qoff_t)(qoff[i] + k), dq + i * (C::Threads * 16));
    };
    C::run(K, fill, wave, lane, acc, store);
  } else {
    const T *pat[WKC ? P::Loads : 1], *qat[Q::Loads];
#pragma unroll
    for (int i = 0; i < Q::Loads; ++i) qat[i] = x + in_x(a, src[i]) * a.ldx + qc;
    if constexpr (WKC) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i) pat[i] = w + min(n0 + P::row(i), a.Nn - 1) * a.wn + pc;
    } else {
      pat[0] = w + n0 + pc;
    }
    uint4 vp[P::Loads], vq[Q::Loads];
    auto load = [&](int s) {
      const int k0 = s * BK;
#pragma unroll
      for (int i = 0; i < P::Loads; ++i) {
        if constexpr (WKC) vp[i] = fetch16<SHORT>(pat[i] + k0, K - k0 - pc);
        else vp[i] = fetch16<SHORT>(pat[0] + min(k0 + P::row(i), K - 1) * a.wk, a.Nn - n0 - pc);
      }
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) vq[i] = fetch16<SHORT>(qat[i] + k0, K - k0 - qc);
    };
    load(0);
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i)
        reinterpret_cast<uint4*>(dp)[i * C::Threads + threadIdx.x] =
            keep16<SHORT, T>(vp[i], WKC ? K - s * BK - pc : a.Nn - n0 - pc, WKC ? K : a.Nn);
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i)
        reinterpret_cast<uint4*>(dq)[i * C::Threads + threadIdx.x] = keep16<SHORT, T>(vq[i], K - s * BK - qc, K);
      if ((s + 1) * BK < K) load(s + 1);
    };
    C::run(K, fill, wave, lane, acc, store);
  }
}

// dW[e][d][f] = Σ_p x[p][d] dy[p][f]: P is dy (columns f), Q is x (rows d).  SPLIT: a group's
// positions are cut into gridDim.y parts, whose sums are written as fp32 and added by grouped_reduce.
template <typename T, bool DIRECT, bool WIDE, bool SPLIT, int BP, int BQ, int WP, int WQ, bool SHORT>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_dw_kernel(GroupedArgs a, int ptiles, int qtiles) {
  typedef Core<T, false, false, BP, BQ, WP, WQ> C;
  typedef typename C::P P;
  typedef typename C::Q Q;
  typedef typename Result<T, SPLIT>::type O;
  constexpr int S = sizeof(T), V = C::V, BK = C::BK;
  // (consecutive workgroups go to the 8 XCDs in turn: each XCD gets a share of every group, whatever their sizes)
  const int id = block_id();
  const int e = id / (ptiles * qtiles), tile = id % (ptiles * qtiles);
  if (e >= a.E) return;
  const int f0 = (tile % ptiles) * BP, d0 = (tile / ptiles) * BQ;
  int lo = offset_at(a, e), hi = offset_at(a, e + 1);
  O* out = static_cast<O*>(a.out) + (int64_t)e * a.K * a.Nn;
  if constexpr (SPLIT) {
    split_part(lo, hi, blockIdx.y, gridDim.y);
    out = a.part + ((int64_t)blockIdx.y * a.E + e) * a.K * a.Nn;
  }
  const int n = hi > lo ? hi - lo : 0;
  if (n == 0) {      // nothing came to this expert
    store_zeros<DIRECT>(out + (int64_t)d0 * a.Nn + f0, a.Nn, min(a.K - d0, BQ), min(a.Nn - f0, BP), C::Threads);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  const int fc = f0 + P::column(), dc = d0 + Q::column();
  f32x16 acc[C::TP][C::TQ] = {};
  auto store = [&](uint8_t* piece) {
    O* at = out + (int64_t)(d0 + q0) * a.Nn + f0 + p0;
    store_tile<DIRECT, O>(piece, acc, lane, a.Nn - f0 - p0, [](int, float (&b)[4]) { b[0] = b[1] = b[2] = b[3] = 0.f; },
                          [&](int r) { return d0 + q0 + r < a.K ? at + (int64_t)r * a.Nn : nullptr; });
  };
  int src[Q::Loads];      // rows of x, read a step ahead; past the last: the last
  auto look = [&](int s) { source_rows(a, src, [&](int i) { return lo + min(s * BK + Q::row(i), n - 1); }); };
  look(0);
  if constexpr (DIRECT) {
    const int64_t ld = a.lddy * S;
    const uint8_t* dy = static_cast<const uint8_t*>(a.dy) + lo * ld;
    const uint8_t* x = static_cast<const uint8_t*>(a.x);
    typedef typename Offset<WIDE>::type qoff_t;
    const uint32_t poff = min(fc, a.Nn - V) * S;
    const int qcol = min(dc, a.K - V);
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
      dp += wave * 1024;
      dq += wave * 1024;
      const int k0 = s * BK;
      qoff_t qoff[Q::Loads];
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) qoff[i] = ((qoff_t)in_x(a, src[i]) * (qoff_t)a.ldx + qcol) * S;
      look(s + 1);
      const uint8_t* ds = dy + k0 * ld;
#pragma unroll
      for (int i = 0; i < P::Loads; ++i)
        fetch_direct(ds, __umul24(min(P::row(i), n - 1 - k0), (uint32_t)ld) + poff, dp + i * (C::Threads * 16));
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) fetch_direct(x, qoff[i], dq + i * (C::Threads * 16));
    };
    C::run(n, fill, wave, lane, acc, store);
  } else {
    const T* dy = static_cast<const T*>(a.dy) + lo * a.lddy + fc;
    const T* x = static_cast<const T*>(a.x) + dc;
    uint4 vp[P::Loads], vq[Q::Loads];
    auto load = [&](int s) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i) vp[i] = fetch16<SHORT>(dy + min(s * BK + P::row(i), n - 1) * a.lddy, a.Nn - fc);
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) vq[i] = fetch16<SHORT>(x + in_x(a, src[i]) * a.ldx, a.K - dc);
      look(s + 1);
    };
    load(0);
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i)
        reinterpret_cast<uint4*>(dp)[i * C::Threads + threadIdx.x] = keep16<SHORT, T>(vp[i], a.Nn - fc, a.Nn);
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i)
        reinterpret_cast<uint4*>(dq)[i * C::Threads + threadIdx.x] = keep16<SHORT, T>(vq[i], a.K - dc, a.K);
      if ((s + 1) * BK < n) load(s + 1);
    };
    C::run(n, fill, wave, lane, acc, store);
  }
}

// Rows of x whose bytes do not fit 32-bit offsets.
template <typename T>
bool wide(const GroupedArgs& a) { return (a.Nx * a.ldx + a.K) * (int64_t)sizeof(T) >= (int64_t(1) << 32); }

template <typename T, bool WKC, bool DIRECT, bool WIDE, int BP, int BQ, int WP, int WQ, bool SHORT = false>
void rows_tiled(const GroupedArgs& a, hipStream_t s) {
  const int ntiles = (a.Nn + BP - 1) / BP;
  grouped_rows_kernel<T, WKC, DIRECT, WIDE, BP, BQ, WP, WQ, SHORT>
      <<<grid_of((a.M / BQ + a.E + 1) * ntiles, 64 * WP * WQ), 64 * WP * WQ, 0, s>>>(a, ntiles);
}

// fp32 tiles of 256 columns by 32 rows where the groups are small: whether they take less matrix work than tiles
// of 128 (a group's last row tile is half full on average).  1024 x 2048 matrices, 64 experts: 95 us and 256 us
// by tiles of 128 at 256 positions (537 MB of weights, 5.6 TB/s), 200 and 260 us at 4096; 16 experts, where both
// leave CUs idle: 42 and 71 us at 128 positions.
inline bool small_groups(const GroupedArgs& a) {
  return (a.M / 32.0 + 0.5 * a.E) * ((a.Nn + 255) / 256) * 0.5 < (a.M / 128.0 + 0.5 * a.E) * ((a.Nn + 127) / 128);
}

template <typename T, bool WKC>
void rows_by(const GroupedArgs& a, bool direct, bool larger, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (direct && larger)
      return wide<T>(a) ? rows_tiled<T, WKC, true, true, 256, 256, 4, 2>(a, s)
                        : rows_tiled<T, WKC, true, false, 256, 256, 4, 2>(a, s);
  } else if (small_groups(a) && a.K >= kVec<T> && a.Nn >= kVec<T>) {
    if (!direct) rows_tiled<T, WKC, false, true, 256, 32, 4, 1>(a, s);
    else if (wide<T>(a)) rows_tiled<T, WKC, true, true, 256, 32, 4, 1>(a, s);
    else rows_tiled<T, WKC, true, false, 256, 32, 4, 1>(a, s);
    return;
  }
  if (a.K < kVec<T> || a.Nn < kVec<T>) rows_tiled<T, WKC, false, true, 128, 128, 2, 2, true>(a, s);
  else if (!direct) rows_tiled<T, WKC, false, true, 128, 128, 2, 2>(a, s);
  else if (wide<T>(a)) rows_tiled<T, WKC, true, true, 128, 128, 2, 2>(a, s);
  else rows_tiled<T, WKC, true, false, 128, 128, 2, 2>(a, s);
}

template <typename T, bool DIRECT, bool WIDE, bool SPLIT, int B, int WP, int WQ, bool SHORT = false>
void dw_tiled(const GroupedArgs& a, int splits, hipStream_t s) {
  const int pt = (a.Nn + B - 1) / B, qt = (a.K + B - 1) / B;
  grouped_dw_kernel<T, DIRECT, WIDE, SPLIT, B, B, WP, WQ, SHORT>
      <<<grid_of((int64_t)a.E * pt * qt, 64 * WP * WQ, splits), 64 * WP * WQ, 0, s>>>(a, pt, qt);
}

template <typename T, bool SPLIT>
void dw_by(const GroupedArgs& a, bool direct, int splits, hipStream_t s) {
  if (a.K < kVec<T> || a.Nn < kVec<T>) dw_tiled<T, false, true, SPLIT, 128, 2, 2, true>(a, splits, s);
  else if (!direct) dw_tiled<T, false, true, SPLIT, 128, 2, 2>(a, splits, s);
  else if (wide<T>(a)) dw_tiled<T, true, true, SPLIT, 128, 2, 2>(a, splits, s);
  else dw_tiled<T, true, false, SPLIT, 128, 2, 2>(a, splits, s);
}

}  // namespace

template <typename T>
void launch_rows_tiles(const GroupedArgs& a, bool direct, bool larger, hipStream_t s) {
  if (a.wk == 1 && a.wn != 1) rows_by<T, true>(a, direct, larger, s);
  else rows_by<T, false>(a, direct, larger, s);
}

template <typename T>
void launch_dw_tiles(const GroupedArgs& a, bool direct, bool larger, int splits, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (direct && larger)
      return wide<T>(a) ? dw_tiled<T, true, true, false, 256, 4, 2>(a, 1, s)
                        : dw_tiled<T, true, false, false, 256, 4, 2>(a, 1, s);
  }
  if (splits > 1) dw_by<T, true>(a, direct, splits, s);
  else dw_by<T, false>(a, direct, 1, s);
}

}  // namespace gx::layer
