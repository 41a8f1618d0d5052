// Grouped products of 16-bit elements on whole 16-byte chunks (see grouped.hip for the
// mathematics and for every other width, stride and type).
//
// A workgroup forms a tile out[q][p], q over BQ rows and p over BP columns, by
// 32 x 32 x 16 MFMA with the column operand first, so that a lane holds one row and
// four adjacent columns of the result.  Both operands are staged 64 deep in LDS by
// loads that write LDS directly, two buffers in turn: the next step's loads are in
// flight while this step's products run.  An operand whose reduction index is
// adjacent in memory lies in LDS as [row][64] and is read 16 bytes a lane; one whose
// reduction index is not (a weight read along its other dimension, both operands of
// the weight's gradient) lies as [64][row] and is read by the transposing LDS loads:
// no copy of either is ever transposed in memory.  A direct load fills LDS in lane
// order, so the order of chunks that keeps the reads free of bank conflicts is made
// by which chunk each lane fetches: chunk c of row r sits at c ^ (r & 7), a 32-byte
// pair u of reduction row k at u ^ (k & 7).
//
// Ragged ends: rows past a group's end are read from its last row and not stored,
// columns past the matrix likewise; past the end of the reduction its last elements
// are read again and masked in registers.

#include <math.h>

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (sizeof(T) == 2 && __is_same(T, bf16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 16 bytes a lane from base + off to the wave's 1024 bytes of LDS at `dst`, in lane order.  With a
// 32-bit off and one base for the wave the address takes no vector arithmetic.
template <typename O>
__device__ __forceinline__ void fetch16(const uint8_t* base, O off, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(base + off),
                                   (__attribute__((address_space(3))) uint32_t*)dst, 16, 0, 0);
}

// Where a lane reads its fragments of one operand's tile.  A fragment is the 8 reduction
// elements 16 kk + 8 (lane / 32) + 0..7 of row 32 i + lane % 32 of the wave's rows.
template <bool KC, int R, int N, int BK>
struct Reader;

// The place of chunk c in row r of a [row][BK] tile: eight rows' same chunk lie in eight different 16-byte
// slots of a 128-byte line.
template <int BK>
__device__ __forceinline__ int swizzle(int c, int r) {
  return BK == 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
}

template <int R, int N, int BK>
struct Reader<true, R, N, BK> {
  int at[BK / 16];      // of i = 0, for each kk
  __device__ __forceinline__ Reader(int r0, int lane) {
    const int r = r0 + (lane & 31);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) at[kk] = r * (BK * 2) + (swizzle<BK>(2 * kk + (lane >> 5), r) << 4);
  }
  __device__ __forceinline__ s16x8 get(const uint8_t* tile, int i, int kk) const {
    return *reinterpret_cast<const s16x8*>(tile + at[kk] + i * (32 * BK * 2));
  }
};

template <int R, int N, int BK>
struct Reader<false, R, N, BK> {
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
  __device__ __forceinline__ s16x8 get(const uint8_t* tile, int i, int kk) const {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + lo[i] + kk * (16 * R * 2)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + hi[i] + kk * (16 * R * 2)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// A thread's share of the loads of an operand's tile: R rows by BK of the reduction.
template <bool KC, int R, int BK, int THREADS>
struct Share {
  static constexpr int Loads = R * BK * 2 / (THREADS * 16);
  static constexpr int PerRow = KC ? BK / 8 : R / 8;          // chunks of a row of the tile
  static constexpr int Step = THREADS / PerRow;               // tile rows between a thread's loads
  static_assert(Loads >= 1 && Step % 8 == 0, "a thread's rows agree modulo 8");
  // Tile row of load i: a row of the operand (KC) or a reduction row.
  __device__ static __forceinline__ int row(int i) { return threadIdx.x / PerRow + i * Step; }
  // First element of the thread's chunk along the tile row.
  __device__ static __forceinline__ int column() {
    const int c = threadIdx.x % PerRow, r = row(0);
    if constexpr (KC) return swizzle<BK>(c, r) * 8;
    else return ((((c >> 1) ^ (r & 7)) << 1) | (c & 1)) * 8;
  }
};

// Byte offsets from an operand's first element.
template <bool WIDE> struct Offset { typedef uint32_t type; };
template <> struct Offset<true> { typedef int64_t type; };

template <typename T, bool PKC, bool QKC, int BP, int BQ, int WP, int WQ, int BK>
struct Core {
  static constexpr int Threads = 64 * WP * WQ;
  static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;    // 32 x 32 tiles of a wave
  typedef Share<PKC, BP, BK, Threads> P;
  typedef Share<QKC, BQ, BK, Threads> Q;
  typedef Reader<PKC, BP, TP, BK> RP;
  typedef Reader<QKC, BQ, TQ, BK> RQ;
  static constexpr int Loads = P::Loads + Q::Loads;             // of a thread for a step
  struct Frags {
    s16x8 p[TP], q[TQ];
    __device__ __forceinline__ void read(const uint8_t* tp, const uint8_t* tq, const RP& rp, const RQ& rq, int kk) {
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] = rp.get(tp, i, kk);
#pragma unroll
      for (int j = 0; j < TQ; ++j) q[j] = rq.get(tq, j, kk);
    }
    // Zeros at reduction elements past the first `left` of this lane's eight.
    __device__ __forceinline__ void mask(int left) {
      typedef int i32x4 __attribute__((ext_vector_type(4)));
      i32x4 m;
#pragma unroll
      for (int d = 0; d < 4; ++d) m[d] = left >= 2 * d + 2 ? -1 : (left == 2 * d + 1 ? 0xffff : 0);
#pragma unroll
      for (int i = 0; i < TP; ++i) p[i] = __builtin_bit_cast(s16x8, __builtin_bit_cast(i32x4, p[i]) & m);
#pragma unroll
      for (int j = 0; j < TQ; ++j) q[j] = __builtin_bit_cast(s16x8, __builtin_bit_cast(i32x4, q[j]) & m);
    }
    __device__ __forceinline__ void multiply(f32x16 (&acc)[TP][TQ]) const {
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = mfma32<T>(p[i], q[j], acc[i][j]);
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
  // Then store(piece) is called with 1/8 (1/4) of the stages' LDS for each of 8 (4) waves: room for the wave's
  // part of the tile in 16 bits.
  template <typename F, typename G>
  __device__ static __forceinline__ void run(int total, F&& fill, int wave, int lane, f32x16 (&acc)[TP][TQ],
                                             G&& store) {
    const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
    __shared__ __align__(16) uint8_t pa[BP * BK * 2], pb[BP * BK * 2], qa[BQ * BK * 2], qb[BQ * BK * 2];
    const RP rp(p0, lane);
    const RQ rq(q0, lane);
    constexpr int KK = BK / 16;
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
    const int left = total - last * BK - 8 * (lane >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if (kk + 1 < KK) f[(kk + 1) & 1].read(p, q, rp, rq, kk + 1);
      __builtin_amdgcn_sched_barrier(0);
      f[kk & 1].mask(left - 16 * kk);
      f[kk & 1].multiply(acc);
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    static_assert(BP == BQ, "every array holds two waves' results");
    store((wave & 4 ? (wave & 2 ? qb : pb) : (wave & 2 ? qa : pa)) + (wave & 1) * (BP * BK));
  }
};

// Writes a wave's results, 64 columns by 32 TQ rows of which a lane holds one row and four adjacent columns
// at a time, as whole 128-byte lines: through the wave's piece of LDS, from which 8 (16 for fp32) lanes take
// a row's 64 columns.  row(r) points to the first of the wave's columns of its row r, or is null; the first
// `cols` columns exist (a multiple of 8).
template <typename O, int TQ, typename B, typename R>
__device__ __forceinline__ void store_tile(uint8_t* piece, const f32x16 (&acc)[2][TQ], int lane, int cols, B&& bias,
                                           R&& row) {
  constexpr int Bytes = 64 * sizeof(O), Chunks = Bytes / 16;       // of a row
  constexpr int Rows = 64 / Chunks;                                // rows that the wave writes at a time
  constexpr int Group = sizeof(O) == 2 ? TQ : TQ / 2;              // 32-row tiles that the piece holds
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
    const int c = lane % Chunks;
    if (c * (16 / (int)sizeof(O)) < cols) {
#pragma unroll 4
      for (int r = lane / Chunks; r < 32 * Group; r += Rows) {
        O* out = row(32 * j0 + r);
        const uint4 v = *reinterpret_cast<const uint4*>(piece + r * Bytes + ((c ^ (r & 7)) << 4));
        if (out) *reinterpret_cast<uint4*>(out + c * (16 / (int)sizeof(O))) = v;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// out = x W + b: P is the weight (columns), Q the rows of x.  WIDE: rows of x lie 2^32 bytes or more
// from its first.
template <typename T, bool WKC, bool WIDE, int BP, int BQ, int WP, int WQ, int BK>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_mma_kernel(GroupedArgs a, int ntiles) {
  typedef Core<T, WKC, true, BP, BQ, WP, WQ, BK> C;
  typedef typename C::P P;
  typedef typename C::Q Q;
  int group, first, end, ntile;
  if (!find_tile<BQ>(a, blockIdx.x, ntiles, group, first, end, ntile)) return;
  const int n0 = ntile * BP;
  const int rows = end - first < BQ ? end - first : BQ;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  f32x16 acc[C::TP][C::TQ] = {};
  if (group < a.E) {
    const int K = a.K, pc = P::column(), qc = Q::column();
    const uint8_t* w = static_cast<const uint8_t*>(a.w) + (int64_t)group * a.we * 2;
    const uint8_t* x = static_cast<const uint8_t*>(a.x);
    const int64_t ld = a.wk * 2;
    typedef typename Offset<WIDE>::type qoff_t;
    uint32_t poff[WKC ? P::Loads : 1];
    qoff_t qoff[Q::Loads];
#pragma unroll
    for (int i = 0; i < Q::Loads; ++i) {
      const int r = Q::row(i) < rows ? Q::row(i) : rows - 1;
      qoff[i] = (qoff_t)(source_row(a, first + r) * a.ldx * 2);
    }
    if constexpr (WKC) {
#pragma unroll
      for (int i = 0; i < P::Loads; ++i) {
        const int n = n0 + P::row(i) < a.Nn ? n0 + P::row(i) : a.Nn - 1;
        poff[i] = (uint32_t)n * (uint32_t)a.wn * 2;
      }
    } else {
      poff[0] = (n0 + pc < a.Nn ? n0 + pc : a.Nn - 8) * 2;
    }
    // (past the end of the reduction: its last chunk or row again)
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
      dp += wave * 1024;
      dq += wave * 1024;
      const int k0 = s * BK;
      if constexpr (WKC) {
        const uint32_t k = (uint32_t)min(k0 + pc, K - 8) * 2;
#pragma unroll
        for (int i = 0; i < P::Loads; ++i) fetch16(w, poff[i] + k, dp + i * (C::Threads * 16));
      } else {
        const uint8_t* ws = w + k0 * ld;
#pragma unroll
        for (int i = 0; i < P::Loads; ++i)
          fetch16(ws, __umul24(min(P::row(i), K - 1 - k0), (uint32_t)ld) + poff[0], dp + i * (C::Threads * 16));
      }
      const uint32_t k = (uint32_t)min(k0 + qc, K - 8) * 2;
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) fetch16(x, (qoff_t)(qoff[i] + k), dq + i * (C::Threads * 16));
    };
    auto bias = [&](int n, float (&b)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) b[c] = 0.f;
      if (a.bias && n0 + p0 + n < a.Nn) {
        const T* at = static_cast<const T*>(a.bias) + (int64_t)group * a.Nn + n0 + p0 + n;
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = to_f32(at[c]);
      }
    };
    C::run(K, fill, wave, lane, acc, [&](uint8_t* piece) {
      const int cols = a.Nn - n0 - p0;
      const int64_t at = (int64_t)(first + q0) * a.Nn + n0 + p0;
      if (a.out_f32) {
        float* out = static_cast<float*>(a.out) + at;
        store_tile<float>(piece, acc, lane, cols, bias,
                          [&](int r) { return q0 + r < rows ? out + (int64_t)r * a.Nn : nullptr; });
      } else {
        T* out = static_cast<T*>(a.out) + at;
        store_tile<T>(piece, acc, lane, cols, bias,
                      [&](int r) { return q0 + r < rows ? out + (int64_t)r * a.Nn : nullptr; });
      }
    });
  } else {      // rows past the last group
    const int per = a.out_f32 ? 4 : 8, chunks = (min(a.Nn - n0, BP) + per - 1) / per;
    uint8_t* out = static_cast<uint8_t*>(a.out) + ((int64_t)first * a.Nn + n0) * (16 / per);
    for (int i = threadIdx.x; i < rows * chunks; i += C::Threads)
      *reinterpret_cast<uint4*>(out + ((int64_t)(i / chunks) * a.Nn * (16 / per)) + (i % chunks) * 16) = make_uint4(0, 0, 0, 0);
  }
}

// dW[e][d][f] = Σ_p x[p][d] dy[p][f]: P is dy (columns f), Q is x (rows d).  SPLIT: a group's
// positions are cut into gridDim.y parts, whose sums are written as fp32 and added by grouped_reduce.
template <typename T, bool WIDE, bool SPLIT, int BP, int BQ, int WP, int WQ, int BK>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_mma_dw_kernel(GroupedArgs a, int ptiles, int qtiles) {
  typedef Core<T, false, false, BP, BQ, WP, WQ, BK> C;
  typedef typename C::P P;
  typedef typename C::Q Q;
  typedef typename Result<T, SPLIT>::type O;
  // (consecutive workgroups go to the 8 XCDs in turn: each XCD gets a share of every group, whatever their sizes)
  const int id = blockIdx.x;
  const int e = id / (ptiles * qtiles), tile = id % (ptiles * qtiles);
  const int f0 = (tile % ptiles) * BP, d0 = (tile / ptiles) * BQ;
  int lo = offset_at(a, e), hi = offset_at(a, e + 1);
  O* out = static_cast<O*>(a.out) + (int64_t)e * a.K * a.Nn;
  if constexpr (SPLIT) {
    split_part(lo, hi, blockIdx.y, gridDim.y);
    out = a.part + ((int64_t)blockIdx.y * a.E + e) * a.K * a.Nn;
  }
  const int n = hi > lo ? hi - lo : 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  f32x16 acc[C::TP][C::TQ] = {};
  if (n > 0) {
    const int fc = f0 + P::column() < a.Nn ? f0 + P::column() : a.Nn - 8;
    const int dc = d0 + Q::column() < a.K ? d0 + Q::column() : a.K - 8;
    const int64_t ld = a.lddy * 2;
    const uint8_t* dy = static_cast<const uint8_t*>(a.dy) + lo * ld;
    const uint8_t* x = static_cast<const uint8_t*>(a.x);
    typedef typename Offset<WIDE>::type qoff_t;
    const uint32_t poff = fc * 2;
    int src[Q::Loads];      // rows of x, read a step ahead; past the last: the last
    auto look = [&](int s) {
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) src[i] = (int)source_row(a, lo + min(s * BK + Q::row(i), n - 1));
    };
    look(0);
    auto fill = [&](int s, uint8_t* dp, uint8_t* dq) {
      dp += wave * 1024;
      dq += wave * 1024;
      const int k0 = s * BK;
      qoff_t qoff[Q::Loads];
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) qoff[i] = ((qoff_t)src[i] * (qoff_t)a.ldx + dc) * 2;
      look(s + 1);
      const uint8_t* ds = dy + k0 * ld;
#pragma unroll
      for (int i = 0; i < P::Loads; ++i)
        fetch16(ds, __umul24(min(P::row(i), n - 1 - k0), (uint32_t)ld) + poff, dp + i * (C::Threads * 16));
#pragma unroll
      for (int i = 0; i < Q::Loads; ++i) fetch16(x, qoff[i], dq + i * (C::Threads * 16));
    };
    C::run(n, fill, wave, lane, acc, [&](uint8_t* piece) {
      O* at = out + (int64_t)(d0 + q0) * a.Nn + f0 + p0;
      store_tile<O>(piece, acc, lane, a.Nn - f0 - p0, [](int, float (&b)[4]) { b[0] = b[1] = b[2] = b[3] = 0.f; },
                    [&](int r) { return d0 + q0 + r < a.K ? at + (int64_t)r * a.Nn : nullptr; });
    });
  } else {      // nothing came to this expert
    constexpr int per = 16 / sizeof(O);
    const int chunks = min(a.Nn - f0, BP) / per, rows = min(a.K - d0, BQ);
    for (int i = threadIdx.x; i < rows * chunks; i += C::Threads)
      *reinterpret_cast<uint4*>(out + (int64_t)(d0 + i / chunks) * a.Nn + f0 + (i % chunks) * per) = make_uint4(0, 0, 0, 0);
  }
}

// Rows of x whose bytes do not fit 32-bit offsets.
bool wide(const GroupedArgs& a) { return a.Nx * a.ldx * 2 + a.K * 2 >= (int64_t(1) << 32); }

template <typename T, bool WKC, int BP, int BQ, int WP, int WQ>
void rows_tiled(const GroupedArgs& a, hipStream_t s) {
  const int ntiles = (a.Nn + BP - 1) / BP;
  const int64_t grid = (a.M / BQ + a.E + 1) * ntiles;
  if (wide(a))
    grouped_mma_kernel<T, WKC, true, BP, BQ, WP, WQ, 64><<<(unsigned)grid, 64 * WP * WQ, 0, s>>>(a, ntiles);
  else
    grouped_mma_kernel<T, WKC, false, BP, BQ, WP, WQ, 64><<<(unsigned)grid, 64 * WP * WQ, 0, s>>>(a, ntiles);
}

// Whether tiles of 256 (one to a CU) beat tiles of 128 (two at a time): the most tiles that a CU gets, in
// 128 x 128 tiles, over the rate measured for each (1170 and 880 TFLOP/s for one product of 8192 x 8192 x
// 8192).  8192 rows of 16 experts, 2048 -> 1024: 56.8 us by 256, 39.5 us by 128; 32768 rows of 32 experts,
// 1024 -> 2048: 172 and 203 us, its gradient for x 190 and 209 us (near ties go to the larger).
bool larger_tiles(double tiles256, double tiles128) {
  return ceil(tiles256 / 256.0) * 4.0 / 1.17 < 1.1 * ceil(tiles128 / 256.0) / 0.88;
}

double tiles(int64_t n, int t) { return (double)((n + t - 1) / t); }

template <typename T, bool WKC>
void rows_mma(const GroupedArgs& a, hipStream_t s) {
  // (a group's last row tile is half full on average)
  if (larger_tiles((a.M / 256.0 + 0.5 * a.E) * tiles(a.Nn, 256), (a.M / 128.0 + 0.5 * a.E) * tiles(a.Nn, 128)))
    rows_tiled<T, WKC, 256, 256, 4, 2>(a, s);
  else
    rows_tiled<T, WKC, 128, 128, 2, 2>(a, s);
}

template <typename T, int BP, int BQ, int WP, int WQ>
void dw_tiled(const GroupedArgs& a, int splits, hipStream_t s) {
  const int pt = (a.Nn + BP - 1) / BP, qt = (a.K + BQ - 1) / BQ, threads = 64 * WP * WQ;
  const dim3 grid((unsigned)(a.E * pt * qt), (unsigned)splits);
  if (splits > 1) {
    if (wide(a)) grouped_mma_dw_kernel<T, true, true, BP, BQ, WP, WQ, 64><<<grid, threads, 0, s>>>(a, pt, qt);
    else grouped_mma_dw_kernel<T, false, true, BP, BQ, WP, WQ, 64><<<grid, threads, 0, s>>>(a, pt, qt);
  } else {
    if (wide(a)) grouped_mma_dw_kernel<T, true, false, BP, BQ, WP, WQ, 64><<<grid, threads, 0, s>>>(a, pt, qt);
    else grouped_mma_dw_kernel<T, false, false, BP, BQ, WP, WQ, 64><<<grid, threads, 0, s>>>(a, pt, qt);
  }
}

bool dw_larger(int64_t E, int64_t K, int64_t N) {
  return larger_tiles(E * tiles(K, 256) * tiles(N, 256), E * tiles(K, 128) * tiles(N, 128));
}

template <typename T>
void dw_mma(const GroupedArgs& a, int splits, hipStream_t s) {
  if (dw_larger(a.E, a.K, a.Nn)) dw_tiled<T, 256, 256, 4, 2>(a, 1, s);
  else dw_tiled<T, 128, 128, 2, 2>(a, splits, s);
}

// What 32-bit offsets reach: 64 rows of a matrix, and the whole of one that is read along its rows.
bool near_rows(int64_t ld) { return ld * 2 < (int64_t(1) << 24); }

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

// Parts that each group's positions are cut into where the tiles leave most of the 512 workgroups that run
// at once idle: no part of an average group below 512 positions.
int grouped_mma_dw_splits(int64_t M, int64_t E, int64_t K, int64_t N) {
  if (dw_larger(E, K, N)) return 1;
  return parts_of(M, E, E * (int64_t)(tiles(K, 128) * tiles(N, 128)), 512, 512);
}

// 16-bit elements in whole 16-byte chunks along every dimension that is read 16 bytes
// at a time.
bool grouped_mma_rows_ok(const GroupedArgs& a) {
  const int64_t outer = a.wk == 1 ? a.wn : a.wk;
  return a.elem != ELEM_F32 && a.K % 8 == 0 && a.Nn % 8 == 0 && a.ldx % 8 == 0 && a.we % 8 == 0 && outer % 8 == 0 &&
         near_rows(outer) && outer * (a.wk == 1 ? a.Nn : 64) * 2 < (int64_t(1) << 32) && aligned16(a.x) &&
         aligned16(a.w) && aligned16(a.out);
}

bool grouped_mma_dw_ok(const GroupedArgs& a) {
  return a.elem != ELEM_F32 && a.K % 8 == 0 && a.Nn % 8 == 0 && a.ldx % 8 == 0 && a.lddy % 8 == 0 && near_rows(a.lddy) &&
         aligned16(a.x) && aligned16(a.dy) && aligned16(a.out);
}

void launch_grouped_mma(const GroupedArgs& a, hipStream_t s) {
  const bool kc = a.wk == 1 && a.wn != 1;
  if (a.elem == ELEM_BF16) kc ? rows_mma<bf16_t, true>(a, s) : rows_mma<bf16_t, false>(a, s);
  else kc ? rows_mma<_Float16, true>(a, s) : rows_mma<_Float16, false>(a, s);
}

void launch_grouped_mma_dw(const GroupedArgs& a, int splits, hipStream_t s) {
  if (a.elem == ELEM_BF16) dw_mma<bf16_t>(a, splits, s);
  else dw_mma<_Float16>(a, splits, s);
}

}  // namespace gx::layer
