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
// columns past the matrix likewise; chunks past the end of the reduction are fetched
// from a page of zeros.

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kBK = 64;

__device__ uint4 zero_page[4];    // (never written)

template <typename T>
__device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (sizeof(T) == 2 && __is_same(T, bf16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) uint8_t* lds_ptr;
typedef const __attribute__((address_space(1))) uint8_t* global_ptr;

// 16 bytes a lane from `src` to the wave's 1024 bytes of LDS at `dst`, in lane order.
__device__ __forceinline__ void fetch16(const void* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                   (__attribute__((address_space(3))) uint32_t*)dst, 16, 0, 0);
}

// Where a lane reads its fragments of one operand's tile.  A fragment is the 8 reduction
// elements 16 kk + 8 (lane / 32) + 0..7 of row 32 i + lane % 32 of the wave's rows.
template <bool KC, int R, int N>
struct Reader;

template <int R, int N>
struct Reader<true, R, N> {
  int at[kBK / 16];      // of i = 0, for each kk
  __device__ __forceinline__ Reader(int r0, int lane) {
    const int r = r0 + (lane & 31);
#pragma unroll
    for (int kk = 0; kk < kBK / 16; ++kk) at[kk] = r * (kBK * 2) + (((2 * kk + (lane >> 5)) ^ (r & 7)) << 4);
  }
  __device__ __forceinline__ s16x8 get(const uint8_t* tile, int i, int kk) const {
    return *reinterpret_cast<const s16x8*>(tile + at[kk] + i * (32 * kBK * 2));
  }
};

template <int R, int N>
struct Reader<false, R, N> {
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

// A thread's share of an operand's tile: R rows by 64 of the reduction.
template <bool KC, int R, int THREADS>
struct Share {
  static constexpr int Loads = R * kBK * 2 / (THREADS * 16);
  static constexpr int PerRow = R / 8;                        // chunks of a reduction row (!KC)
  const uint8_t* at[Loads];   // KC: each load's row; !KC: at[0]: the thread's first reduction row
  int64_t ld;                 // !KC: bytes between reduction rows

  // KC: chunk index of every load; !KC: reduction row of load i is first_k() + i step_k()
  __device__ static __forceinline__ int chunk() { return (threadIdx.x & 7) ^ ((threadIdx.x >> 3) & 7); }
  __device__ static __forceinline__ int row(int i) { return (i * THREADS + threadIdx.x) >> 3; }
  __device__ static __forceinline__ int first_k() { return threadIdx.x / PerRow; }
  static constexpr int step_k = THREADS / PerRow;
  __device__ static __forceinline__ int column() {
    const int c = threadIdx.x % PerRow, k = first_k();
    static_assert(step_k % 8 == 0 || KC, "a thread's reduction rows agree modulo 8");
    return ((((c >> 1) ^ (k & 7)) << 1) | (c & 1)) * 8;
  }
};

template <typename T, bool PKC, bool QKC, int BP, int BQ, int WP, int WQ>
struct Core {
  static constexpr int Threads = 64 * WP * WQ;
  static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;    // 32 x 32 tiles of a wave
  typedef Share<PKC, BP, Threads> P;
  typedef Share<QKC, BQ, Threads> Q;

  typedef Reader<PKC, BP, TP> RP;
  typedef Reader<QKC, BQ, TQ> RQ;

  // One step's products; the fragments of the next 16 are read while these 16 multiply.
  __device__ static __forceinline__ void products(const uint8_t* tp, const uint8_t* tq, const RP& rp, const RQ& rq,
                                                  f32x16 (&acc)[TP][TQ]) {
    s16x8 fp[2][TP], fq[2][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i) fp[0][i] = rp.get(tp, i, 0);
#pragma unroll
    for (int j = 0; j < TQ; ++j) fq[0][j] = rq.get(tq, j, 0);
#pragma unroll
    for (int kk = 0; kk < kBK / 16; ++kk) {
      const int now = kk & 1, next = now ^ 1;
      if (kk + 1 < kBK / 16) {
#pragma unroll
        for (int i = 0; i < TP; ++i) fp[next][i] = rp.get(tp, i, kk + 1);
#pragma unroll
        for (int j = 0; j < TQ; ++j) fq[next][j] = rq.get(tq, j, kk + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = mfma32<T>(fp[now][i], fq[now][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Sums over `steps` steps of 64; fill_p / fill_q(step, dst) start one step's loads.
  template <typename FP, typename FQ>
  __device__ static __forceinline__ void run(int steps, FP&& fill_p, FQ&& fill_q, int p0, int q0, int lane,
                                             f32x16 (&acc)[TP][TQ]) {
    __shared__ __align__(16) uint8_t p_even[BP * kBK * 2], q_even[BQ * kBK * 2];
    __shared__ __align__(16) uint8_t p_odd[BP * kBK * 2], q_odd[BQ * kBK * 2];
    if (steps <= 0) return;
    const RP rp(p0, lane);
    const RQ rq(q0, lane);
    fill_p(0, p_even);
    fill_q(0, q_even);
    int s = 0;
    for (; s + 1 < steps; s += 2) {
      __syncthreads();      // waits for the loads of step s, and for the readers of the other buffers
      fill_p(s + 1, p_odd);
      fill_q(s + 1, q_odd);
      products(p_even, q_even, rp, rq, acc);
      __syncthreads();
      if (s + 2 < steps) {
        fill_p(s + 2, p_even);
        fill_q(s + 2, q_even);
      }
      products(p_odd, q_odd, rp, rq, acc);
    }
    if (s < steps) {
      __syncthreads();
      products(p_even, q_even, rp, rq, acc);
    }
  }
};

// Four adjacent results.
template <typename O>
__device__ __forceinline__ void store4(O* p, int valid, const float (&v)[4]) {
  typedef O vec __attribute__((ext_vector_type(4)));
  if (valid >= 4) {
    vec o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (O)v[i];
    *reinterpret_cast<vec*>(p) = o;
  }
}

// Tile index of a workgroup: consecutive workgroups go to the 8 XCDs in turn, so each
// XCD gets a contiguous run of tiles and its L2 keeps their operands.
__device__ __forceinline__ int64_t xcd_tile(int64_t id, int64_t total) {
  const int64_t per = total / 8, rest = total % 8, x = id % 8;
  return x * per + (x < rest ? x : rest) + id / 8;
}

// out = x W + b: P is the weight (columns), Q the rows of x.
template <typename T, bool WKC, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_mma_kernel(GroupedArgs a, int ntiles) {
  typedef Core<T, WKC, true, BP, BQ, WP, WQ> C;
  const int64_t id = xcd_tile(blockIdx.x, gridDim.x);
  int group;
  int64_t first, end;
  if (!find_tile<BQ>(a, id / ntiles, group, first, end)) return;
  const int n0 = (int)(id % ntiles) * BP;
  const int rows = (int)(end - first < BQ ? end - first : BQ);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  f32x16 acc[C::TP][C::TQ] = {};
  if (group < a.E) {
    typename C::P sp;
    typename C::Q sq;
    const int K = a.K;
    const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.we;
    const T* x = static_cast<const T*>(a.x);
#pragma unroll
    for (int i = 0; i < C::Q::Loads; ++i) {
      const int r = C::Q::row(i) < rows ? C::Q::row(i) : rows - 1;
      sq.at[i] = reinterpret_cast<const uint8_t*>(x + source_row(a, first + r) * a.ldx + C::Q::chunk() * 8);
    }
    if constexpr (WKC) {
#pragma unroll
      for (int i = 0; i < C::P::Loads; ++i) {
        const int n = n0 + C::P::row(i) < a.Nn ? n0 + C::P::row(i) : a.Nn - 1;
        sp.at[i] = reinterpret_cast<const uint8_t*>(w + (int64_t)n * a.wn + C::P::chunk() * 8);
      }
    } else {
      const int n = n0 + C::P::column() < a.Nn ? n0 + C::P::column() : a.Nn - 8;
      sp.ld = a.wk * 2;
      sp.at[0] = reinterpret_cast<const uint8_t*>(w + n) + C::P::first_k() * sp.ld;
    }
    const uint8_t* zeros = reinterpret_cast<const uint8_t*>(zero_page);
    const int wbase = wave * 1024;
    auto fill_q = [&](int s, uint8_t* dst) {
      const bool whole = (s + 1) * kBK <= K || s * kBK + C::Q::chunk() * 8 < K;
#pragma unroll
      for (int i = 0; i < C::Q::Loads; ++i)
        fetch16(whole ? sq.at[i] + (int64_t)s * (kBK * 2) : zeros, dst + i * (C::Threads * 16) + wbase);
    };
    auto fill_p = [&](int s, uint8_t* dst) {
      if constexpr (WKC) {
        const bool whole = (s + 1) * kBK <= K || s * kBK + C::P::chunk() * 8 < K;
#pragma unroll
        for (int i = 0; i < C::P::Loads; ++i)
          fetch16(whole ? sp.at[i] + (int64_t)s * (kBK * 2) : zeros, dst + i * (C::Threads * 16) + wbase);
      } else {
        const uint8_t* from = sp.at[0] + (int64_t)s * kBK * sp.ld;
        if ((s + 1) * kBK <= K) {
#pragma unroll
          for (int i = 0; i < C::P::Loads; ++i)
            fetch16(from + i * C::P::step_k * sp.ld, dst + i * (C::Threads * 16) + wbase);
        } else {
#pragma unroll
          for (int i = 0; i < C::P::Loads; ++i)
            fetch16(s * kBK + C::P::first_k() + i * C::P::step_k < K ? from + i * C::P::step_k * sp.ld : zeros,
                    dst + i * (C::Threads * 16) + wbase);
        }
      }
    };
    C::run((K + kBK - 1) / kBK, fill_p, fill_q, p0, q0, lane, acc);
  }
  const bool has_bias = a.bias && group < a.E;
#pragma unroll
  for (int i = 0; i < C::TP; ++i) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int n = n0 + p0 + 32 * i + 8 * v + 4 * (lane >> 5);
      if (n >= a.Nn) continue;
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (has_bias) {
        const T* bp = static_cast<const T*>(a.bias) + (int64_t)group * a.Nn + n;
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = to_f32(bp[c]);
      }
#pragma unroll
      for (int j = 0; j < C::TQ; ++j) {
        const int r = q0 + 32 * j + (lane & 31);
        if (r >= rows) continue;
        float o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = acc[i][j][4 * v + c] + b[c];
        const int64_t at = (first + r) * a.Nn + n;
        if (a.out_f32) store4(static_cast<float*>(a.out) + at, 4, o);
        else store4(static_cast<T*>(a.out) + at, 4, o);
      }
    }
  }
}

// dW[e][d][f] = Σ_p x[p][d] dy[p][f]: P is dy (columns f), Q is x (rows d).
template <typename T, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void grouped_mma_dw_kernel(GroupedArgs a, int ptiles, int qtiles) {
  typedef Core<T, false, false, BP, BQ, WP, WQ> C;
  const int64_t id = xcd_tile(blockIdx.x, gridDim.x);
  const int e = (int)(id / (ptiles * qtiles)), tile = (int)(id % (ptiles * qtiles));
  const int f0 = (tile % ptiles) * BP, d0 = (tile / ptiles) * BQ;
  const int64_t lo = offset_at(a, e), hi = offset_at(a, e + 1);
  const int n = (int)(hi > lo ? hi - lo : 0);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p0 = (wave % WP) * (BP / WP), q0 = (wave / WP) * (BQ / WQ);
  f32x16 acc[C::TP][C::TQ] = {};
  const int fc = f0 + C::P::column() < a.Nn ? f0 + C::P::column() : a.Nn - 8;
  const int dc = d0 + C::Q::column() < a.K ? d0 + C::Q::column() : a.K - 8;
  const T* dy = static_cast<const T*>(a.dy) + lo * a.lddy + fc;
  const T* x = static_cast<const T*>(a.x) + dc;
  const void* zeros = zero_page;
  const int wbase = wave * 1024;
  auto fill_p = [&](int s, uint8_t* dst) {
#pragma unroll
    for (int i = 0; i < C::P::Loads; ++i) {
      const int k = s * kBK + C::P::first_k() + i * C::P::step_k;
      fetch16(k < n ? dy + (int64_t)k * a.lddy : zeros, dst + i * (C::Threads * 16) + wbase);
    }
  };
  // (the rows' indices are read a step ahead)
  int src[C::Q::Loads];
  auto look = [&](int s) {
#pragma unroll
    for (int i = 0; i < C::Q::Loads; ++i) {
      const int k = s * kBK + C::Q::first_k() + i * C::Q::step_k;
      src[i] = k < n ? (int)source_row(a, lo + k) : 0;
    }
  };
  look(0);
  auto fill_q = [&](int s, uint8_t* dst) {
    const T* from[C::Q::Loads];
#pragma unroll
    for (int i = 0; i < C::Q::Loads; ++i) from[i] = x + (int64_t)src[i] * a.ldx;
    look(s + 1);
#pragma unroll
    for (int i = 0; i < C::Q::Loads; ++i) {
      const int k = s * kBK + C::Q::first_k() + i * C::Q::step_k;
      fetch16(k < n ? static_cast<const void*>(from[i]) : zeros, dst + i * (C::Threads * 16) + wbase);
    }
  };
  C::run((n + kBK - 1) / kBK, fill_p, fill_q, p0, q0, lane, acc);
  T* out = static_cast<T*>(a.out) + (int64_t)e * a.K * a.Nn;
#pragma unroll
  for (int i = 0; i < C::TP; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int f = f0 + p0 + 32 * i + 8 * v + 4 * (lane >> 5);
      if (f >= a.Nn) continue;
#pragma unroll
      for (int j = 0; j < C::TQ; ++j) {
        const int d = d0 + q0 + 32 * j + (lane & 31);
        if (d >= a.K) continue;
        float o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = acc[i][j][4 * v + c];
        store4(out + (int64_t)d * a.Nn + f, 4, o);
      }
    }
}

// db[e][f] = Σ_p dy[p][f]: 16 threads of 8 columns by 16 row lanes a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void grouped_db_kernel(GroupedArgs a) {
  __shared__ float part[16][128 + 4];
  const int e = blockIdx.y, f = blockIdx.x * 128 + (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4;
  const int64_t lo = offset_at(a, e), hi = offset_at(a, e + 1);
  float s[8] = {};
  if (f < a.Nn) {
    const T* dy = static_cast<const T*>(a.dy) + f;
#pragma unroll 4
    for (int64_t p = lo + r0; p < hi; p += 16) {
      float v[8];
      load_row(dy + p * a.lddy, 8, v);
#pragma unroll
      for (int c = 0; c < 8; ++c) s[c] += v[c];
    }
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) part[r0][(threadIdx.x & 15) * 8 + c] = s[c];
  __syncthreads();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (threadIdx.x < 128 && c < a.Nn) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) t += part[r][threadIdx.x];
    static_cast<T*>(a.dbias)[(int64_t)e * a.Nn + c] = (T)t;
  }
}

template <typename T, bool WKC>
void rows_mma(const GroupedArgs& a, hipStream_t s) {
  constexpr int BP = 256, BQ = 256;
  const int ntiles = (a.Nn + BP - 1) / BP;
  const int64_t grid = (a.M / BQ + a.E + 1) * ntiles;
  grouped_mma_kernel<T, WKC, BP, BQ, 4, 2><<<(unsigned)grid, 512, 0, s>>>(a, ntiles);
}

template <typename T>
void dw_mma(const GroupedArgs& a, hipStream_t s) {
  constexpr int BP = 256, BQ = 256;
  const int pt = (a.Nn + BP - 1) / BP, qt = (a.K + BQ - 1) / BQ;
  grouped_mma_dw_kernel<T, BP, BQ, 4, 2><<<(unsigned)(a.E * pt * qt), 512, 0, s>>>(a, pt, qt);
  if (a.dbias) grouped_db_kernel<T><<<dim3((unsigned)((a.Nn + 127) / 128), (unsigned)a.E), 256, 0, s>>>(a);
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

}  // namespace

// 16-bit elements in whole 16-byte chunks along every dimension that is read 16 bytes
// at a time.
bool grouped_mma_rows_ok(const GroupedArgs& a) {
  const int64_t outer = a.wk == 1 ? a.wn : a.wk;
  return a.elem != ELEM_F32 && a.K % 8 == 0 && a.Nn % 8 == 0 && a.ldx % 8 == 0 && a.we % 8 == 0 && outer % 8 == 0 &&
         aligned16(a.x) && aligned16(a.w) && aligned16(a.out);
}

bool grouped_mma_dw_ok(const GroupedArgs& a) {
  return a.elem != ELEM_F32 && a.K % 8 == 0 && a.Nn % 8 == 0 && a.ldx % 8 == 0 && a.lddy % 8 == 0 && aligned16(a.x) &&
         aligned16(a.dy) && aligned16(a.out);
}

void launch_grouped_mma(const GroupedArgs& a, hipStream_t s) {
  const bool kc = a.wk == 1 && a.wn != 1;
  if (a.elem == ELEM_BF16) kc ? rows_mma<bf16_t, true>(a, s) : rows_mma<bf16_t, false>(a, s);
  else kc ? rows_mma<_Float16, true>(a, s) : rows_mma<_Float16, false>(a, s);
}

void launch_grouped_mma_dw(const GroupedArgs& a, hipStream_t s) {
  if (a.elem == ELEM_BF16) dw_mma<bf16_t>(a, s);
  else dw_mma<_Float16>(a, s);
}

}  // namespace gx::layer
