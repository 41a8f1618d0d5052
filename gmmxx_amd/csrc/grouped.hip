// Matrix products grouped by expert, with ragged group sizes.
//
//   out[p] = x[rows[p]] W[e] + b[e]          for the positions p of group e      (rows kernel)
//   dW[e]  = Σ_p x[rows[p]]ᵀ dy[p],  db[e] = Σ_p dy[p]                           (weight-gradient kernel)
// The gradient with respect to x is the rows kernel on dy with the weight's two
// strides exchanged.
//
// The groups' offsets stay on the device: the grid is sized for the most tiles that
// any offsets can give (M / tile + E + 1), and each workgroup finds its group by
// counting tiles.  Positions past offsets[E] get rows of zeros.  Offsets and row
// indices are clamped to their arrays, so no values of theirs lead out of bounds.

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

// Products of one 16 x 16 tile: 32-deep for 16-bit elements, 4-deep for fp32.
template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
  static constexpr int K = 32, Per = 8;
  typedef bf16x8 Frag;
  __device__ static __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<_Float16> {
  static constexpr int K = 32, Per = 8;
  typedef f16x8 Frag;
  __device__ static __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  static constexpr int K = 4, Per = 1;
  typedef float Frag;
  __device__ static __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
};

// A 64 x 64 tile by four waves of 32 x 32, both operands staged in LDS with the
// reduction index innermost.
constexpr int kThreads = 256;
template <typename T>
struct Tile {
  static constexpr int BM = 64, BN = 64, BK = sizeof(T) == 2 ? 64 : 32;
  static constexpr int LD = BK + 16 / (int)sizeof(T);    // 16 bytes of padding: rows start on other banks
  T a[BM][LD];
  T b[BN][LD];
};

template <typename T>
__device__ __forceinline__ void multiply(const Tile<T>& t, int wm, int wn, int lane, f32x4 (&acc)[2][2]) {
  typedef Mma<T> M;
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int k = 0; k < Tile<T>::BK; k += M::K) {
    typename M::Frag fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = *reinterpret_cast<const typename M::Frag*>(&t.a[wm + 16 * i + r][k + q * M::Per]);
      fb[i] = *reinterpret_cast<const typename M::Frag*>(&t.b[wn + 16 * i + r][k + q * M::Per]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = M::run(fa[i], fb[j], acc[i][j]);
  }
}

// One row tile by one column tile of out = x W + b.
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_rows_kernel(GroupedArgs a) {
  typedef Tile<T> Tl;
  __shared__ __align__(16) Tl t;
  int group;
  int64_t first, end;
  if (!find_tile<Tl::BM>(a, blockIdx.x, group, first, end)) return;
  const int n0 = blockIdx.y * Tl::BN, tid = threadIdx.x;
  const int rows = (int)(end - first < Tl::BM ? end - first : Tl::BM);
  const int lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  if (group < a.E) {
    const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.we;
    const bool k_inner = a.wk == 1;
    for (int k0 = 0; k0 < a.K; k0 += Tl::BK) {
      __syncthreads();
      for (int i = tid; i < Tl::BM * Tl::BK; i += kThreads) {
        const int r = i / Tl::BK, k = i % Tl::BK;
        T v = (T)0.f;
        if (r < rows && k0 + k < a.K) v = static_cast<const T*>(a.x)[source_row(a, first + r) * a.ldx + k0 + k];
        t.a[r][k] = v;
      }
      for (int i = tid; i < Tl::BN * Tl::BK; i += kThreads) {
        const int n = k_inner ? i / Tl::BK : i % Tl::BN, k = k_inner ? i % Tl::BK : i / Tl::BN;
        t.b[n][k] = n0 + n < a.Nn && k0 + k < a.K ? w[(k0 + k) * a.wk + (n0 + n) * a.wn] : (T)0.f;
      }
      __syncthreads();
      multiply(t, wm, wn, lane, acc);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 16 * j + (lane & 15);
    if (n >= a.Nn) continue;
    const float bias = a.bias && group < a.E ? to_f32(static_cast<const T*>(a.bias)[(int64_t)group * a.Nn + n]) : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = wm + 16 * i + (lane >> 4) * 4 + v;
        if (r >= rows) continue;
        const int64_t at = (first + r) * a.Nn + n;
        if (a.out_f32) static_cast<float*>(a.out)[at] = acc[i][j][v] + bias;
        else static_cast<T*>(a.out)[at] = (T)(acc[i][j][v] + bias);
      }
  }
}

// One K x Nn tile of an expert's weight gradient; the first row of tiles adds db.
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_dw_kernel(GroupedArgs a) {
  typedef Tile<T> Tl;
  __shared__ __align__(16) Tl t;
  const int e = blockIdx.z, k0 = blockIdx.x * Tl::BM, n0 = blockIdx.y * Tl::BN, tid = threadIdx.x;
  const int64_t lo = offset_at(a, e), hi = offset_at(a, e + 1);
  const int lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  float db = 0.f;
  for (int64_t p0 = lo; p0 < hi; p0 += Tl::BK) {
    __syncthreads();
    for (int i = tid; i < Tl::BM * Tl::BK; i += kThreads) {
      const int m = i % Tl::BM, p = i / Tl::BM;
      T v = (T)0.f;
      if (p0 + p < hi && k0 + m < a.K) v = static_cast<const T*>(a.x)[source_row(a, p0 + p) * a.ldx + k0 + m];
      t.a[m][p] = v;
    }
    for (int i = tid; i < Tl::BN * Tl::BK; i += kThreads) {
      const int n = i % Tl::BN, p = i / Tl::BN;
      t.b[n][p] = p0 + p < hi && n0 + n < a.Nn ? static_cast<const T*>(a.dy)[(p0 + p) * a.lddy + n0 + n] : (T)0.f;
    }
    __syncthreads();
    multiply(t, wm, wn, lane, acc);
    if (a.dbias && blockIdx.x == 0 && tid < Tl::BN) {
#pragma unroll 8
      for (int p = 0; p < Tl::BK; ++p) db += to_f32(t.b[tid][p]);
    }
  }
  T* out = static_cast<T*>(a.out) + (int64_t)e * a.K * a.Nn;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 16 * j + (lane & 15);
    if (n >= a.Nn) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int m = k0 + wm + 16 * i + (lane >> 4) * 4 + v;
        if (m < a.K) out[(int64_t)m * a.Nn + n] = (T)acc[i][j][v];
      }
  }
  if (a.dbias && blockIdx.x == 0 && tid < Tl::BN && n0 + tid < a.Nn)
    static_cast<T*>(a.dbias)[(int64_t)e * a.Nn + n0 + tid] = (T)db;
}

template <typename T>
void rows_typed(const GroupedArgs& a, hipStream_t s) {
  typedef Tile<T> Tl;
  const int64_t tiles = a.M / Tl::BM + a.E + 1;
  dim3 grid((unsigned)tiles, (unsigned)((a.Nn + Tl::BN - 1) / Tl::BN));
  grouped_rows_kernel<T><<<grid, kThreads, 0, s>>>(a);
}

template <typename T>
void dw_typed(const GroupedArgs& a, hipStream_t s) {
  typedef Tile<T> Tl;
  dim3 grid((unsigned)((a.K + Tl::BM - 1) / Tl::BM), (unsigned)((a.Nn + Tl::BN - 1) / Tl::BN), (unsigned)a.E);
  grouped_dw_kernel<T><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

void launch_grouped(const GroupedArgs& a, hipStream_t s) {
  if (grouped_mma_rows_ok(a)) launch_grouped_mma(a, s);
  else if (a.elem == ELEM_F32) rows_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) rows_typed<bf16_t>(a, s);
  else rows_typed<_Float16>(a, s);
}

void launch_grouped_dw(const GroupedArgs& a, hipStream_t s) {
  if (grouped_mma_dw_ok(a)) launch_grouped_mma_dw(a, s);
  else if (a.elem == ELEM_F32) dw_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) dw_typed<bf16_t>(a, s);
  else dw_typed<_Float16>(a, s);
}

}  // namespace gx::layer
