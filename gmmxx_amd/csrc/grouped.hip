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
__global__ __launch_bounds__(kThreads) void grouped_rows_kernel(GroupedArgs a, int ntiles) {
  typedef Tile<T> Tl;
  __shared__ __align__(16) Tl t;
  int group, first, end, ntile;
  if (!find_tile<Tl::BM>(a, blockIdx.x, ntiles, group, first, end, ntile)) return;
  const int n0 = ntile * Tl::BN, tid = threadIdx.x;
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
        t.b[n][k] = n0 + n < a.Nn && k0 + k < a.K ? w[(int64_t)(k0 + k) * a.wk + (int64_t)(n0 + n) * a.wn] : (T)0.f;
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
        const int64_t at = (int64_t)(first + r) * a.Nn + n;
        if (a.out_f32) static_cast<float*>(a.out)[at] = acc[i][j][v] + bias;
        else static_cast<T*>(a.out)[at] = (T)(acc[i][j][v] + bias);
      }
  }
}

// One K x Nn tile of an expert's weight gradient, whole or (SPLIT) of one part of its positions.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kThreads) void grouped_dw_kernel(GroupedArgs a, int ktiles) {
  typedef Tile<T> Tl;
  typedef typename Result<T, SPLIT>::type O;
  __shared__ __align__(16) Tl t;
  const int e = blockIdx.y, k0 = (blockIdx.x % ktiles) * Tl::BM, n0 = (blockIdx.x / ktiles) * Tl::BN, tid = threadIdx.x;
  int lo = offset_at(a, e), hi = offset_at(a, e + 1);
  O* out = static_cast<O*>(a.out) + (int64_t)e * a.K * a.Nn;
  if constexpr (SPLIT) {
    split_part(lo, hi, blockIdx.z, gridDim.z);
    out = a.part + ((int64_t)blockIdx.z * a.E + e) * a.K * a.Nn;
  }
  const int lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  f32x4 acc[2][2] = {};
  for (int p0 = lo; p0 < hi; p0 += Tl::BK) {
    __syncthreads();
    for (int i = tid; i < Tl::BM * Tl::BK; i += kThreads) {
      const int m = i % Tl::BM, p = i / Tl::BM;
      T v = (T)0.f;
      if (p0 + p < hi && k0 + m < a.K) v = static_cast<const T*>(a.x)[source_row(a, p0 + p) * a.ldx + k0 + m];
      t.a[m][p] = v;
    }
    for (int i = tid; i < Tl::BN * Tl::BK; i += kThreads) {
      const int n = i % Tl::BN, p = i / Tl::BN;
      t.b[n][p] = p0 + p < hi && n0 + n < a.Nn ? static_cast<const T*>(a.dy)[(int64_t)(p0 + p) * a.lddy + n0 + n] : (T)0.f;
    }
    __syncthreads();
    multiply(t, wm, wn, lane, acc);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 16 * j + (lane & 15);
    if (n >= a.Nn) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int m = k0 + wm + 16 * i + (lane >> 4) * 4 + v;
        if (m < a.K) out[(int64_t)m * a.Nn + n] = (O)acc[i][j][v];
      }
  }
}

// db[e][n] = Σ_p dy[p][n]: 16 threads of one vector of columns by 16 row lanes a workgroup.
constexpr int kBiasLanes = 16;
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kThreads) void grouped_bias_kernel(GroupedArgs a) {
  constexpr int V = kVec<T>, Cols = 16 * V;
  __shared__ float part[kBiasLanes][Cols + 4];
  const int e = blockIdx.y, c = threadIdx.x & 15, n = blockIdx.x * Cols + c * V, r0 = threadIdx.x >> 4;
  int lo = offset_at(a, e), hi = offset_at(a, e + 1);
  if constexpr (SPLIT) split_part(lo, hi, blockIdx.z, gridDim.z);
  float s[V] = {};
  const T* dy = static_cast<const T*>(a.dy) + n;
#pragma unroll 4
  for (int p = lo + r0; p < hi; p += kBiasLanes) {
    float v[V];
    load_row(dy + p * a.lddy, a.Nn - n, v);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] += v[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[r0][c * V + i] = s[i];
  __syncthreads();
  const int col = blockIdx.x * Cols + threadIdx.x;
  if (threadIdx.x < Cols && col < a.Nn) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < kBiasLanes; ++r) t += part[r][threadIdx.x];
    if constexpr (SPLIT) a.bias_part[((int64_t)blockIdx.z * a.E + e) * a.Nn + col] = t;
    else static_cast<T*>(a.dbias)[(int64_t)e * a.Nn + col] = (T)t;
  }
}

// The parts' sums added in order: dW's (unless it has one part), then db's.
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_reduce_kernel(GroupedArgs a, int splits, int bias_splits) {
  const int64_t weights = splits > 1 ? (int64_t)a.E * a.K * a.Nn : 0;
  const int64_t biases = bias_splits > 1 ? (int64_t)a.E * a.Nn : 0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < weights + biases;
       i += (int64_t)gridDim.x * kThreads) {
    const bool w = i < weights;
    const float* p = w ? a.part + i : a.bias_part + (i - weights);
    const int64_t stride = w ? weights : biases;
    float s = 0.f;
#pragma unroll 8
    for (int q = 0; q < (w ? splits : bias_splits); ++q) s += p[q * stride];
    if (w) static_cast<T*>(a.out)[i] = (T)s;
    else static_cast<T*>(a.dbias)[i - weights] = (T)s;
  }
}

template <typename T>
void rows_typed(const GroupedArgs& a, hipStream_t s) {
  typedef Tile<T> Tl;
  const int ntiles = (a.Nn + Tl::BN - 1) / Tl::BN;
  grouped_rows_kernel<T><<<(unsigned)((a.M / Tl::BM + a.E + 1) * ntiles), kThreads, 0, s>>>(a, ntiles);
}

int64_t dw_tiles(int64_t E, int64_t K, int64_t N) { return E * ((K + 63) / 64) * ((N + 63) / 64); }

template <typename T>
void dw_typed(const GroupedArgs& a, int splits, hipStream_t s) {
  const int ktiles = (a.K + 63) / 64;
  const dim3 grid((unsigned)(ktiles * ((a.Nn + 63) / 64)), (unsigned)a.E, (unsigned)splits);
  if (splits == 1) grouped_dw_kernel<T, false><<<grid, kThreads, 0, s>>>(a, ktiles);
  else grouped_dw_kernel<T, true><<<grid, kThreads, 0, s>>>(a, ktiles);
}

// The rest of the weight gradient's pass: db, and the sums of parts.
template <typename T>
void dw_rest(const GroupedArgs& a, int splits, int bias_splits, hipStream_t s) {
  if (a.dbias) {
    const dim3 grid((unsigned)((a.Nn + 16 * kVec<T> - 1) / (16 * kVec<T>)), (unsigned)a.E, (unsigned)bias_splits);
    if (bias_splits == 1) grouped_bias_kernel<T, false><<<grid, kThreads, 0, s>>>(a);
    else grouped_bias_kernel<T, true><<<grid, kThreads, 0, s>>>(a);
  }
  const int64_t all = (splits > 1 ? (int64_t)a.E * a.K * a.Nn : 0) + (bias_splits > 1 ? (int64_t)a.E * a.Nn : 0);
  const int64_t blocks = (all + kThreads - 1) / kThreads;
  if (all) grouped_reduce_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), kThreads, 0, s>>>(a, splits, bias_splits);
}

int general_dw_splits(int64_t M, int64_t E, int64_t K, int64_t N) { return parts_of(M, E, dw_tiles(E, K, N), 1024, 256); }
int bias_splits(int64_t M, int64_t E, int64_t N) { return parts_of(M, E, E * ((N + 127) / 128), 2048, 128); }

}  // namespace

int parts_of(int64_t M, int64_t E, int64_t groups, int64_t want, int64_t least) {
  const int64_t by_groups = (want + groups - 1) / groups, by_rows = M / (E * least);
  const int64_t s = by_groups < by_rows ? by_groups : by_rows;
  return (int)(s < 1 ? 1 : s < 65535 ? s : 65535);
}

int64_t grouped_workspace_bytes(int64_t M, int64_t E, int64_t K, int64_t N) {
  const int a = general_dw_splits(M, E, K, N), b = grouped_mma_dw_splits(M, E, K, N), s = a > b ? a : b;
  const int t = bias_splits(M, E, N);
  return ((s > 1 ? s * E * K * N : 0) + (t > 1 ? t * E * N : 0)) * (int64_t)sizeof(float);
}

void launch_grouped(const GroupedArgs& a, hipStream_t s) {
  if (grouped_few_better(a)) launch_grouped_few(a, s);
  else if (grouped_mma_rows_ok(a)) launch_grouped_mma(a, s);
  else if (a.elem == ELEM_F32) rows_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) rows_typed<bf16_t>(a, s);
  else rows_typed<_Float16>(a, s);
}

void launch_grouped_dw(const GroupedArgs& args, hipStream_t s) {
  GroupedArgs a = args;
  const bool mma = grouped_mma_dw_ok(a);
  const int splits = mma ? grouped_mma_dw_splits(a.M, a.E, a.K, a.Nn) : general_dw_splits(a.M, a.E, a.K, a.Nn);
  const int bs = a.dbias ? bias_splits(a.M, a.E, a.Nn) : 1;
  a.bias_part = a.part + (splits > 1 ? (int64_t)splits * a.E * a.K * a.Nn : 0);
  if (mma) launch_grouped_mma_dw(a, splits, s);
  else if (a.elem == ELEM_F32) dw_typed<float>(a, splits, s);
  else if (a.elem == ELEM_BF16) dw_typed<bf16_t>(a, splits, s);
  else dw_typed<_Float16>(a, splits, s);
  if (a.elem == ELEM_F32) dw_rest<float>(a, splits, bs, s);
  else if (a.elem == ELEM_BF16) dw_rest<bf16_t>(a, splits, bs, s);
  else dw_rest<_Float16>(a, splits, bs, s);
}

}  // namespace gx::layer
