// Layer norm of rows and its gradient.
//
//   y = (x - μ) ρ w + b,  μ = mean x,  ρ = 1 / sqrt(mean (x - μ)² + ε)
// and with h = (x - μ) ρ, g = dy·w:
//   dx = ρ (g - mean g - h mean(g h)),  dw = Σ_rows dy·h,  db = Σ_rows dy.
//
// A group of G threads holds a row in registers (up to 16 elements a thread, 32 and
// 64 for the widest rows), so x is read once and the mean is taken out before the
// squares are summed: rows whose mean is large beside their spread lose nothing.
// Everything is fp32; the one rounding is the store.  G is the smallest group that
// holds the row, so narrow rows share a wave.  Groups stride over the rows and keep
// w and b in registers.
//
// The backward pass keeps each column's Σ dy·h and Σ dy in registers over the rows
// of its workgroup, writes one partial row per workgroup, and a second kernel adds
// the partials: two fixed orders of additions, no atomics.

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

namespace {

constexpr int kNormThreads = 256;
constexpr int kFwdMaxBlocks = 2048;

template <typename T, typename WT, int G, int NV>
struct Norm {
  static constexpr int V = kVec<T>;
  static constexpr int Threads = G > kNormThreads ? G : kNormThreads;
  static constexpr int RPB = Threads / G;     // rows of a workgroup at a time

  // This thread's elements of a row: vector i covers columns (i G + lane) V ...
  __device__ static __forceinline__ int col(int i, int lane) { return (i * G + lane) * V; }

  __device__ static __forceinline__ void load(const T* row, int D, int lane, float (&v)[NV][V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load_row(row + col(i, lane), D - col(i, lane), v[i]);
  }
  __device__ static __forceinline__ void load_param(const void* p, int D, int lane, float fill, float (&v)[NV][V]) {
    const WT* w = static_cast<const WT*>(p);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = col(i, lane) + j;
        v[i][j] = c < D ? (w ? to_f32(w[c]) : fill) : 0.f;
      }
    }
  }
};

template <typename T, typename WT, int G, int NV>
__global__ __launch_bounds__((Norm<T, WT, G, NV>::Threads)) void norm_fwd_kernel(NormArgs a) {
  using L = Norm<T, WT, G, NV>;
  constexpr int V = L::V;
  __shared__ float red[2][16];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float w[NV][V], b[NV][V];
  L::load_param(a.weight, a.D, lane, 1.f, w);
  L::load_param(a.bias, a.D, lane, 0.f, b);
  const float inv = 1.f / (float)a.D;
  for (int64_t row = (int64_t)blockIdx.x * L::RPB + sub; row < a.N; row += (int64_t)gridDim.x * L::RPB) {
    float x[NV][V];
    L::load(static_cast<const T*>(a.x) + row * a.ldx, a.D, lane, x);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += x[i][j];
    const float mean = group_sum<G>(s, red, turn) * inv;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] = L::col(i, lane) + j < a.D ? x[i][j] - mean : 0.f;
        q = fmaf(x[i][j], x[i][j], q);
      }
    const float rstd = 1.f / sqrtf(group_sum<G>(q, red, turn) * inv + a.eps);
    T* out = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = fmaf(x[i][j] * rstd, w[i][j], b[i][j]);
      store_row(out + L::col(i, lane), a.D - L::col(i, lane), x[i]);
    }
    if (lane == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename WT, int G, int NV>
__global__ __launch_bounds__((Norm<T, WT, G, NV>::Threads)) void norm_bwd_kernel(NormArgs a) {
  using L = Norm<T, WT, G, NV>;
  constexpr int V = L::V;
  __shared__ float red[2][16];
  __shared__ float cols[L::RPB > 1 ? L::Threads * NV * V : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float w[NV][V], dw[NV][V], db[NV][V];
  L::load_param(a.weight, a.D, lane, 1.f, w);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  const float inv = 1.f / (float)a.D;
  for (int64_t row = (int64_t)blockIdx.x * L::RPB + sub; row < a.N; row += (int64_t)gridDim.x * L::RPB) {
    float h[NV][V], g[NV][V];
    L::load(static_cast<const T*>(a.x) + row * a.ldx, a.D, lane, h);
    L::load(static_cast<const T*>(a.dy) + row * a.lddy, a.D, lane, g);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = L::col(i, lane) + j < a.D ? (h[i][j] - mean) * rstd : 0.f;
        dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
        db[i][j] += g[i][j];
        g[i][j] *= w[i][j];
        sg += g[i][j];
        sgh = fmaf(g[i][j], h[i][j], sgh);
      }
    const float mg = group_sum<G>(sg, red, turn) * inv;
    const float mgh = group_sum<G>(sgh, red, turn) * inv;
    T* out = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) g[i][j] = rstd * (g[i][j] - mg - h[i][j] * mgh);
      store_row(out + L::col(i, lane), a.D - L::col(i, lane), g[i]);
    }
  }
  if (!a.part) return;
  float* part = a.part + (size_t)blockIdx.x * 2 * a.D;
  if constexpr (L::RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = L::col(i, lane) + j;
        if (c < a.D) {
          part[c] = dw[i][j];
          part[a.D + c] = db[i][j];
        }
      }
  } else {
    constexpr int W = G * NV * V;    // columns held by a group
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) cols[sub * W + L::col(i, lane) + j] = half ? db[i][j] : dw[i][j];
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += L::Threads) {
        float s = 0.f;
#pragma unroll 8
        for (int r = 0; r < L::RPB; ++r) s += cols[r * W + c];
        part[half * a.D + c] = s;
      }
    }
  }
}

// Sums the workgroups' partial rows: 16 columns by 64 row lanes a workgroup.
constexpr int kSumCols = 16, kSumRows = 64;
template <typename WT>
__global__ __launch_bounds__(kSumCols* kSumRows) void norm_sum_kernel(NormArgs a, int blocks) {
  __shared__ float red[kSumRows][kSumCols + 1];
  const int cl = threadIdx.x % kSumCols, r0 = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + cl;     // column of the 2 D wide partial rows
  float s = 0.f;
  if (c < 2 * a.D) {
#pragma unroll 4
    for (int r = r0; r < blocks; r += kSumRows) s += a.part[(size_t)r * 2 * a.D + c];
  }
  red[r0][cl] = s;
  __syncthreads();
  for (int half = kSumRows / 2; half >= 1; half /= 2) {
    if (r0 < half) red[r0][cl] += red[r0 + half][cl];
    __syncthreads();
  }
  if (r0 == 0 && c < 2 * a.D) {
    WT* out = static_cast<WT*>(c < a.D ? a.dweight : a.dbias);
    if (out) out[c < a.D ? c : c - a.D] = (WT)red[0][cl];
  }
}

// Calls f.template operator()<G, NV>() for the smallest group that holds a row of D.
template <typename T, typename F>
void with_group(int D, F&& f) {
  constexpr int N16 = 16 / kVec<T>;    // vectors of 16 elements
  if (D <= 8 * 16) f.template operator()<8, N16>();
  else if (D <= 16 * 16) f.template operator()<16, N16>();
  else if (D <= 32 * 16) f.template operator()<32, N16>();
  else if (D <= 64 * 16) f.template operator()<64, N16>();
  else if (D <= 256 * 16) f.template operator()<256, N16>();
  else if (D <= 256 * 32) f.template operator()<256, 2 * N16>();
  else f.template operator()<1024, 4 * N16>();
}

template <typename F>
void with_elems(int x_elem, int w_elem, F&& f) {
  if (x_elem == ELEM_F32) f.template operator()<float, float>();
  else if (x_elem == ELEM_BF16 && w_elem == ELEM_F32) f.template operator()<__bf16, float>();
  else if (x_elem == ELEM_BF16) f.template operator()<__bf16, __bf16>();
  else if (w_elem == ELEM_F32) f.template operator()<_Float16, float>();
  else f.template operator()<_Float16, _Float16>();
}

int rows_per_block(int D) {
  if (D > 64 * 16) return 1;
  const int g = D <= 8 * 16 ? 8 : D <= 16 * 16 ? 16 : D <= 32 * 16 ? 32 : 64;
  return kNormThreads / g;
}

struct FwdOp {
  const NormArgs& a; hipStream_t s;
  template <typename T, typename WT> void operator()() {
    Go<T, WT> go{a, s};
    with_group<T>(a.D, go);
  }
  template <typename T, typename WT> struct Go {
    const NormArgs& a; hipStream_t s;
    template <int G, int NV> void operator()() {
      using L = Norm<T, WT, G, NV>;
      const int64_t need = (a.N + L::RPB - 1) / L::RPB;
      const int grid = (int)(need < kFwdMaxBlocks ? need : kFwdMaxBlocks);
      norm_fwd_kernel<T, WT, G, NV><<<grid, L::Threads, 0, s>>>(a);
    }
  };
};

struct BwdOp {
  const NormArgs& a; hipStream_t s; int blocks;
  template <typename T, typename WT> void operator()() {
    Go<T, WT> go{a, s, blocks};
    with_group<T>(a.D, go);
    if (a.part) norm_sum_kernel<WT><<<(2 * a.D + kSumCols - 1) / kSumCols, kSumCols * kSumRows, 0, s>>>(a, blocks);
  }
  template <typename T, typename WT> struct Go {
    const NormArgs& a; hipStream_t s; int blocks;
    template <int G, int NV> void operator()() {
      norm_bwd_kernel<T, WT, G, NV><<<blocks, Norm<T, WT, G, NV>::Threads, 0, s>>>(a);
    }
  };
};

}  // namespace

int norm_blocks(int64_t N, int D) {
  const int rpb = rows_per_block(D);
  const int64_t need = (N + rpb - 1) / rpb;
  return (int)(need < kNormMaxBlocks ? need : kNormMaxBlocks);
}

void launch_norm_fwd(const NormArgs& a, hipStream_t s) {
  FwdOp op{a, s};
  with_elems(a.x_elem, a.w_elem, op);
}

void launch_norm_bwd(const NormArgs& a, hipStream_t s) {
  BwdOp op{a, s, norm_blocks(a.N, a.D)};
  with_elems(a.x_elem, a.w_elem, op);
}

}  // namespace gx::layer
