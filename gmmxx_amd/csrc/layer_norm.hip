// Layer norm of rows and its gradient.
//
//   y = (x - μ) ρ w + b,  μ = mean x,  ρ = 1 / sqrt(mean (x - μ)² + ε)
// and with h = (x - μ) ρ, g = dy·w:
//   dx = ρ (g - mean g - h mean(g h)),  dw = Σ_rows dy·h,  db = Σ_rows dy.
//
// A group of G threads holds a row in registers (up to 16 elements a thread, 32 above
// 16384 columns and 64 above 32768, where part of it spills), so x is read once and
// the mean is taken out before the squares are summed.  A sum's mean is off by units of
// the mean itself; the mean of what it left, which comes with the squares, is taken out
// too, so rows whose mean is large beside their spread keep the spread's precision (the
// backward pass reads the two together, rounded to fp32: half a unit of the mean).
// Everything is fp32; the one rounding is the store.  G is the smallest group that holds
// the row, so narrow rows share a wave.  Groups stride over the rows, keep w and b in
// registers and have the next row's loads in flight while a row's sums pass between lanes.
//
// The backward pass keeps each column's Σ dy·h and Σ dy in registers over the rows
// of its workgroup, writes one partial row per workgroup, and a second kernel adds
// the partials: two fixed orders of additions, no atomics.
//
// Bound by bytes.  16384 x 4096 bf16: forward 48 us (5.5 TB/s), backward 87 us (4.6 TB/s),
// the partials' sum 8 us; 100003 x 100 fp32: 19 us (4.3), 24 us (5.1) and 4 us.  One row
// is a launch: 2.6 us.

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

namespace {

constexpr int kNormThreads = 256;
constexpr int kFwdMaxBlocks = 1024;

template <typename T, typename WT, int G, int NV, bool SHORT>
struct Norm {
  static constexpr int V = kVec<T>;
  static constexpr int Threads = G > kNormThreads ? G : kNormThreads;
  static constexpr int RPB = Threads / G;     // rows of a workgroup at a time

  // This thread's elements of a row: vector i covers columns (i G + lane) V ...
  __device__ static __forceinline__ int col(int i, int lane) { return (i * G + lane) * V; }

  __device__ static __forceinline__ void fetch(const T* row, int D, int lane, uint4 (&u)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = fetch16<SHORT>(row + col(i, lane), D - col(i, lane));
  }
  __device__ static __forceinline__ void unpack(const uint4 (&u)[NV], int D, int lane, float (&v)[NV][V]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack16<T>(keep16<SHORT, T>(u[i], D - col(i, lane), D), v[i]);
  }
  // This thread's columns of w or b, or `fill` where there is none.
  __device__ static __forceinline__ void load_param(const void* p, int D, int lane, float fill, float (&v)[NV][V]) {
    if (!p) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = fill;
      return;
    }
    constexpr int H = V / kVec<WT>, W = kVec<WT>;      // vectors of w for one of x
    const WT* w = static_cast<const WT*>(p);
    uint4 u[NV][H];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int h = 0; h < H; ++h) u[i][h] = fetch16<SHORT>(w + col(i, lane) + h * W, D - col(i, lane) - h * W);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        float e[W];
        unpack16<WT>(keep16<SHORT, WT>(u[i][h], D - col(i, lane) - h * W, D), e);
#pragma unroll
        for (int j = 0; j < W; ++j) v[i][h * W + j] = e[j];
      }
  }
};

// a b, rounded: not fused into what uses it.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

template <typename T, typename WT, int G, int NV, bool SHORT>
__global__ __launch_bounds__((Norm<T, WT, G, NV, SHORT>::Threads)) void norm_fwd_kernel(NormArgs a) {
  using L = Norm<T, WT, G, NV, SHORT>;
  constexpr int V = L::V;
  __shared__ float red_sum[2][16][1], red[2][16][2];
  int turn_sum = 0, turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int64_t step = (int64_t)gridDim.x * L::RPB;
  int64_t row = (int64_t)blockIdx.x * L::RPB + sub;
  if (row >= a.N) return;
  const T* x0 = static_cast<const T*>(a.x);
  uint4 next[NV];
  L::fetch(x0 + row * a.ldx, a.D, lane, next);
  float w[NV][V], b[NV][V];
  L::load_param(a.weight, a.D, lane, 1.f, w);
  L::load_param(a.bias, a.D, lane, 0.f, b);
  const float inv = 1.f / (float)a.D;
  for (; row < a.N; row += step) {
    float x[NV][V];
    L::unpack(next, a.D, lane, x);
    if (row + step < a.N) L::fetch(x0 + (row + step) * a.ldx, a.D, lane, next);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += x[i][j];
    group_sums<G>(s, red_sum, turn_sum);
    const float about = product(s[0], inv);
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] = L::col(i, lane) + j < a.D ? x[i][j] - about : 0.f;
        q[0] = fmaf(x[i][j], x[i][j], q[0]);
        q[1] += x[i][j];
      }
    group_sums<G>(q, red, turn);
    const float rest = q[1] * inv, var = q[0] * inv - rest * rest;
    const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);      // (NaN stays)
    const float shift = -rest * rstd;
    T* out = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = fmaf(fmaf(x[i][j], rstd, shift), w[i][j], b[i][j]);
      store_row(out + L::col(i, lane), a.D - L::col(i, lane), x[i]);
    }
    if (lane == 0 && a.mean) {
      a.mean[row] = about + rest;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename WT, int G, int NV, bool SHORT>
__global__ __launch_bounds__((Norm<T, WT, G, NV, SHORT>::Threads)) void norm_bwd_kernel(NormArgs a) {
  using L = Norm<T, WT, G, NV, SHORT>;
  constexpr int V = L::V;
  __shared__ float red[2][16][2];
  __shared__ float cols[L::RPB > 1 ? L::Threads * NV * V : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const int64_t step = (int64_t)gridDim.x * L::RPB;
  int64_t row = (int64_t)blockIdx.x * L::RPB + sub;
  const T *x0 = static_cast<const T*>(a.x), *dy0 = static_cast<const T*>(a.dy);
  uint4 next_x[NV], next_dy[NV];
  float next_mean = 0.f, next_rstd = 0.f;
  auto fetch = [&](int64_t r) {
    L::fetch(x0 + r * a.ldx, a.D, lane, next_x);
    L::fetch(dy0 + r * a.lddy, a.D, lane, next_dy);
    next_mean = a.mean[r];
    next_rstd = a.rstd[r];
  };
  if (row < a.N) fetch(row);
  float w[NV][V], dw[NV][V], db[NV][V];
  L::load_param(a.weight, a.D, lane, 1.f, w);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  const float inv = 1.f / (float)a.D;
  for (; row < a.N; row += step) {
    float h[NV][V], g[NV][V];
    L::unpack(next_x, a.D, lane, h);
    L::unpack(next_dy, a.D, lane, g);
    const float mean = next_mean, rstd = next_rstd;
    if (row + step < a.N) fetch(row + step);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = L::col(i, lane) + j < a.D ? (h[i][j] - mean) * rstd : 0.f;
        dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
        db[i][j] += g[i][j];
        g[i][j] *= w[i][j];
        s[0] += g[i][j];
        s[1] = fmaf(g[i][j], h[i][j], s[1]);
      }
    group_sums<G>(s, red, turn);
    const float mg = s[0] * inv, mgh = s[1] * inv;
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

// Calls f.template operator()<G, NV, SHORT>() for the smallest group that holds a row of D.
// (4096 x 16384 bf16: backward 199 us by 1024 threads, 207 us by 512 with twice the vectors)
template <typename T, typename F>
void with_group(int D, F&& f) {
  constexpr int N16 = 16 / kVec<T>;    // vectors of 16 elements
  if (D < kVec<T>) f.template operator()<8, N16, true>();
  else if (D <= 8 * 16) f.template operator()<8, N16, false>();
  else if (D <= 16 * 16) f.template operator()<16, N16, false>();
  else if (D <= 32 * 16) f.template operator()<32, N16, false>();
  else if (D <= 64 * 16) f.template operator()<64, N16, false>();
  else if (D <= 256 * 16) f.template operator()<256, N16, false>();
  else if (D <= 512 * 16) f.template operator()<512, N16, false>();
  else if (D <= 1024 * 16) f.template operator()<1024, N16, false>();
  else if (D <= 1024 * 32) f.template operator()<1024, 2 * N16, false>();
  else f.template operator()<1024, 4 * N16, false>();
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
    template <int G, int NV, bool SHORT> void operator()() {
      using L = Norm<T, WT, G, NV, SHORT>;
      const int64_t need = (a.N + L::RPB - 1) / L::RPB;
      const int grid = (int)(need < kFwdMaxBlocks ? need : kFwdMaxBlocks);
      norm_fwd_kernel<T, WT, G, NV, SHORT><<<grid, L::Threads, 0, s>>>(a);
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
    template <int G, int NV, bool SHORT> void operator()() {
      norm_bwd_kernel<T, WT, G, NV, SHORT><<<blocks, Norm<T, WT, G, NV, SHORT>::Threads, 0, s>>>(a);
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
