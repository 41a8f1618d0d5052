// Grouped products of few rows (serving): out[p] = x[rows[p]] W[e] + b[e] where groups have a handful of rows.
//
// Each weight is used once or a few times, so the pass is a stream of the chosen experts' weights: a workgroup
// of eight waves takes up to four rows of one group and 8 vectors of columns, and reads its weights once from
// memory, 16 bytes a lane, straight to registers; the products are fp32 multiply-adds.  Larger groups take
// several workgroups, which find the weights in cache.  The reduction is cut over the lanes and waves of the
// workgroup and joined in a fixed order.  Any width, stride and type.  Bound by the weights' bytes and by the
// chain of waits before them (offsets, then weights and rows together, then the join): 8 rows of 8 experts,
// 1024 -> 2048 bf16, 34 MB from memory in 14.4 us.

#include <type_traits>

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kRows = 4;         // of a workgroup
constexpr int kChunk = 1024;     // reduction elements of x staged at a time

// x's rows as xs[k][row], zeros past K (up to a multiple of 128).
template <typename T>
__device__ __forceinline__ void stage(const GroupedArgs& a, int first, int rows, int k0, float4* xs) {
  const int r = threadIdx.x & 3, lane = threadIdx.x >> 2;
  const int at = first + (r < rows ? r : 0);
  const T* x = static_cast<const T*>(a.x) + in_x(a, a.rows ? a.rows[at] : at) * a.ldx + k0;
  const int most = min(kChunk, a.K - k0);
#pragma unroll
  for (int i = 0; i < kChunk / (kThreads / 4); ++i) {
    if (i * (kThreads / 4) >= most) break;
    const int k = lane + i * (kThreads / 4);
    reinterpret_cast<float*>(xs)[k * 4 + r] = r < rows && k < most ? to_f32(x[k]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ float element(const uint4& v, int i) {
  union { uint4 u; T t[kVec<T>]; } r;
  r.u = v;
  return to_f32(r.t[i]);
}

__device__ __forceinline__ void add_products(float (&acc)[kRows], const float4& x, float w) {
  acc[0] = fmaf(x.x, w, acc[0]);
  acc[1] = fmaf(x.y, w, acc[1]);
  acc[2] = fmaf(x.z, w, acc[2]);
  acc[3] = fmaf(x.w, w, acc[3]);
}

// Whole chunks without conditions (their loads are all in flight before the first is used), then the rest.
template <typename F>
__device__ __forceinline__ void over_chunks(int K, F&& chunk) {
  int k0 = 0;
  for (; k0 + kChunk <= K; k0 += kChunk) chunk(k0, std::true_type());
  if (k0 < K) chunk(k0, std::false_type());
}

template <typename T, bool KC, bool SHORT>
__global__ __launch_bounds__(kThreads) void grouped_few_kernel(GroupedArgs a, int ntiles) {
  constexpr int V = kVec<T>, Cols = 8 * V;     // columns of a workgroup
  constexpr int Loads = 16;                    // 16-byte loads of a thread for a chunk, all in flight at once
  __shared__ __align__(16) float4 xs[kChunk];
  __shared__ float part[kWaves][kRows][Cols];
  int group, first, end, ntile;
  if (!find_tile<kRows>(a, block_id(), ntiles, group, first, end, ntile)) return;
  const int rows = min(end - first, kRows), n0 = ntile * Cols;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (group < a.E) {
    const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.we;
    const int c = lane & 7;
    uint4 v[Loads];
    if constexpr (KC) {
      // 8 lanes share a column and V columns a thread; a wave takes every 8th stretch of 8 V reduction elements.
      constexpr int Span = 8 * V, Parts = kChunk / (Span * kWaves);
      static_assert(V * Parts == Loads, "");
      float acc[V][kRows] = {};
      auto chunk = [&](int k0, auto whole) {
#pragma unroll
        for (int q = 0; q < Parts; ++q)
#pragma unroll
          for (int b = 0; b < V; ++b) {
            if (!whole && k0 + (q * kWaves + wave) * Span >= a.K) continue;
            const int n = min(n0 + 8 * b + (lane >> 3), a.Nn - 1), k = k0 + (q * kWaves + wave) * Span + c * V;
            v[q * V + b] = fetch16<SHORT>(w + n * a.wn + k, whole ? V : a.K - k);
          }
        __syncthreads();
        stage<T>(a, first, rows, k0, xs);
        __syncthreads();
        if (!whole) {
#pragma unroll
          for (int q = 0; q < Parts; ++q)
#pragma unroll
            for (int b = 0; b < V; ++b)
              v[q * V + b] = keep16<SHORT, T>(v[q * V + b], a.K - (k0 + (q * kWaves + wave) * Span + c * V), a.K);
        }
#pragma unroll
        for (int q = 0; q < Parts; ++q)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (!whole && k0 + (q * kWaves + wave) * Span >= a.K) continue;
            const float4 x = xs[(q * kWaves + wave) * Span + c * V + i];
#pragma unroll
            for (int b = 0; b < V; ++b) add_products(acc[b], x, element<T>(v[q * V + b], i));
          }
      };
      over_chunks(a.K, chunk);
#pragma unroll
      for (int b = 0; b < V; ++b)
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float s = lanes_sum<8>(acc[b][r]);
          if (c == 0) part[wave][r][8 * b + (lane >> 3)] = s;
        }
    } else {
      // 8 lanes share a reduction row; 64 rows at a time.
      static_assert(Loads * kThreads / 8 == kChunk, "");
      const int kr = tid >> 3, n = n0 + c * V;
      float acc[V][kRows] = {};
      auto chunk = [&](int k0, auto whole) {
#pragma unroll
        for (int u = 0; u < Loads; ++u) {
          if (!whole && k0 + u * (kThreads / 8) >= a.K) continue;
          const int k = k0 + kr + u * (kThreads / 8);
          v[u] = fetch16<SHORT>(w + (whole ? k : min(k, a.K - 1)) * a.wk + n, a.Nn - n);
        }
        __syncthreads();
        stage<T>(a, first, rows, k0, xs);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < Loads; ++u) {
          if (!whole && k0 + u * (kThreads / 8) >= a.K) continue;
          const float4 x = xs[kr + u * (kThreads / 8)];
          v[u] = keep16<SHORT, T>(v[u], whole || k0 + kr + u * (kThreads / 8) < a.K ? a.Nn - n : 0, a.Nn);
#pragma unroll
          for (int i = 0; i < V; ++i) add_products(acc[i], x, element<T>(v[u], i));
        }
      };
      over_chunks(a.K, chunk);
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // the wave's 8 reduction rows: lanes 8, 16 and 32 apart
          const auto plus = [](float p, float q) { return p + q; };
          float s = acc[i][r] + __shfl_xor(acc[i][r], 8);
          s = with_other<32>(with_other<16>(s, plus), plus);
          if (lane < 8) part[wave][r][lane * V + i] = s;
        }
    }
  }
  __syncthreads();
  for (int i = tid; i < rows * Cols; i += kThreads) {
    const int r = i / Cols, n = n0 + i % Cols;
    if (n >= a.Nn) continue;
    float s = 0.f;
    if (group < a.E) {
#pragma unroll
      for (int q = 0; q < kWaves; ++q) s += part[q][r][i % Cols];
      if (a.bias) s += to_f32(static_cast<const T*>(a.bias)[(int64_t)group * a.Nn + n]);
    }
    const int64_t at = (int64_t)(first + r) * a.Nn + n;
    if (a.out_f32) static_cast<float*>(a.out)[at] = s;
    else static_cast<T*>(a.out)[at] = (T)s;
  }
}

template <typename T, bool KC>
void few_typed(const GroupedArgs& a, hipStream_t s) {
  const int cols = 8 * kVec<T>, ntiles = (a.Nn + cols - 1) / cols;
  // (groups with rows, and the rows past the last group: no more than there are positions)
  const int64_t tiles = a.M / kRows + (a.M < a.E + 1 ? a.M : a.E + 1);
  const dim3 grid = grid_of(tiles * ntiles, kThreads);
  if ((KC ? a.K : a.Nn) < kVec<T>) grouped_few_kernel<T, KC, true><<<grid, kThreads, 0, s>>>(a, ntiles);
  else grouped_few_kernel<T, KC, false><<<grid, kThreads, 0, s>>>(a, ntiles);
}

template <typename T>
void few(const GroupedArgs& a, hipStream_t s) {
  a.wk == 1 && a.wn != 1 ? few_typed<T, true>(a, s) : few_typed<T, false>(a, s);
}

}  // namespace

// Up to which number of positions this is taken, and what calls in a row took by it and by the tiles.  Whole 16-bit
// chunks: 8 (1024 x 2048 matrices, 16 experts: 14.0 and 14.5 us at 8 positions, 24 and 19.5 us at 16).  Other 16-bit
// shapes: two an expert (100 x 77, 64 experts, 32 positions: 7.4 and 8.2 us with the columns adjacent, 9.0 and 7.4 us
// with the reduction).  fp32: one an expert or 32 (256 x 512: 16 experts 8.0 and 14.4 us at 32 positions, 12.0 and
// 14.4 us at 64; 64 experts 12.1 and 14.5 us at 32, 17.6 and 14.9 us at 64).  The rule does not know the matrices'
// size: 100 x 77 would stay faster by this up to 256 positions (6.3 and 12.4 us), 1024 x 2048 of 64 experts would be
// faster by the tiles from 32 positions on (72 and 47 us; 113 and 77 us at 64).
bool grouped_few_better(const GroupedArgs& a) {
  if (a.elem == ELEM_F32) return a.M <= (a.E > 32 ? a.E : 32);
  return a.M <= 8 || (!grouped_direct(a) && a.M <= 2 * (int64_t)a.E);
}

void launch_grouped_few(const GroupedArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) few<float>(a, s);
  else if (a.elem == ELEM_BF16) few<bf16_t>(a, s);
  else few<_Float16>(a, s);
}

}  // namespace gx::layer
