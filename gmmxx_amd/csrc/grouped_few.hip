// Grouped products of few rows (serving): out[p] = x[rows[p]] W[e] + b[e] where groups have a handful of rows.
//
// Each weight is used once or a few times, so the pass is a stream of the chosen experts' weights: a workgroup
// of eight waves takes up to four rows of one group and 8 vectors of columns, and reads its weights once from
// memory, 16 bytes a lane, straight to registers; the products are fp32 multiply-adds.  Larger groups take
// several workgroups, which find the weights in cache.  The reduction is cut over the lanes and waves of the
// workgroup and joined in a fixed order.  Any width, stride and type.

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kRows = 4;         // of a workgroup
constexpr int kChunk = 1024;     // reduction elements of x staged at a time

// x's rows as xs[k][row], zeros past K.
template <typename T>
__device__ __forceinline__ void stage(const GroupedArgs& a, int first, int rows, int k0, float4* xs) {
  const int r = threadIdx.x & 3, lane = threadIdx.x >> 2;
  const T* x = static_cast<const T*>(a.x) + source_row(a, first + (r < rows ? r : 0)) * a.ldx;
  const int most = min(kChunk, a.K - k0);
  for (int k = lane; k < kChunk; k += kThreads / 4)
    reinterpret_cast<float*>(xs)[k * 4 + r] = r < rows && k < most ? to_f32(x[k0 + k]) : 0.f;
}

template <typename T, bool KC>
__global__ __launch_bounds__(kThreads) void grouped_few_kernel(GroupedArgs a, int ntiles) {
  constexpr int V = kVec<T>;
  constexpr int Cols = KC ? 64 : 8 * V;        // columns of a workgroup
  __shared__ __align__(16) float4 xs[kChunk];
  __shared__ float part[kWaves][kRows][Cols];
  int group, first, end, ntile;
  if (!find_tile<kRows>(a, blockIdx.x, ntiles, group, first, end, ntile)) return;
  const int rows = min(end - first, kRows), n0 = ntile * Cols;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (group < a.E) {
    const T* w = static_cast<const T*>(a.w) + (int64_t)group * a.we;
    if constexpr (KC) {
      // 8 lanes share a column; a wave takes every 8th stretch of 8 V reduction elements.
      constexpr int Span = 8 * V, Parts = kChunk / (Span * kWaves);
      const int c = lane & 7;
      for (int i = tid; i < kWaves * kRows * Cols; i += kThreads) (&part[0][0][0])[i] = 0.f;
      for (int k0 = 0; k0 < a.K; k0 += kChunk) {
        __syncthreads();
        stage<T>(a, first, rows, k0, xs);
        __syncthreads();
        for (int b = 0; b < Cols; b += 8) {
          const int n = n0 + b + (lane >> 3);
          float acc[kRows] = {};
#pragma unroll
          for (int q = 0; q < Parts; ++q) {
            const int k = (q * kWaves + wave) * Span + c * V;
            float v[V];
            load_row(w + (int64_t)n * a.wn + k0 + k, n < a.Nn ? a.K - k0 - k : 0, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float4 xv = xs[k + i];
              acc[0] = fmaf(xv.x, v[i], acc[0]);
              acc[1] = fmaf(xv.y, v[i], acc[1]);
              acc[2] = fmaf(xv.z, v[i], acc[2]);
              acc[3] = fmaf(xv.w, v[i], acc[3]);
            }
          }
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            acc[r] = lanes_sum<8>(acc[r]);
            if (c == 0) part[wave][r][b + (lane >> 3)] += acc[r];
          }
        }
      }
    } else {
      // 8 lanes share a reduction row; 64 rows at a time.
      const int c = lane & 7, kr = tid >> 3, n = n0 + c * V;
      float acc[kRows][V] = {};
      for (int k0 = 0; k0 < a.K; k0 += kChunk) {
        __syncthreads();
        stage<T>(a, first, rows, k0, xs);
        __syncthreads();
        const int most = min(kChunk, a.K - k0);
#pragma unroll 8
        for (int k = kr; k < most; k += kThreads / 8) {
          float v[V];
          load_row(w + (int64_t)(k0 + k) * a.wk + n, a.Nn - n, v);
          const float4 xv = xs[k];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            acc[0][i] = fmaf(xv.x, v[i], acc[0][i]);
            acc[1][i] = fmaf(xv.y, v[i], acc[1][i]);
            acc[2][i] = fmaf(xv.z, v[i], acc[2][i]);
            acc[3][i] = fmaf(xv.w, v[i], acc[3][i]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float s = acc[r][i];
          s += __shfl_xor(s, 8);
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
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
  const int cols = KC ? 64 : 8 * kVec<T>, ntiles = (a.Nn + cols - 1) / cols;
  // (groups with rows, and the rows past the last group: no more than there are positions)
  const int64_t tiles = a.M / kRows + (a.M < a.E + 1 ? a.M : a.E + 1);
  grouped_few_kernel<T, KC><<<(unsigned)(tiles * ntiles), kThreads, 0, s>>>(a, ntiles);
}

template <typename T>
void few(const GroupedArgs& a, hipStream_t s) {
  a.wk == 1 && a.wn != 1 ? few_typed<T, true>(a, s) : few_typed<T, false>(a, s);
}

}  // namespace

// Up to which number of positions this beats the tiles: of 1024 x 2048 matrices, 8 positions of 16 experts
// 11.9 and 12.6 us, 16 positions 30.6 and 15.5 us by tiles of whole chunks; the element-wise tiles are slower
// by far (fp32, 64 experts, 128 positions: 230 and 292 us).
bool grouped_few_better(const GroupedArgs& a) {
  return a.M <= 8 || (!grouped_mma_rows_ok(a) && a.M <= 2 * (int64_t)a.E);
}

void launch_grouped_few(const GroupedArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) few<float>(a, s);
  else if (a.elem == ELEM_BF16) few<bf16_t>(a, s);
  else few<_Float16>(a, s);
}

}  // namespace gx::layer
