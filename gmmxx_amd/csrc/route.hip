// Rows sent to their best experts, and the rows grouped by expert.
//
// A row's candidates are its scores that are neither -inf nor NaN.  The k best are
// chosen (ties: the lower index), the gates are w = exp(s - max) over the sum of the
// chosen ones' w, or of all candidates' w; of +inf scores each weighs 1 and every
// finite one 0.  A choice that finds no candidate left is expert -1 with gate 0 and
// is placed after all groups.
//
// Grouping is stable (by expert, then by row), so it is a function of the scores
// alone.  Three launches:
//   top:   choices, gates and, for each block of rows, the count of every expert;
//   scan:  the counts become exclusive prefixes over the blocks, and their totals;
//   place: every block adds the experts' offsets to its prefixes and ranks its own
//          choices in order: waves take contiguous parts, 64 choices at a time,
//          equal experts found by ballots over the index bits.
// Integer counts do not depend on the order of the additions.

#include <math.h>

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;
constexpr int kPassRows = 64;          // rows whose choices are staged in LDS at a time
constexpr int kMaxBlocks = 4096;

// Rows of a block: 64, more when that gave more than kMaxBlocks blocks.
int64_t block_rows(int64_t N) {
  int64_t r = kPassRows;
  while ((N + r - 1) / r > kMaxBlocks) r *= 2;
  return r;
}

// The weight of score v beside the row's largest m.
__device__ __forceinline__ float weight_of(float v, float m) {
  return v == m ? 1.f : (v == -INFINITY ? 0.f : expf(v - m));
}

template <typename T, int G, int V>
__global__ __launch_bounds__(kThreads) void route_top_kernel(RouteArgs a, int64_t rpb) {
  __shared__ int count[kRouteMaxE + 1];
  __shared__ int sel[kPassRows * kRouteMaxK];
  __shared__ float wsel[kPassRows * kRouteMaxK];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  constexpr int R = kThreads / G;
  for (int e = threadIdx.x; e <= a.E; e += kThreads) count[e] = 0;
  const int64_t first = blockIdx.x * rpb, last = first + rpb < a.N ? first + rpb : a.N;
  for (int64_t base = first; base < last; base += kPassRows) {
    const int rows = (int)(last - base < kPassRows ? last - base : kPassRows);
    __syncthreads();
    for (int r = sub; r < rows; r += R) {
      const T* row = static_cast<const T*>(a.scores) + (base + r) * a.lds;
      float v[V];
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = lane * V + i;
        const float s = c < a.E ? to_f32(row[c]) : -INFINITY;
        v[i] = s == s ? s : -INFINITY;
        m = fmaxf(m, v[i]);
      }
#pragma unroll
      for (int off = G / 2; off >= 1; off /= 2) m = fmaxf(m, __shfl_xor(m, off));
      float sum = 0.f;
      if (!a.renormalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += weight_of(v[i], m);
        sum = lanes_sum<G>(sum);
      }
      float chosen = 0.f;
      for (int j = 0; j < a.k; ++j) {
        float best = v[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < V; ++i)
          if (v[i] > best) {
            best = v[i];
            at = i;
          }
        int idx = lane * V + at;
#pragma unroll
        for (int off = G / 2; off >= 1; off /= 2) {
          const float b2 = __shfl_xor(best, off);
          const int i2 = __shfl_xor(idx, off);
          if (b2 > best || (b2 == best && i2 < idx)) {
            best = b2;
            idx = i2;
          }
        }
        const bool none = best == -INFINITY;
        const float w = none ? 0.f : weight_of(best, m);
        chosen += w;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (idx == lane * V + i) v[i] = -INFINITY;
        if (lane == 0) {
          sel[r * a.k + j] = none ? -1 : idx;
          wsel[r * a.k + j] = w;
        }
      }
      if (a.renormalize) sum = chosen;
      const float inv = m == -INFINITY ? 0.f : 1.f / sum;
      // (the lanes of a group are one wave's: lane 0's LDS writes above come first)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int j = lane; j < a.k; j += G) wsel[r * a.k + j] *= inv;
      if (lane == 0 && a.norm) a.norm[base + r] = make_float2(m, inv);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * a.k; i += kThreads) {
      const int e = sel[i];
      a.experts[base * a.k + i] = e;
      a.gates[base * a.k + i] = wsel[i];
      atomicAdd(&count[e < 0 ? a.E : e], 1);
    }
  }
  __syncthreads();
  int32_t* hist = a.hist + (int64_t)blockIdx.x * (a.E + 1);
  for (int e = threadIdx.x; e <= a.E; e += kThreads) hist[e] = count[e];
}

// Exclusive prefixes over the blocks for 16 experts a workgroup: 64 row lanes take
// contiguous parts, add them up, and write the prefixes in a second sweep.
constexpr int kScanCols = 16, kScanParts = 64;
__global__ __launch_bounds__(kScanCols* kScanParts) void route_scan_kernel(RouteArgs a, int blocks) {
  __shared__ int part[kScanParts][kScanCols + 1];
  const int cl = threadIdx.x % kScanCols, p = threadIdx.x / kScanCols;
  const int e = blockIdx.x * kScanCols + cl;
  const int per = (blocks + kScanParts - 1) / kScanParts;
  const int b0 = p * per < blocks ? p * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
  int s = 0;
  if (e <= a.E) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) s += a.hist[(int64_t)b * (a.E + 1) + e];
  }
  part[p][cl] = s;
  __syncthreads();
  int before = 0;
  for (int q = 0; q < p; ++q) before += part[q][cl];
  if (e <= a.E) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
      int32_t* h = a.hist + (int64_t)b * (a.E + 1) + e;
      const int n = *h;
      *h = before;
      before += n;
    }
    if (p == kScanParts - 1) a.totals[e] = before;
  }
}

template <int MAXE>
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a, int64_t rpb) {
  constexpr int W = kThreads / 64;
  __shared__ int next[W][MAXE + 1];      // counts of a wave's part, then the next position of each expert
  __shared__ int wave_sum[W];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int groups = a.E + 1;            // the last: choices without an expert
  const int64_t first = blockIdx.x * rpb * a.k;
  const int64_t all = a.N * a.k, last = first + rpb * a.k < all ? first + rpb * a.k : all;
  const int64_t per = (last - first + W * 64 - 1) / (W * 64) * 64;
  const int64_t lo = first + w * per < last ? first + w * per : last, hi = lo + per < last ? lo + per : last;
  for (int e = threadIdx.x; e < W * groups; e += kThreads) next[e / groups][e % groups] = 0;
  __syncthreads();
  for (int64_t i = lo + lane; i < hi; i += 64) {
    const int e = a.experts[i];
    atomicAdd(&next[w][e < 0 ? a.E : e], 1);
  }
  // The experts' offsets: an exclusive scan of the totals, each thread a contiguous part.
  const int chunk = (groups + kThreads - 1) / kThreads;
  const int e0 = threadIdx.x * chunk < groups ? threadIdx.x * chunk : groups;
  const int e1 = e0 + chunk < groups ? e0 + chunk : groups;
  int s = 0;
  for (int e = e0; e < e1; ++e) s += a.totals[e];
  int incl = s;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 63) wave_sum[w] = incl;
  __syncthreads();
  int off0 = incl - s;
  for (int q = 0; q < w; ++q) off0 += wave_sum[q];
  const int32_t* before = a.hist + (int64_t)blockIdx.x * groups;
  for (int e = e0; e < e1; ++e) {
    if (blockIdx.x == 0) a.offsets[e] = off0;
    int at = off0 + before[e];
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const int n = next[q][e];
      next[q][e] = at;
      at += n;
    }
    off0 += a.totals[e];
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < groups) ++bits;
  for (int64_t i0 = lo; i0 < hi; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool in = i < hi;
    int e = in ? a.experts[i] : 0;
    e = e < 0 ? a.E : e;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int pos = next[w][e] + rank;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && rank == 0) next[w][e] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      a.slots[i] = pos;
      a.rows[pos] = (int32_t)(i / a.k);
    }
  }
}

// Gradient of the scores: renormalised gates  ds_e = g_e (dg_e - Σ g dg) for the chosen, 0 elsewhere;
// otherwise  ds_e = [e chosen] g_e dg_e - p_e Σ g dg,  p_e = w_e / Σ w.
template <typename T>
__global__ __launch_bounds__(kThreads) void route_bwd_kernel(RouteArgs a, int tile) {
  extern __shared__ float lds[];
  constexpr int V = kVec<T>;
  int* sel = reinterpret_cast<int*>(lds);             // [tile][k]
  float* coef = lds + tile * a.k;                     // [tile][k]
  float* mean = coef + tile * a.k;                    // [tile]
  const int64_t base = (int64_t)blockIdx.x * tile;
  const int rows = (int)(a.N - base < tile ? a.N - base : tile);
  for (int i = threadIdx.x; i < rows * a.k; i += kThreads) {
    sel[i] = a.experts[base * a.k + i];
    coef[i] = sel[i] >= 0 ? a.gates[base * a.k + i] * a.dgates[base * a.k + i] : 0.f;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += kThreads) {
    float s = 0.f;
    for (int j = 0; j < a.k; ++j) s += coef[r * a.k + j];
    mean[r] = s;
  }
  __syncthreads();
  if (a.renormalize) {
    for (int i = threadIdx.x; i < rows * a.k; i += kThreads)
      if (sel[i] >= 0) coef[i] = a.gates[base * a.k + i] * (a.dgates[base * a.k + i] - mean[i / a.k]);
    __syncthreads();
  }
  const int nvec = (a.E + V - 1) / V;
  for (int i = threadIdx.x; i < rows * nvec; i += kThreads) {
    const int r = i / nvec, c = (i - r * nvec) * V;
    float o[V];
    if (a.renormalize) {
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = 0.f;
    } else {
      load_row(static_cast<const T*>(a.scores) + (base + r) * a.lds + c, a.E - c, o);
      const float2 nm = a.norm[base + r];
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = -mean[r] * (o[q] == o[q] && nm.y != 0.f ? weight_of(o[q], nm.x) * nm.y : 0.f);
    }
    for (int j = 0; j < a.k; ++j) {
      const int e = sel[r * a.k + j];
      const float v = coef[r * a.k + j];
#pragma unroll
      for (int q = 0; q < V; ++q)
        if (e == c + q) o[q] += v;
    }
    store_row(static_cast<T*>(a.dscores) + (base + r) * a.E + c, a.E - c, o);
  }
}

template <typename T>
void top_typed(const RouteArgs& a, int64_t rpb, unsigned grid, hipStream_t s) {
  if (a.E <= 8) route_top_kernel<T, 8, 1><<<grid, kThreads, 0, s>>>(a, rpb);
  else if (a.E <= 64) route_top_kernel<T, 16, 4><<<grid, kThreads, 0, s>>>(a, rpb);
  else if (a.E <= 256) route_top_kernel<T, 64, 4><<<grid, kThreads, 0, s>>>(a, rpb);
  else if (a.E <= 1024) route_top_kernel<T, 64, 16><<<grid, kThreads, 0, s>>>(a, rpb);
  else route_top_kernel<T, 64, 64><<<grid, kThreads, 0, s>>>(a, rpb);
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

int64_t route_workspace_bytes(int64_t N, int E) {
  const int64_t rpb = block_rows(N), blocks = (N + rpb - 1) / rpb;
  return (int64_t)(align256((size_t)blocks * (E + 1) * 4) + align256((size_t)(E + 1) * 4));
}

int64_t route_totals_offset(int64_t N, int E) {
  return route_workspace_bytes(N, E) - (int64_t)align256((size_t)(E + 1) * 4);
}

void launch_route(const RouteArgs& a, hipStream_t s) {
  const int64_t rpb = block_rows(a.N);
  const unsigned blocks = (unsigned)((a.N + rpb - 1) / rpb);
  if (a.elem == ELEM_F32) top_typed<float>(a, rpb, blocks, s);
  else if (a.elem == ELEM_BF16) top_typed<__bf16>(a, rpb, blocks, s);
  else top_typed<_Float16>(a, rpb, blocks, s);
  route_scan_kernel<<<(a.E + 1 + kScanCols - 1) / kScanCols, kScanCols * kScanParts, 0, s>>>(a, (int)blocks);
  if (a.E <= 512) route_place_kernel<512><<<blocks, kThreads, 0, s>>>(a, rpb);
  else route_place_kernel<kRouteMaxE><<<blocks, kThreads, 0, s>>>(a, rpb);
}

void launch_route_bwd(const RouteArgs& a, hipStream_t s) {
  const int tile = 32;
  const unsigned grid = (unsigned)((a.N + tile - 1) / tile);
  const size_t lds = (size_t)(2 * tile * a.k + tile) * 4;
  if (a.elem == ELEM_F32) route_bwd_kernel<float><<<grid, kThreads, lds, s>>>(a, tile);
  else if (a.elem == ELEM_BF16) route_bwd_kernel<__bf16><<<grid, kThreads, lds, s>>>(a, tile);
  else route_bwd_kernel<_Float16><<<grid, kThreads, lds, s>>>(a, tile);
}

}  // namespace gx::layer
