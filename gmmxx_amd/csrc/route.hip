// Rows sent to their best experts, and the rows grouped by expert.
//
// A row's candidates are its scores that are neither -inf nor NaN.  The k best are
// chosen (ties: the lower index), the gates are w = exp(s - max) over the sum of the
// chosen ones' w, or of all candidates' w; of +inf scores each weighs 1 and every
// finite one 0.  A choice that finds no candidate left is expert -1 with gate 0 and
// is placed after all groups.
//
// Grouping is stable (by expert, then by row), so it is a function of the scores
// alone.  Three launches (one for up to 64 rows and 512 experts):
//   top:   choices, gates and, for each block of rows, the count of every expert;
//   scan:  the counts become exclusive prefixes over the blocks, and their totals;
//   place: every block adds the experts' offsets to its prefixes and ranks its own
//          choices in order: waves take contiguous parts, 64 choices at a time,
//          equal experts found by ballots over the index bits.
// Integer counts do not depend on the order of the additions.
//
// The choice takes mostly instructions (see choose_rows), the gradient of gates over all
// candidates bytes, the rest waits.  100000 x 500 fp32, 4 of all: top 76 us (the scores at 2.6 TB/s), scan
// 13 us, place 10 us, gradient 79 us (5.1 TB/s).  65537 x 64, 8 of 64: 13, 7, 7 and
// 10 us.  Three rows of 64 in one launch: 4.4 us.

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

// exp(x) for x <= 0, 0 for NaN: by the hardware's power of two, with the rounding of x log2(e) put back in first
// order.
__device__ __forceinline__ float exp_below(float x) {
  x = fmaxf(x, -110.f);                   // (exp(-110) is 0; finite, so is what follows)
  const float y = x * kLog2e;
  const float lost = fmaf(x, 1.925963033500e-8f, fmaf(x, kLog2e, -y));      // (log2(e) = kLog2e + 1.926e-8)
  return fast_exp2(y) * fmaf(lost, kLn2, 1.f);
}

// The weight of score v beside the row's largest m (v <= m): 1 for each of several +inf.
__device__ __forceinline__ float weight_of(float v, float m) { return v == m ? 1.f : exp_below(v - m); }

// Integers in the order of the scores; -0 as 0.  kNone, the key of -inf, and below: no candidate.
__device__ __forceinline__ int key_of(float v) {
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float score_of(int key) { return __int_as_float(key ^ ((key >> 31) & 0x7fffffff)); }
constexpr int kNone = (int)0x807fffffu;

// op over a group's lanes for integers (see lanes_reduce).
template <int G, typename F>
__device__ __forceinline__ int lanes_reduce_int(int v, F&& op) {
  return __float_as_int(lanes_reduce<G>(__int_as_float(v), [&](float a, float b) {
    return __int_as_float(op(__float_as_int(a), __float_as_int(b)));
  }));
}

// The choices of up to kPassRows rows, to LDS.  G lanes share a row, NV vectors of its scores each: vector i of
// lane l holds the scores from (i G + l) kVec on, as integers in their order.  Each round takes the group's
// largest remaining score, then the lowest index that has it.  With few rows to a wave (G from 16 on) a round
// passes over the vectors in which no row of the wave has its score: 134217 x 500, 4 each 93 us by it and 98 us
// without, 16777 x 4000, 8 each 201 and 252 us, but 200000 x 64, 8 each 59 and 57 us.  About 5 instructions a
// held score and round where nothing is passed over, and 14 for its exponential where all candidates count:
// 100000 x 500, 4 of all take 30 million of a wave, 48 us of what the card issues.  So G is the smallest that
// holds the row in 32 scores a lane (64 at the most experts): what lanes exchange is the smaller part.
template <typename T, int G, int NV, bool SHORT>
__device__ __forceinline__ void choose_rows(const RouteArgs& a, int64_t base, int rows, int* sel, float* wsel) {
  constexpr int VV = kVec<T>, R = kThreads / G;
  constexpr bool kSkip = G >= 16;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const auto larger = [](int p, int q) { return p > q ? p : q; };
  const auto smaller = [](int p, int q) { return p < q ? p : q; };
  for (int r0 = 0; r0 < rows; r0 += R) {        // (all lanes stay in the loop: groups exchange across the wave)
    const int r = r0 + sub;
    const bool there = r < rows;
    const T* row = static_cast<const T*>(a.scores) + (base + (there ? r : 0)) * a.lds;
    int v[NV][VV];
    uint4 u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = fetch16<SHORT>(row + (i * G + lane) * VV, a.E - (i * G + lane) * VV);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * VV;
      float s[VV];
      unpack16<T>(keep16<SHORT, T>(u[i], a.E - c, a.E), s);
#pragma unroll
      for (int j = 0; j < VV; ++j) v[i][j] = s[j] == s[j] && c + j < a.E ? key_of(s[j]) : INT32_MIN;
    }
    int top[NV], best = INT32_MIN;              // of each vector, and of the row
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      top[i] = INT32_MIN;
#pragma unroll
      for (int q = 0; q < VV; ++q) top[i] = larger(top[i], v[i][q]);
      best = larger(best, top[i]);
    }
    best = lanes_reduce_int<G>(best, larger);
    const float m = best > kNone ? score_of(best) : -INFINITY;
    float sum = 0.f;
    if (!a.renormalize) {
      if (fabsf(m) < INFINITY) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int q = 0; q < VV; ++q) sum += exp_below(score_of(v[i][q]) - m);      // (no candidate: -inf or NaN)
      } else {      // of +inf each weighs 1
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int q = 0; q < VV; ++q) sum += v[i][q] == best ? 1.f : 0.f;
      }
      sum = lanes_sum<G>(sum);
    }
    float chosen = 0.f;
    int mine = 0;                               // the last choice, as this lane's score 0 would be 0
    for (int j = 0; j < a.k; ++j) {
      if (j > 0) {
        best = INT32_MIN;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!kSkip || __any((unsigned)(mine - i * G * VV) < (unsigned)VV)) {
            top[i] = INT32_MIN;
#pragma unroll
            for (int q = 0; q < VV; ++q) {
              v[i][q] = mine == i * G * VV + q ? INT32_MIN : v[i][q];
              top[i] = larger(top[i], v[i][q]);
            }
          }
          best = larger(best, top[i]);
        }
        best = lanes_reduce_int<G>(best, larger);
      }
      int at = INT32_MAX;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (!kSkip || __any(top[i] == best)) {
#pragma unroll
          for (int q = VV - 1; q >= 0; --q) at = v[i][q] == best ? i * G * VV + q : at;
        }
      at = lanes_reduce_int<G>(at == INT32_MAX ? at : at + lane * VV, smaller);
      const bool none = best <= kNone;
      const float w = none ? 0.f : weight_of(score_of(best), m);
      chosen += w;
      mine = at - lane * VV;
      if (lane == 0 && there) {
        sel[r * a.k + j] = none ? -1 : at;
        wsel[r * a.k + j] = w;
      }
    }
    if (a.renormalize) sum = chosen;
    const float inv = m == -INFINITY ? 0.f : 1.f / sum;
    // (the lanes of a group are one wave's: lane 0's LDS writes above come first)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (there) {
      for (int j = lane; j < a.k; j += G) wsel[r * a.k + j] *= inv;
      if (lane == 0 && a.norm) a.norm[base + r] = make_float2(m, inv);
    }
  }
}

template <typename T, int G, int NV, bool SHORT>
__global__ __launch_bounds__(kThreads) void route_top_kernel(RouteArgs a, int64_t rpb) {
  extern __shared__ int lds[];           // choices, their weights, counts: top_lds()
  int* sel = lds;
  float* wsel = reinterpret_cast<float*>(lds + kPassRows * a.k);
  int* count = lds + 2 * kPassRows * a.k;
  for (int e = threadIdx.x; e <= a.E; e += kThreads) count[e] = 0;
  const int64_t first = blockIdx.x * rpb, last = first + rpb < a.N ? first + rpb : a.N;
  for (int64_t base = first; base < last; base += kPassRows) {
    const int rows = (int)(last - base < kPassRows ? last - base : kPassRows);
    __syncthreads();
    choose_rows<T, G, NV, SHORT>(a, base, rows, sel, wsel);
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

// Positions of choices first .. last - 1 (expert(i): that of choice i, a.E for none), given total(e), how many
// choices expert e has, and before(e), how many of them come before `first`.
template <int MAXE, typename X, typename N, typename B>
__device__ __forceinline__ void place(const RouteArgs& a, int64_t first, int64_t last, X&& expert, N&& total,
                                      B&& before) {
  constexpr int W = kThreads / 64;
  __shared__ int next[W][MAXE + 1];      // counts of a wave's part, then the next position of each expert
  __shared__ int wave_sum[W];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int groups = a.E + 1;            // the last: choices without an expert
  const int64_t per = (last - first + W * 64 - 1) / (W * 64) * 64;
  const int64_t lo = first + w * per < last ? first + w * per : last, hi = lo + per < last ? lo + per : last;
  for (int e = threadIdx.x; e < groups; e += kThreads)
#pragma unroll
    for (int q = 0; q < W; ++q) next[q][e] = 0;
  __syncthreads();
  for (int64_t i = lo + lane; i < hi; i += 64) atomicAdd(&next[w][expert(i)], 1);
  // The experts' offsets: an exclusive scan of the totals, each thread a contiguous part.
  const int chunk = (groups + kThreads - 1) / kThreads;
  const int e0 = threadIdx.x * chunk < groups ? threadIdx.x * chunk : groups;
  const int e1 = e0 + chunk < groups ? e0 + chunk : groups;
  int s = 0;
  for (int e = e0; e < e1; ++e) s += total(e);
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
  for (int e = e0; e < e1; ++e) {
    if (blockIdx.x == 0) a.offsets[e] = off0;
    int at = off0 + before(e);
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const int n = next[q][e];
      next[q][e] = at;
      at += n;
    }
    off0 += total(e);
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < groups) ++bits;
  for (int64_t i0 = lo; i0 < hi; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool in = i < hi;
    const int e = in ? expert(i) : 0;
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

template <int MAXE>
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a, int64_t rpb) {
  const int64_t first = blockIdx.x * rpb * a.k, all = a.N * a.k, last = first + rpb * a.k < all ? first + rpb * a.k : all;
  const int32_t* before = a.hist + (int64_t)blockIdx.x * (a.E + 1);
  place<MAXE>(
      a, first, last,
      [&](int64_t i) {
        const int e = a.experts[i];
        return e < 0 ? a.E : e;
      },
      [&](int e) { return a.totals[e]; }, [&](int e) { return before[e]; });
}

// Few rows (one pass of one block) in one launch.
constexpr int kOneMaxE = 512;
template <typename T, int G, int NV, bool SHORT>
__global__ __launch_bounds__(kThreads) void route_one_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int* sel = lds;
  float* wsel = reinterpret_cast<float*>(lds + kPassRows * a.k);
  int* count = lds + 2 * kPassRows * a.k;
  for (int e = threadIdx.x; e <= a.E; e += kThreads) count[e] = 0;
  choose_rows<T, G, NV, SHORT>(a, 0, (int)a.N, sel, wsel);
  __syncthreads();
  const int all = (int)a.N * a.k;
  for (int i = threadIdx.x; i < all; i += kThreads) {
    const int e = sel[i];
    a.experts[i] = e;
    a.gates[i] = wsel[i];
    atomicAdd(&count[e < 0 ? a.E : e], 1);
  }
  __syncthreads();
  place<kOneMaxE>(
      a, 0, all, [&](int64_t i) { return sel[i] < 0 ? a.E : sel[i]; }, [&](int e) { return count[e]; },
      [](int) { return 0; });
}

// Gradient of the scores: renormalised gates  ds_e = g_e (dg_e - Σ g dg) for the chosen, 0 elsewhere;
// otherwise  ds_e = [e chosen] g_e dg_e - p_e Σ g dg,  p_e = w_e / Σ w.
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void route_bwd_kernel(RouteArgs a, int tile) {
  extern __shared__ int lds[];
  constexpr int V = kVec<T>;
  int* sel = lds;                                                      // [tile][k]
  float* coef = reinterpret_cast<float*>(lds + tile * a.k);            // [tile][k]
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
      unpack16<T>(keep16<SHORT, T>(fetch16<SHORT>(static_cast<const T*>(a.scores) + (base + r) * a.lds + c, a.E - c), a.E - c, a.E), o);
      const float2 nm = a.norm[base + r];
#pragma unroll
      for (int q = 0; q < V; ++q) o[q] = -mean[r] * (o[q] > -INFINITY ? weight_of(o[q], nm.x) * nm.y : 0.f);      // (NaN and -inf: no candidates)
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

size_t top_lds(const RouteArgs& a) { return (size_t)(2 * kPassRows * a.k + a.E + 1) * 4; }

template <typename T, int G, int NV, bool SHORT>
void top_shaped(const RouteArgs& a, int64_t rpb, unsigned grid, hipStream_t s) {
  if constexpr (G * NV * kVec<T> <= kOneMaxE) {
    if (a.N <= kPassRows) return route_one_kernel<T, G, NV, SHORT><<<1, kThreads, top_lds(a), s>>>(a);
  }
  route_top_kernel<T, G, NV, SHORT><<<grid, kThreads, top_lds(a), s>>>(a, rpb);
}

template <typename T>
void top_typed(const RouteArgs& a, int64_t rpb, unsigned grid, hipStream_t s) {
  constexpr int N8 = 8 / kVec<T>;       // vectors of 8 scores
  if (a.E < kVec<T>) top_shaped<T, 4, N8, true>(a, rpb, grid, s);
  else if (a.E <= 32) top_shaped<T, 4, N8, false>(a, rpb, grid, s);
  else if (a.E <= 64) top_shaped<T, 4, 2 * N8, false>(a, rpb, grid, s);
  else if (a.E <= 128) top_shaped<T, 8, 2 * N8, false>(a, rpb, grid, s);
  else if (a.E <= 256) top_shaped<T, 8, 4 * N8, false>(a, rpb, grid, s);
  else if (a.E <= 512) top_shaped<T, 16, 4 * N8, false>(a, rpb, grid, s);
  else if (a.E <= 1024) top_shaped<T, 32, 4 * N8, false>(a, rpb, grid, s);
  else if (a.E <= 2048) top_shaped<T, 64, 4 * N8, false>(a, rpb, grid, s);
  else top_shaped<T, 64, 8 * N8, false>(a, rpb, grid, s);
}

template <typename T>
void bwd_typed(const RouteArgs& a, int tile, unsigned grid, size_t lds, hipStream_t s) {
  if (a.E < kVec<T>) route_bwd_kernel<T, true><<<grid, kThreads, lds, s>>>(a, tile);
  else route_bwd_kernel<T, false><<<grid, kThreads, lds, s>>>(a, tile);
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
  if (a.N <= kPassRows && a.E <= kOneMaxE) return;
  route_scan_kernel<<<(a.E + 1 + kScanCols - 1) / kScanCols, kScanCols * kScanParts, 0, s>>>(a, (int)blocks);
  if (a.E <= 512) route_place_kernel<512><<<blocks, kThreads, 0, s>>>(a, rpb);
  else route_place_kernel<kRouteMaxE><<<blocks, kThreads, 0, s>>>(a, rpb);
}

void launch_route_bwd(const RouteArgs& a, hipStream_t s) {
  int tile = 32;            // rows of a block; more where the grid's threads would pass 2^31 (k is small there)
  while ((a.N + tile - 1) / tile > (int64_t(1) << 31) / kThreads) tile *= 2;
  const unsigned grid = (unsigned)((a.N + tile - 1) / tile);
  const size_t lds = (size_t)(2 * tile * a.k + tile) * 4;
  if (a.elem == ELEM_F32) bwd_typed<float>(a, tile, grid, lds, s);
  else if (a.elem == ELEM_BF16) bwd_typed<__bf16>(a, tile, grid, lds, s);
  else bwd_typed<_Float16>(a, tile, grid, lds, s);
}

}  // namespace gx::layer
