// The experts' results added up for each row, and the gradient of that sum.
//
//   out[n] = Σ_j gate[n,j] · y[slot[n,j]]
//   dy[slot[n,j]] = gate[n,j] · dout[n],   dgate[n,j] = <dout[n], y[slot[n,j]]>
//
// slot is a permutation of the M positions, so every row of dy is written once and
// no atomics are needed.  Positions from offsets[E] on are choices that no expert
// took: they add nothing, and their dy and dgate are zero.  Sums are fp32, with one
// rounding at the store.  Both directions move bytes only: 16-byte vectors, four
// rows of y in flight per thread.  16384 rows of 4 choices, 2048 columns of bf16:
// forward 82 us (335 MB, 4.1 TB/s), backward 111 us (604 MB, 5.4 TB/s).  Eight rows of
// two choices are a launch: 3.0 us.

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 20;    // beyond it blocks take several rows

unsigned grid_of(int64_t N, int rows_per_block) {
  const int64_t need = (N + rows_per_block - 1) / rows_per_block;
  return (unsigned)(need < kMaxBlocks ? need : kMaxBlocks);
}

// Position of a choice that an expert took, -1 otherwise.
__device__ __forceinline__ int taken(int slot, int total) { return (unsigned)slot < (unsigned)total ? slot : -1; }

__device__ __forceinline__ int taken_total(const CombineArgs& a) {
  const int t = a.offsets[a.E];
  return t < 0 ? 0 : (t < a.M ? t : (int)a.M);
}

// tx threads (a power of two) share a row's vectors.
template <typename Y, typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombineArgs a, int tx) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & (tx - 1), rpb = kThreads / tx;
  const int total = taken_total(a);
  const Y* y = static_cast<const Y*>(a.y);
  for (int64_t n = (int64_t)blockIdx.x * rpb + threadIdx.x / tx; n < a.N; n += (int64_t)gridDim.x * rpb) {
    T* out = static_cast<T*>(a.out) + n * a.F;
    for (int c = lane * V; c < a.F; c += tx * V) {
      float acc[V];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.f;
      for (int j0 = 0; j0 < a.k; j0 += 4) {
        constexpr int H = (int)(sizeof(Y) / sizeof(T));      // vectors of y for one of out
        uint4 u[4][H];
        float g[4];
        bool there[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int slot = j0 + j < a.k ? taken(a.slots[n * a.k + j0 + j], total) : -1;
          there[j] = slot >= 0;
          g[j] = there[j] && a.gates ? a.gates[n * a.k + j0 + j] : 1.f;
          const Y* p = y + (int64_t)(there[j] ? slot : 0) * a.ldy + c;
          if (j0 + j < a.k) {
#pragma unroll
            for (int h = 0; h < H; ++h) u[j][h] = fetch16<SHORT>(p + h * kVec<Y>, a.F - c - h * kVec<Y>);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j0 + j >= a.k) break;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            float v[kVec<Y>];
            unpack16<Y>(keep16<SHORT, Y>(u[j][h], there[j] ? a.F - c - h * kVec<Y> : 0, a.F), v);
#pragma unroll
            for (int i = 0; i < kVec<Y>; ++i)
              acc[h * kVec<Y> + i] = fmaf(g[j], there[j] ? v[i] : 0.f, acc[h * kVec<Y> + i]);
          }
        }
      }
      store_row(out + c, a.F - c, acc);
    }
  }
}

// G lanes of a wave share a row; KC choices at a time (dout is read again for every KC).
template <typename T, int G, int KC, bool SHORT>
__global__ __launch_bounds__(kThreads) void combine_bwd_kernel(CombineArgs a) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x % G;
  constexpr int R = kThreads / G;
  const int total = taken_total(a);
  const T* y = static_cast<const T*>(a.y);
  T* dy = static_cast<T*>(a.out);
  for (int64_t n = (int64_t)blockIdx.x * R + threadIdx.x / G; n < a.N; n += (int64_t)gridDim.x * R) {
    const T* dout = static_cast<const T*>(a.dout) + n * a.lddout;
    for (int j0 = 0; j0 < a.k; j0 += KC) {
      int pos[KC], slot[KC];
      float g[KC], dot[KC];
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const bool in = j0 + j < a.k;
        pos[j] = in ? a.slots[n * a.k + j0 + j] : -1;
        pos[j] = (unsigned)pos[j] < (unsigned)a.M ? pos[j] : -1;
        slot[j] = taken(pos[j], total);
        g[j] = slot[j] >= 0 ? a.gates[n * a.k + j0 + j] : 0.f;
        dot[j] = 0.f;
      }
      for (int c = lane * V; c < a.F; c += G * V) {
        uint4 ud = fetch16<SHORT>(dout + c, a.F - c), u[KC];
#pragma unroll
        for (int j = 0; j < KC; ++j) u[j] = fetch16<SHORT>(y + (int64_t)(slot[j] >= 0 ? slot[j] : 0) * a.ldy + c, a.F - c);
        float d[V];
        unpack16<T>(keep16<SHORT, T>(ud, a.F - c, a.F), d);
#pragma unroll
        for (int j = 0; j < KC; ++j) {
          float o[V], v[V];
          unpack16<T>(keep16<SHORT, T>(u[j], a.F - c, a.F), v);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dot[j] = fmaf(d[i], v[i], dot[j]);
            o[i] = slot[j] >= 0 ? g[j] * d[i] : 0.f;
          }
          store_row(dy + (int64_t)(pos[j] >= 0 ? pos[j] : 0) * a.F + c, pos[j] >= 0 ? a.F - c : 0, o);
        }
      }
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        const float s = lanes_sum<G>(dot[j]);
        if (lane == 0 && j0 + j < a.k) a.dgates[n * a.k + j0 + j] = slot[j] >= 0 ? s : 0.f;
      }
    }
  }
}

template <typename Y, typename T>
void combine_typed(const CombineArgs& a, hipStream_t s) {
  const int nvec = (a.F + kVec<T> - 1) / kVec<T>;
  int tx = 1;
  while (tx < nvec && tx < kThreads) tx *= 2;
  // (vectors of fp32 y are the shorter)
  if (a.F < kVec<T>) combine_kernel<Y, T, true><<<grid_of(a.N, kThreads / tx), kThreads, 0, s>>>(a, tx);
  else combine_kernel<Y, T, false><<<grid_of(a.N, kThreads / tx), kThreads, 0, s>>>(a, tx);
}

template <typename T, int G, bool SHORT>
void combine_bwd_group(const CombineArgs& a, hipStream_t s) {
  const unsigned grid = grid_of(a.N, kThreads / G);
  if (a.k <= 1) combine_bwd_kernel<T, G, 1, SHORT><<<grid, kThreads, 0, s>>>(a);
  else if (a.k <= 2) combine_bwd_kernel<T, G, 2, SHORT><<<grid, kThreads, 0, s>>>(a);
  else combine_bwd_kernel<T, G, 4, SHORT><<<grid, kThreads, 0, s>>>(a);
}

template <typename T>
void combine_bwd_typed(const CombineArgs& a, hipStream_t s) {
  const int nvec = (a.F + kVec<T> - 1) / kVec<T>;
  if (a.F < kVec<T>) combine_bwd_group<T, 8, true>(a, s);
  else if (nvec <= 8) combine_bwd_group<T, 8, false>(a, s);
  else if (nvec <= 32) combine_bwd_group<T, 32, false>(a, s);
  else combine_bwd_group<T, 64, false>(a, s);
}

}  // namespace

void launch_combine(const CombineArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) combine_typed<float, float>(a, s);
  else if (a.elem == ELEM_BF16 && a.y_f32) combine_typed<float, __bf16>(a, s);
  else if (a.elem == ELEM_BF16) combine_typed<__bf16, __bf16>(a, s);
  else if (a.y_f32) combine_typed<float, _Float16>(a, s);
  else combine_typed<_Float16, _Float16>(a, s);
}

void launch_combine_bwd(const CombineArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) combine_bwd_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) combine_bwd_typed<__bf16>(a, s);
  else combine_bwd_typed<_Float16>(a, s);
}

}  // namespace gx::layer
