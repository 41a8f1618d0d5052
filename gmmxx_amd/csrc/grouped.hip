// Matrix products grouped by expert, with ragged group sizes.
//
//   out[p] = x[rows[p]] W[e] + b[e]          for the positions p of group e      (rows kernel)
//   dW[e]  = Σ_p x[rows[p]]ᵀ dy[p],  db[e] = Σ_p dy[p]                           (weight-gradient kernel)
// The gradient with respect to x is the rows kernel on dy with the weight's two
// strides exchanged.
//
// The groups' offsets stay on the device: the grid is sized for the most tiles that
// any offsets can give (M / tile + E + 1), and each workgroup finds its group by
// counting tiles (grouped_core.hpp).  The tiles are in grouped_tiles.hpp, products of few rows in
// grouped_few.hip; here are the choice among them, db and the sums of parts.  Positions
// past offsets[E] get rows of zeros.  Offsets and row indices are clamped to their
// arrays, so no values of theirs lead out of bounds.
//
// Bound by the matrix units and, around each tile, by the waits before its first and
// after its last product.  One bf16 product of 8192 x 8192 x 8192: 920 us, 1.19 PFLOP/s
// (fp32 143 TFLOP/s).  32768 positions of 32 uneven groups, 1024 x 2048 bf16: forward
// 193 us, for x 193 us, for W 183 us (137 GFLOP each, 710 - 750 TFLOP/s: about 1150 tiles
// are 4.5 for each CU), db 28 us.  100003 fp32 rows of 200 groups, 100 x 77: 62, 48, 83
// and 12 us.

#include <math.h>

#include "grouped_core.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;

// db[e][n] = Σ_p dy[p][n]: 16 threads of one vector of columns by 16 row lanes a workgroup.
constexpr int kBiasLanes = 16;
template <typename T, bool SPLIT, bool SHORT>
__global__ __launch_bounds__(kThreads) void grouped_bias_kernel(GroupedArgs a) {
  constexpr int V = kVec<T>, Cols = 16 * V;
  __shared__ float part[kBiasLanes][Cols + 4];
  const int e = blockIdx.y, c = threadIdx.x & 15, n = blockIdx.x * Cols + c * V, r0 = threadIdx.x >> 4;
  int lo = offset_at(a, e), hi = offset_at(a, e + 1);
  if constexpr (SPLIT) split_part(lo, hi, blockIdx.z, gridDim.z);
  float s[V] = {};
  const T* dy = static_cast<const T*>(a.dy) + n;
  constexpr int B = 8;      // rows in flight
  for (int p = lo + r0; p < hi; p += B * kBiasLanes) {
    uint4 u[B];
#pragma unroll
    for (int b = 0; b < B; ++b) u[b] = fetch16<SHORT>(dy + min(p + b * kBiasLanes, hi - 1) * a.lddy, a.Nn - n);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      float v[V];
      unpack16<T>(keep16<SHORT, T>(u[b], a.Nn - n, a.Nn), v);
      const bool in = p + b * kBiasLanes < hi;
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += in ? v[i] : 0.f;
    }
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

// Whether tiles of 256 (one to a CU) beat tiles of 128 (two at a time): the most tiles that a CU gets, in
// 128 x 128 tiles, over the rate measured for each (1170 and 880 TFLOP/s for one product of 8192 x 8192 x
// 8192).  The groups' sizes are on the device, so they are taken to be uneven; near ties go to the larger.  Calls by
// 256 and by 128, bf16: 8192 rows of 16 uneven experts, 2048 -> 1024, 60 and 67 us (of 8 experts 54 and 60; exactly
// even groups, whose last tiles are full, 63 and 49); 16384 rows of 16, 113 and 106 us (even 70 and 84); 32768 rows
// of 32 experts, 1024 -> 2048, 190 and 201 us.  The weight's gradient there: 191 and 205 us, but 307 and 234 us where
// a few groups have most of the rows, which tiles of 128 cut into parts.
bool larger_tiles(double tiles256, double tiles128) {
  return ceil(tiles256 / 256.0) * 4.0 / 1.17 < 1.1 * ceil(tiles128 / 256.0) / 0.88;
}

int64_t tiles(int64_t n, int t) { return (n + t - 1) / t; }

// What the direct loads' 32-bit offsets reach: 64 rows of a matrix, and the whole of one that is read along
// its rows.
bool near_rows(int64_t bytes) { return bytes < (int64_t(1) << 24); }
bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Whole, aligned 16-byte chunks along every dimension that is read 16 bytes at a time.
bool rows_direct(const GroupedArgs& a) {
  const int64_t outer = a.wk == 1 && a.wn != 1 ? a.wn : a.wk, size = a.elem == ELEM_F32 ? 4 : 2, v = 16 / size;
  return a.K % v == 0 && a.Nn % v == 0 && a.ldx % v == 0 && a.we % v == 0 && outer % v == 0 &&
         near_rows(outer * size) && outer * size * (a.wk == 1 && a.wn != 1 ? a.Nn : 64) < (int64_t(1) << 32) &&
         aligned16(a.x) && aligned16(a.w) && aligned16(a.out);
}

bool dw_direct(const GroupedArgs& a) {
  const int64_t size = a.elem == ELEM_F32 ? 4 : 2, v = 16 / size;
  return a.K % v == 0 && a.Nn % v == 0 && a.ldx % v == 0 && a.lddy % v == 0 && near_rows(a.lddy * size) &&
         aligned16(a.x) && aligned16(a.dy) && aligned16(a.out);
}

bool dw_larger(int64_t E, int64_t K, int64_t N) {
  return larger_tiles((double)E * tiles(K, 256) * tiles(N, 256), (double)E * tiles(K, 128) * tiles(N, 128));
}

// The rest of the weight gradient's pass: db, and the sums of parts.
template <typename T>
void dw_rest(const GroupedArgs& a, int splits, int bias_splits, hipStream_t s) {
  if (a.dbias) {
    const dim3 grid((unsigned)((a.Nn + 16 * kVec<T> - 1) / (16 * kVec<T>)), (unsigned)a.E, (unsigned)bias_splits);
    const bool whole = a.Nn >= kVec<T>;
    if (bias_splits == 1 && whole) grouped_bias_kernel<T, false, false><<<grid, kThreads, 0, s>>>(a);
    else if (bias_splits == 1) grouped_bias_kernel<T, false, true><<<grid, kThreads, 0, s>>>(a);
    else if (whole) grouped_bias_kernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
    else grouped_bias_kernel<T, true, true><<<grid, kThreads, 0, s>>>(a);
  }
  const int64_t all = (splits > 1 ? (int64_t)a.E * a.K * a.Nn : 0) + (bias_splits > 1 ? (int64_t)a.E * a.Nn : 0);
  const int64_t blocks = (all + kThreads - 1) / kThreads;
  if (all) grouped_reduce_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), kThreads, 0, s>>>(a, splits, bias_splits);
}

// Parts that an average group's positions are cut into, given the workgroups without parts, the workgroups
// wanted and the fewest positions of a part.
int parts_of(int64_t M, int64_t E, int64_t groups, int64_t want, int64_t least) {
  const int64_t by_groups = (want + groups - 1) / groups, by_rows = M / (E * least);
  const int64_t s = by_groups < by_rows ? by_groups : by_rows;
  return (int)(s < 1 ? 1 : s < 65535 ? s : 65535);
}

// Parts of the weight gradient by tiles of 128, of which 512 run at once, and of db.  Twice as many workgroups
// even out groups of uneven sizes: 100003 fp32 rows, 200 experts, 100 x 77 in 3 parts 111 us, in 6 parts 83 us
// and 3 us more for their sums.
int dw_parts(int64_t M, int64_t E, int64_t K, int64_t N, int size) {
  return parts_of(M, E, E * tiles(K, 128) * tiles(N, 128), 1024, 256 / size);
}
int bias_parts(int64_t M, int64_t E, int64_t N) { return parts_of(M, E, E * tiles(N, 128), 2048, 128); }

template <typename T>
void rows_typed(const GroupedArgs& a, hipStream_t s) {
  // (a group's last row tile is half full on average)
  const bool larger = larger_tiles((a.M / 256.0 + 0.5 * a.E) * tiles(a.Nn, 256), (a.M / 128.0 + 0.5 * a.E) * tiles(a.Nn, 128));
  launch_rows_tiles<T>(a, rows_direct(a), larger, s);
}

template <typename T>
void dw_typed(GroupedArgs a, hipStream_t s) {
  const bool direct = dw_direct(a), larger = sizeof(T) == 2 && direct && dw_larger(a.E, a.K, a.Nn);
  const int splits = larger || !a.out ? 1 : dw_parts(a.M, a.E, a.K, a.Nn, sizeof(T)), bs = a.dbias ? bias_parts(a.M, a.E, a.Nn) : 1;
  a.bias_part = a.part + (splits > 1 ? (int64_t)splits * a.E * a.K * a.Nn : 0);
  if (a.out) launch_dw_tiles<T>(a, direct, larger, splits, s);
  dw_rest<T>(a, splits, bs, s);
}

}  // namespace

int64_t grouped_workspace_bytes(int64_t M, int64_t E, int64_t K, int64_t N) {
  const int s = dw_parts(M, E, K, N, 4), b = bias_parts(M, E, N);
  return ((s > 1 ? s * E * K * N : 0) + (b > 1 ? b * E * N : 0)) * (int64_t)sizeof(float);
}

bool grouped_direct(const GroupedArgs& a) { return rows_direct(a); }

void launch_grouped(const GroupedArgs& a, hipStream_t s) {
  if (grouped_few_better(a)) launch_grouped_few(a, s);
  else if (a.elem == ELEM_F32) rows_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) rows_typed<bf16_t>(a, s);
  else rows_typed<_Float16>(a, s);
}

void launch_grouped_dw(const GroupedArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) dw_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) dw_typed<bf16_t>(a, s);
  else dw_typed<_Float16>(a, s);
}

}  // namespace gx::layer
