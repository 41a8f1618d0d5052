// Tile lookup shared by the grouped products' kernels.
#pragma once

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

typedef __bf16 bf16_t;

// The tiles (grouped_tiles.hpp): by direct loads or not, 256 wide (16-bit elements, direct) or 128.
template <typename T> void launch_rows_tiles(const GroupedArgs& a, bool direct, bool larger, hipStream_t s);
template <typename T> void launch_dw_tiles(const GroupedArgs& a, bool direct, bool larger, int splits, hipStream_t s);

// offsets[e], within the positions (M < 2^30).
__device__ __forceinline__ int offset_at(const GroupedArgs& a, int e) {
  if (e <= 0) return 0;
  const int64_t v = a.off64 ? static_cast<const int64_t*>(a.offsets)[e] : static_cast<const int32_t*>(a.offsets)[e];
  return (int)(v < 0 ? 0 : (v < a.M ? v : a.M));
}

// Rows of x at the positions at(0) .. at(N - 1), as read: in flight together (a wait for each would cost the
// chain of them).  in_x() brings one into x.
template <int N, typename F>
__device__ __forceinline__ void source_rows(const GroupedArgs& a, int (&row)[N], F&& at) {
  if (a.rows) {
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = a.rows[at(i)];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) row[i] = at(i);
  }
}
__device__ __forceinline__ int in_x(const GroupedArgs& a, int row) { return min(max(row, 0), (int)a.Nx - 1); }

template <int BM>
__device__ __forceinline__ int tiles_of(int lo, int hi) {
  return hi > lo ? (hi - lo + BM - 1) / BM : 0;
}

// Part `part` of `parts` of positions lo .. hi - 1, in whole 64s.
__device__ __forceinline__ void split_part(int& lo, int& hi, int part, int parts) {
  const int per = ((hi - lo + parts - 1) / parts + 63) / 64 * 64;
  const int64_t from = lo + (int64_t)part * per;
  lo = from < hi ? (int)from : hi;
  hi = from + per < hi ? (int)(from + per) : hi;
}

// The type that a weight gradient's kernel writes.
template <typename T, bool SPLIT> struct Result { typedef T type; };
template <typename T> struct Result<T, true> { typedef float type; };

// Tile number of a workgroup among `total`: consecutive workgroups go to the 8 XCDs in turn, so each XCD
// gets a contiguous run of tiles, whose operands its L2 keeps.
__device__ __forceinline__ int xcd_tile(int id, int total) {
  const int per = total / 8, rest = total % 8, x = id % 8;
  return x * per + (x < rest ? x : rest) + id / 8;
}

// The tile of workgroup `id`: its group, positions (BM a tile) and column tile (of `ntiles`, innermost).
// Group E is the rows past the last group.  False: there is no such tile; the grid holds the most that
// ascending offsets can give.  Every wave counts the groups' tiles for itself, 64 groups at a time.
template <int BM>
__device__ __forceinline__ bool find_tile(const GroupedArgs& a, int id, int ntiles, int& group, int& first, int& end,
                                          int& ntile) {
  const int lane = threadIdx.x & 63;
  int all = 0, past = 0, lo = 0, hi = 0;
  for (int base = 0; base < a.E; base += 64) {
    const int e = base + lane;
    lo = e < a.E ? offset_at(a, e) : 0;
    hi = e < a.E ? offset_at(a, e + 1) : 0;
    all += tiles_of<BM>(lo, hi);
    past = max(past, hi);
  }
#pragma unroll
  for (int off = 32; off >= 1; off /= 2) {
    all += __shfl_xor(all, off);
    past = max(past, __shfl_xor(past, off));
  }
  all = __builtin_amdgcn_readfirstlane(all + tiles_of<BM>(past, (int)a.M)) * ntiles;
  if (id >= all) return false;
  const int tile = xcd_tile(id, all), t = tile / ntiles;
  ntile = tile - t * ntiles;
  int before = 0;
  for (int base = 0; base <= a.E; base += 64) {
    const int e = base + lane;
    if (a.E >= 64) {      // (else as they were)
      lo = e < a.E ? offset_at(a, e) : 0;
      hi = e < a.E ? offset_at(a, e + 1) : 0;
    }
    if (e == a.E) {
      lo = past;
      hi = (int)a.M;
    }
    const int tiles = tiles_of<BM>(lo, hi);
    int incl = tiles;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int v = __shfl_up(incl, off);
      if (lane >= off) incl += v;
    }
    const uint64_t hit = __ballot(before + incl > t);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      const int skipped = before + __shfl(incl - tiles, src);
      group = __builtin_amdgcn_readfirstlane(base + src);
      first = __builtin_amdgcn_readfirstlane(__shfl(lo, src) + (t - skipped) * BM);
      end = __builtin_amdgcn_readfirstlane(__shfl(hi, src));
      return true;
    }
    before += __shfl(incl, 63);
  }
  return false;
}

}  // namespace gx::layer
