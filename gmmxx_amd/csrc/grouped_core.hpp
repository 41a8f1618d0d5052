// Tile lookup shared by the grouped products' kernels.
#pragma once

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

typedef __bf16 bf16_t;

// The tiles (grouped_tiles.hpp): by direct loads or not, 256 wide (16-bit elements, direct) or 128.
template <typename T> void launch_rows_tiles(const GroupedArgs& a, bool direct, bool larger, hipStream_t s);
template <typename T> void launch_dw_tiles(const GroupedArgs& a, bool direct, bool larger, int splits, hipStream_t s);

// A grid of `blocks` workgroups and `parts` along y.  A dimension's threads are counted in 32 bits, so what passes
// 2^31 of them goes along z (the last layer may have workgroups to spare).
inline dim3 grid_of(int64_t blocks, int threads, int parts = 1) {
  const int64_t most = (int64_t(1) << 31) / threads;
  if (blocks <= most) return dim3((unsigned)blocks, (unsigned)parts);
  return dim3((unsigned)most, (unsigned)parts, (unsigned)((blocks + most - 1) / most));
}
__device__ __forceinline__ int block_id() { return (int)(blockIdx.z * gridDim.x + blockIdx.x); }

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

// op over lanes 0 .. l in lane l, for values that are not negative (0 changes nothing): within rows of 16 lanes,
// then across them.
template <typename F>
__device__ __forceinline__ int lanes_scan(int v, F&& op) {
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));      // shifted by 1, 2, 4 and 8 lanes
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));      // lane 15 to rows 1 and 3
  return op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));   // lane 31 to rows 2 and 3
}

// The tile of workgroup `id`: its group, positions (BM a tile) and column tile (of `ntiles`, innermost).
// Group E is the rows past the last group.  False: there is no such tile; the grid holds the most that
// ascending offsets can give.  Every wave counts the groups' tiles for itself, 256 groups at a time: four a lane,
// all their offsets in flight together, since each product waits for this (of 200 groups, 100003 fp32 rows, 32 x
// 128: 25 us, 29 us by 64 groups at a time and sums through LDS).
template <int BM>
__device__ __forceinline__ bool find_tile(const GroupedArgs& a, int id, int ntiles, int& group, int& first, int& end,
                                          int& ntile) {
  constexpr int PER = 4, Sweep = 64 * PER;
  const int lane = threadIdx.x & 63;
  const auto add = [](int p, int q) { return p + q; };
  const auto larger = [](int p, int q) { return p > q ? p : q; };
  int off[PER + 1], count = 0, incl = 0;
  auto sweep = [&](int base) {
#pragma unroll
    for (int i = 0; i <= PER; ++i) off[i] = offset_at(a, min(base + lane * PER + i, a.E));
    count = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) count += tiles_of<BM>(off[i], off[i + 1]);
    incl = lanes_scan(count, add);
  };
  int all = 0, past = 0;
  for (int base = 0; base < a.E; base += Sweep) {
    sweep(base);
    all += __builtin_amdgcn_readlane(incl, 63);
    int most = off[0];
#pragma unroll
    for (int i = 1; i <= PER; ++i) most = max(most, off[i]);
    past = max(past, __builtin_amdgcn_readlane(lanes_scan(most, larger), 63));
  }
  const int total = (all + tiles_of<BM>(past, (int)a.M)) * ntiles;
  if (id >= total) return false;
  const int tile = xcd_tile(id, total), t = tile / ntiles;
  ntile = tile - t * ntiles;
  if (t >= all) {
    group = a.E;
    first = past + (t - all) * BM;
    end = (int)a.M;
    return true;
  }
  int before = 0;
  for (int base = 0; base < a.E; base += Sweep) {
    if (a.E > Sweep) sweep(base);      // (else as they were)
    const uint64_t hit = __ballot(before + incl > t);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      int rest = t - before - __builtin_amdgcn_readlane(incl - count, src);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int lo = __builtin_amdgcn_readlane(off[i], src), hi = __builtin_amdgcn_readlane(off[i + 1], src);
        const int tiles = tiles_of<BM>(lo, hi);
        if (rest >= 0 && rest < tiles) {
          group = base + src * PER + i;
          first = lo + rest * BM;
          end = hi;
        }
        rest -= tiles;
      }
      return true;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

}  // namespace gx::layer
