// Tile lookup shared by the grouped products' kernels.
#pragma once

#include "experts.hpp"
#include "rows.hpp"

namespace gx::layer {

typedef __bf16 bf16_t;

__device__ __forceinline__ int64_t offset_at(const GroupedArgs& a, int e) {
  const int64_t v = e <= 0 ? 0 : a.off64 ? static_cast<const int64_t*>(a.offsets)[e] : static_cast<const int32_t*>(a.offsets)[e];
  return v < 0 ? 0 : (v < a.M ? v : a.M);
}

// Row of x at position p, within x.
__device__ __forceinline__ int64_t source_row(const GroupedArgs& a, int64_t p) {
  int64_t src = a.rows ? a.rows[p] : p;
  return src < 0 ? 0 : (src < a.Nx ? src : a.Nx - 1);
}

// Group and first position of row tile t (BM positions each): group E is the rows
// past the last group.  False: there is no such tile.
template <int BM>
__device__ __forceinline__ bool find_tile(const GroupedArgs& a, int64_t t, int& group, int64_t& first, int64_t& end) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int base = 0; base <= a.E; base += 64) {
    const int e = base + lane;
    int64_t lo = 0, hi = 0;
    if (e <= a.E) {
      lo = offset_at(a, e);
      hi = e < a.E ? offset_at(a, e + 1) : a.M;
    }
    const int64_t tiles = hi > lo ? (hi - lo + BM - 1) / BM : 0;
    int64_t incl = tiles;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int64_t v = __shfl_up(incl, off);
      if (lane >= off) incl += v;
    }
    const uint64_t hit = __ballot(before + incl > t);
    if (hit) {
      const int src = __ffsll((unsigned long long)hit) - 1;
      const int64_t skipped = before + __shfl(incl - tiles, src);
      group = base + src;
      first = __shfl(lo, src) + (t - skipped) * BM;
      end = __shfl(hi, src);
      return true;
    }
    before += __shfl(incl, 63);
  }
  return false;
}

}  // namespace gx::layer
