// Rows of a table looked up by token, and the table's gradient.
//
//   out[t] = scale table[index[t]],   dtable[v] = scale Σ_{t: index[t] = v} dy[t]
//
// A token outside 0 .. V-1 gives zeros and adds nothing.  The gradient is summed in the
// order of the sorted tokens (equal ones by position): a stable radix sort of the tokens,
// then tiles of kTile sorted positions, which add each run of equal tokens in fp32.  A run
// inside a tile is a row of the result, rounded once; the parts of a run that reaches over
// tiles are written as fp32 (at most two rows a tile: the run that enters it and the run
// that leaves it) and added in order by a second kernel, a workgroup for each run and
// columns.  Rows without a token, of which the sort's last pass leaves a mark in every other, are zeroed
// by workgroups of the same launch.  No sum depends on the order in which
// workgroups finish.
//
// The sort takes the fewest passes of at most 11 bits; a pass counts digits by block,
// turns the counts into prefixes over the blocks and places: waves rank 64 tokens at a
// time by ballots over the digit's bits.  Few tokens are sorted by one workgroup, or in parts that are merged.
//
// 16384 tokens of 65536, 2048 columns bf16: lookup 25 us (rows written once, the frequent ones read from
// caches: 87 MB at the least, 17 us); sort 15 us, sums 69 us (335 MB, 4.9 TB/s: bytes), parts of
// runs 8 us.  100003 of 500, 100 columns fp32: 12; 15, 12 and 6 us: waits more than bytes.  One token is a launch: 2.5 us.

#include <algorithm>
#include <type_traits>

#include "rows.hpp"
#include "tokens.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;
constexpr int kTile = 32;              // sorted positions whose rows one group of threads adds
constexpr int kMaxBits = 11;
constexpr int kSortThreads = 512;
constexpr int kSortRows = 1024;        // tokens of a block of the sort, more where that gives over kMaxSortBlocks
constexpr int64_t kMaxSortBlocks = 4096;
constexpr int kFewBlocks = 32;         // up to which the blocks form the prefixes themselves
constexpr int64_t kMaxBlocks = 1 << 20;

__host__ __device__ inline int key_bits(int64_t V) {
  int b = 1;
  while ((int64_t(1) << b) <= V) ++b;  // keys 0 .. V
  return b;
}

int64_t sort_rows(int64_t N) {
  int64_t r = kSortRows;
  while ((N + r - 1) / r > kMaxSortBlocks) r *= 2;
  return r;
}

__device__ __forceinline__ int64_t token_at(const EmbedArgs& a, int64_t t) {
  return a.index64 ? static_cast<const int64_t*>(a.index)[t] : static_cast<const int32_t*>(a.index)[t];
}

// --- lookup -------------------------------------------------------------------

// tx threads (a power of two) share a row's vectors; each takes four rows at a time.
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void embed_kernel(EmbedArgs a, int tx) {
  constexpr int V = kVec<T>, U = 4;
  const int lane = threadIdx.x & (tx - 1), rpb = kThreads / tx;
  const T* table = static_cast<const T*>(a.table);
  for (int64_t n0 = (int64_t)blockIdx.x * rpb * U + threadIdx.x / tx; n0 < a.N; n0 += (int64_t)gridDim.x * rpb * U) {
    int64_t row[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t n = n0 + j * rpb;
      row[j] = n < a.N ? token_at(a, n) : -1;
      if ((uint64_t)row[j] >= (uint64_t)a.V) row[j] = -1;
    }
    for (int c = lane * V; c < a.D; c += tx * V) {
      uint4 u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = fetch16<SHORT>(table + (row[j] < 0 ? 0 : row[j]) * a.ldt + c, a.D - c);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t n = n0 + j * rpb;
        float v[V];
        unpack16<T>(keep16<SHORT, T>(u[j], a.D - c, a.D), v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = row[j] < 0 ? 0.f : v[i] * a.scale;
        if (n < a.N) store_row(static_cast<T*>(a.out) + n * a.D + c, a.D - c, v);
      }
    }
  }
}

// --- sort ---------------------------------------------------------------------

// The token of sorted-so-far place i: of the first pass the given ones, V for none.
__device__ __forceinline__ uint32_t key_at(const EmbedArgs& a, int from, int64_t i) {
  if (from >= 0) return a.key[from][i];
  const int64_t t = token_at(a, i);
  return (uint64_t)t < (uint64_t)a.V ? (uint32_t)t : (uint32_t)a.V;
}

// Zeros in seen, by all threads of the grid (in a launch before those that set it).
__device__ __forceinline__ void clear_seen(const EmbedArgs& a, int threads) {
  for (int64_t i = ((int64_t)blockIdx.x * threads + threadIdx.x) * 16; i < a.V; i += (int64_t)gridDim.x * threads * 16)
    *reinterpret_cast<uint4*>(a.seen + i) = make_uint4(0, 0, 0, 0);      // (room for whole 256 bytes)
}

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(EmbedArgs a, int from, int shift, int bits,
                                                                  int64_t rpb) {
  extern __shared__ int count[];
  const int bins = 1 << bits;
  if (from < 0) clear_seen(a, kSortThreads);
  for (int b = threadIdx.x; b < bins; b += kSortThreads) count[b] = 0;
  __syncthreads();
  const int64_t first = blockIdx.x * rpb, last = first + rpb < a.N ? first + rpb : a.N;
#pragma unroll 2
  for (int64_t i = first + threadIdx.x; i < last; i += kSortThreads)
    atomicAdd(&count[(key_at(a, from, i) >> shift) & (bins - 1)], 1);
  __syncthreads();
  int32_t* hist = a.hist + (int64_t)blockIdx.x * bins;
  for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = count[b];
}

// Exclusive prefixes over the blocks for 16 digits a workgroup: 64 parts of the blocks,
// added up, then written in a second sweep.
constexpr int kScanCols = 16, kScanParts = 64;
__global__ __launch_bounds__(kScanCols* kScanParts) void sort_scan_kernel(EmbedArgs a, int bits, int blocks) {
  __shared__ int part[kScanParts][kScanCols + 1];
  const int cl = threadIdx.x % kScanCols, p = threadIdx.x / kScanCols, bins = 1 << bits;
  const int b = blockIdx.x * kScanCols + cl;
  const int per = (blocks + kScanParts - 1) / kScanParts;
  const int b0 = p * per < blocks ? p * per : blocks, b1 = b0 + per < blocks ? b0 + per : blocks;
  int s = 0;
  if (b < bins) {
#pragma unroll 4
    for (int i = b0; i < b1; ++i) s += a.hist[(int64_t)i * bins + b];
  }
  part[p][cl] = s;
  __syncthreads();
  int before = 0;
  for (int q = 0; q < p; ++q) before += part[q][cl];
  if (b < bins) {
#pragma unroll 4
    for (int i = b0; i < b1; ++i) {
      int32_t* h = a.hist + (int64_t)i * bins + b;
      const int n = *h;
      *h = before;
      before += n;
    }
    if (p == kScanParts - 1) a.totals[b] = before;
  }
}

// FEW: the counts are as they were counted.
template <bool FEW>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(EmbedArgs a, int from, int to, int shift, int bits,
                                                                  int64_t rpb, int last_pass) {
  constexpr int W = kSortThreads / 64, PER = (1 << kMaxBits) / kSortThreads;
  extern __shared__ int next[];        // [W][bins]: counts of a wave's part, then the next place of each digit
  __shared__ int wave_sum[W];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
  const int64_t first = blockIdx.x * rpb, last = first + rpb < a.N ? first + rpb : a.N;
  const int64_t per = (last - first + W * 64 - 1) / (W * 64) * 64;
  const int64_t lo = first + w * per < last ? first + w * per : last, hi = lo + per < last ? lo + per : last;
  // This thread's digits, a contiguous part of them: how many there are in all, and in the blocks before.
  const int chunk = (bins + kSortThreads - 1) / kSortThreads, b0 = threadIdx.x * chunk;
  int total[PER], before[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = b0 + j;
    const bool in = j < chunk && b < bins;
    total[j] = before[j] = 0;
    if constexpr (FEW) {
      if (in) {
#pragma unroll 8
        for (int i = 0; i < (int)gridDim.x; ++i) {
          const int n = a.hist[i * bins + b];
          total[j] += n;
          before[j] += i < (int)blockIdx.x ? n : 0;
        }
      }
    } else if (in) {
      total[j] = a.totals[b];
      before[j] = a.hist[(int64_t)blockIdx.x * bins + b];
    }
  }
  for (int b = threadIdx.x; b < W * bins; b += kSortThreads) next[b] = 0;
  __syncthreads();
#pragma unroll 2
  for (int64_t i = lo + lane; i < hi; i += 64) atomicAdd(&next[w * bins + ((key_at(a, from, i) >> shift) & (bins - 1))], 1);
  // The digits' first places: an exclusive scan of the totals.
  int s = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) s += total[j];
  const int incl = lanes_scan(s, [](int p, int q) { return p + q; });
  if (lane == 63) wave_sum[w] = incl;
  __syncthreads();
  int at0 = incl - s;
  for (int q = 0; q < w; ++q) at0 += wave_sum[q];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = b0 + j;
    if (j < chunk && b < bins) {
      int at = at0 + before[j];
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int n = next[q * bins + b];
        next[q * bins + b] = at;
        at += n;
      }
      at0 += total[j];
    }
  }
  __syncthreads();
  for (int64_t i0 = lo; i0 < hi; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool in = i < hi;
    const uint32_t key = in ? key_at(a, from, i) : 0;
    const int32_t pos = !in ? 0 : from < 0 ? (int32_t)i : a.pos[from][i];
    const int d = (key >> shift) & (bins - 1);
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int at = next[w * bins + d] + rank;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && rank == 0) next[w * bins + d] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      a.key[to][at] = key;
      a.pos[to][at] = pos;
      if (last_pass && key < a.V) a.seen[key] = 1;
    }
  }
}

// A part of `rows` tokens sorted by a workgroup in LDS, at most kOneBits a pass.  Up to kOneRows tokens are one part: a
// training step of few tokens takes one launch for the sort where it took up to six (each several us of the
// host's time).  Up to kMergeRows, parts of kPart tokens are sorted so and then merged: 4096, 16384 and 32768 tokens of 17
// bits in 11, 16 and 22 us, where one workgroup takes 15 us for 4096 and digits over all of them 20, 22 and 27.
constexpr int kOneRows = 2048, kOneThreads = 1024, kOneBits = 9;
constexpr int kPart = 1024, kMergeRows = 32768;
// Rows whose marks few workgroups clear: of more, the sort by parts has workgroups that do nothing else (2000 tokens of
// 2^24 rows 16 us against 119, 5000 of them 19 against 35, 1000 of a million 13 against 16).
constexpr int kOneClear = 1 << 18;
__global__ __launch_bounds__(kOneThreads) void sort_one_kernel(EmbedArgs a, int rows, int all, int bits) {
  constexpr int W = kOneThreads / 64, Bins = 1 << kOneBits;
  __shared__ uint32_t key[2][kOneRows];
  __shared__ uint16_t pos[2][kOneRows];
  __shared__ int next[W][Bins], wave_sum[Bins / 64];
  const int base = blockIdx.x * rows, N = max(min((int)a.N - base, rows), 0);   // (the last workgroups only clear)
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int per = (N + W * 64 - 1) / (W * 64) * 64, lo = min(w * per, N), hi = min(lo + per, N);
  for (int i = threadIdx.x; i < N; i += kOneThreads) {
    key[0][i] = key_at(a, -1, base + i);
    pos[0][i] = (uint16_t)i;
  }
  clear_seen(a, kOneThreads);
  int from = 0;
  for (int shift = 0; shift < all; shift += bits, from ^= 1) {
    for (int b = threadIdx.x; b < W * Bins; b += kOneThreads) next[0][b] = 0;
    __syncthreads();
    for (int i = lo + lane; i < hi; i += 64) atomicAdd(&next[w][key[from][i] >> shift & ((1 << bits) - 1)], 1);
    __syncthreads();
    int total = 0, incl = 0;
    if (threadIdx.x < Bins) {
#pragma unroll
      for (int q = 0; q < W; ++q) total += next[q][threadIdx.x];
      incl = lanes_scan(total, [](int p, int q) { return p + q; });
      if (lane == 63) wave_sum[w] = incl;
    }
    __syncthreads();
    if (threadIdx.x < Bins) {
      int at = incl - total;
      for (int q = 0; q < w; ++q) at += wave_sum[q];
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int n = next[q][threadIdx.x];
        next[q][threadIdx.x] = at;
        at += n;
      }
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const int i = i0 + lane;
      const bool in = i < hi;
      const uint32_t k = in ? key[from][i] : 0;
      const int d = k >> shift & ((1 << bits) - 1);
      uint64_t same = __ballot(in);
      for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int at = next[w][d] + rank;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (in && rank == 0) next[w][d] += __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (in) {
        key[from ^ 1][at] = k;
        pos[from ^ 1][at] = pos[from][i];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < N; i += kOneThreads) {
    a.key[0][base + i] = key[from][i];
    a.pos[0][base + i] = base + pos[from][i];
    if (gridDim.x == 1 && key[from][i] < a.V) a.seen[key[from][i]] = 1;
  }
}

// The sorted parts merged: a token's place is its own in its part and, of every other part, how many come before it
// (equal ones too where the part does), which binary searches in all parts' tokens in LDS count, four at a time.
__global__ __launch_bounds__(kThreads) void sort_merge_kernel(EmbedArgs a, int parts) {
  extern __shared__ __align__(16) uint32_t part_keys[];
  constexpr int L = kPart / 4 * 4 / kThreads;             // 16 bytes at a time, four parts' in flight
  for (int t0 = 0; t0 < parts; t0 += 4) {
    uint4 v[L];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int i = (t0 * (kPart / 4) + j * kThreads + (int)threadIdx.x) * 4;
      v[j] = i < a.N ? *reinterpret_cast<const uint4*>(a.key[0] + i) : make_uint4(~0u, ~0u, ~0u, ~0u);   // (256 bytes)
      if (i + 1 >= a.N) v[j].y = ~0u;
      if (i + 2 >= a.N) v[j].z = ~0u;
      if (i + 3 >= a.N) v[j].w = ~0u;
    }
#pragma unroll
    for (int j = 0; j < L; ++j) {
      const int i = t0 * (kPart / 4) + j * kThreads + threadIdx.x;
      if (i < parts * (kPart / 4)) reinterpret_cast<uint4*>(part_keys)[i] = v[j];
    }
  }
  __syncthreads();
  const int i = blockIdx.x * kThreads + threadIdx.x, mine = i / kPart;
  if (i >= a.N) return;
  const uint32_t key = part_keys[i];
  const int32_t pos = a.pos[0][i];
  int place = i % kPart;
  constexpr int U = 4;
  for (int t0 = 0; t0 < parts; t0 += U) {
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = 0;
#pragma unroll
    for (int step = kPart / 2; step >= 1; step /= 2)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = min(t0 + u, parts - 1);
        at[u] += part_keys[t * kPart + at[u] + step - 1] < key + (t < mine) ? step : 0;
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(t0 + u, parts - 1);
      at[u] += part_keys[t * kPart + at[u]] < key + (t < mine);
      place += t0 + u < parts && t != mine ? at[u] : 0;
    }
  }
  a.key[1][place] = key;
  a.pos[1][place] = pos;
  if (key < a.V) a.seen[key] = 1;
}

// --- sums ---------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ void store_scaled(T* p, int valid, const float (&v)[kVec<T>], float scale) {
  float o[kVec<T>];
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) o[i] = v[i] * scale;
  store_row(p, valid, o);
}
template <int V>
__device__ __forceinline__ void store_part(float* p, int valid, const float (&v)[V]) {
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    const float q[4] = {v[h], v[h + 1], v[h + 2], v[h + 3]};
    if (valid > h) store_row(p + h, valid - h, q);
  }
}

// The first `tiles` workgroups along x add tiles, the others zero rows without a token (64 rows each).  tx threads
// share a tile's columns; y counts columns of tx V.
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(EmbedArgs a, int tx, int64_t tile_blocks, int sorted) {
  constexpr int V = kVec<T>, U = 8;
  const uint32_t* key = a.key[sorted];
  T* out = static_cast<T*>(a.out);
  if ((int64_t)blockIdx.x >= tile_blocks) {
    __shared__ uint8_t seen[64];
    const int64_t v0 = ((int64_t)blockIdx.x - tile_blocks) * 64;
    if (threadIdx.x < 64) seen[threadIdx.x] = v0 + threadIdx.x < a.V ? a.seen[v0 + threadIdx.x] : 1;
    __syncthreads();
    const int lane = threadIdx.x & (tx - 1), step = kThreads / tx;
    float zero[V] = {};
    const int c = ((int)blockIdx.y * tx + lane) * V;
    if (c < a.D)
      for (int r = threadIdx.x / tx; r < 64 && v0 + r < a.V; r += step)
        if (!seen[r]) store_row(out + (v0 + r) * a.D + c, a.D - c, zero);
    return;
  }
  const int lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx, per = kThreads / tx;
  // This workgroup's tiles: their tokens, with those before and after, their positions and where their runs end.
  __shared__ uint32_t keys[kThreads / 8][kTile + 2], ends[kThreads / 8];
  __shared__ int32_t pos[kThreads / 8][kTile];
  const uint32_t none = (uint32_t)a.V;
  const int64_t t0 = (int64_t)blockIdx.x * per;
  if ((int)threadIdx.x < per) ends[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < per * (kTile + 2); i += kThreads) {
    const int64_t at = (t0 + i / (kTile + 2)) * kTile + i % (kTile + 2) - 1;
    keys[i / (kTile + 2)][i % (kTile + 2)] = at >= 0 && at < a.N ? key[at] : none;
  }
  for (int i = threadIdx.x; i < per * kTile; i += kThreads) {
    const int64_t at = t0 * kTile + i;
    pos[i / kTile][i % kTile] = at < a.N ? a.pos[sorted][at] : 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < per * kTile; i += kThreads) {
    const uint32_t* k = keys[i / kTile] + 1 + i % kTile;
    if (k[0] != none && (k[0] != k[1] || i % kTile == kTile - 1)) atomicOr(&ends[i / kTile], 1u << (i % kTile));
  }
  __syncthreads();
  const int c = ((int)blockIdx.y * tx + lane) * V;
  const int64_t tile = t0 + sub;
  const uint32_t marks = ends[sub];
  if (c >= a.D || marks == 0) return;              // (no token in it)
  const int n = 32 - __clz((int)marks);            // its tokens: a run ends with the last of them
  const uint32_t* k = keys[sub] + 1;
  const T* dy = static_cast<const T*>(a.dy) + c;
  float acc[V] = {};
  bool entered = tile > 0 && k[-1] == k[0];        // the run at hand began in an earlier tile
  const bool leaves = n == kTile && k[kTile] == k[kTile - 1];
  uint4 next[U];
  const auto fetch = [&](int i0) {
#pragma unroll
    for (int j = 0; j < U; ++j) next[j] = fetch16<SHORT>(dy + (int64_t)pos[sub][i0 + j] * a.lddy, a.D - c);
  };
  fetch(0);
  for (int i0 = 0; i0 < n; i0 += U) {
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = next[j];
    if (i0 + U < n) fetch(i0 + U);
#pragma unroll
    for (int j = 0; j < U; ++j) {                  // (what is added after the last end is not used)
      float v[V];
      unpack16<T>(keep16<SHORT, T>(u[j], a.D - c, a.D), v);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += v[i];
      if (marks >> (i0 + j) & 1) {
        const bool away = leaves && i0 + j == kTile - 1;
        if (entered || away) store_part(a.part + (tile * 2 + !entered) * a.D + c, a.D - c, acc);
        else store_scaled(out + (int64_t)k[i0 + j] * a.D + c, a.D - c, acc, a.scale);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
        entered = false;
      }
    }
  }
}

// The runs that leave the tile in which they began: that tile's part and those of the tiles after it.  A workgroup
// takes a tile and 64 V columns, its four waves contiguous parts of the run.
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void embed_join_kernel(EmbedArgs a, int sorted) {
  constexpr int V = 4, W = kThreads / 64;
  const uint32_t* key = a.key[sorted];
  const int64_t tiles = (a.N + kTile - 1) / kTile;
  __shared__ float sums[W][64][V + 1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = ((int)blockIdx.y * 64 + lane) * V;
  for (int64_t tile = blockIdx.x; tile + 1 < tiles; tile += gridDim.x) {
    // (the keys at the tile's ends and at the starts of the next 64 tiles, in flight together)
    const uint32_t v = key[tile * kTile + kTile - 1], start = key[tile * kTile], prior = tile > 0 ? key[tile * kTile - 1] : ~0u;
    const auto starts = [&](int64_t q) { return (tile + q) * kTile < a.N ? key[(tile + q) * kTile] : ~0u; };
    uint64_t same = __ballot(starts(1 + lane) == v);
    if (v == (uint32_t)a.V || !(same & 1) || (start == v && prior == v)) continue;
    int64_t parts = 0;                                          // tiles after this one that the run enters
    while (same == ~0ull) {
      parts += 64;
      same = __ballot(starts(parts + 1 + lane) == v);
    }
    parts += __ffsll((unsigned long long)~same) - 1;
    const int64_t per = (parts + W - 1) / W, lo = w * per < parts ? w * per : parts, hi = lo + per < parts ? lo + per : parts;
    float acc[V] = {};
    if (c < a.D) {
      const auto part = [&](int64_t row) { return fetch16<SHORT>(a.part + row * a.D + c, a.D - c); };
      const auto add = [&](uint4 u) {
        float v[V];
        unpack16<float>(keep16<SHORT, float>(u, a.D - c, a.D), v);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += v[i];
      };
      if (w == 0) add(part(tile * 2 + 1));
      constexpr int U = 8;             // rows in flight
      int64_t q = lo;
      for (; q + U <= hi; q += U) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = part((tile + 1 + q + j) * 2);
#pragma unroll
        for (int j = 0; j < U; ++j) add(u[j]);
      }
      for (; q < hi; ++q) add(part((tile + 1 + q) * 2));
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[w][lane][i] = acc[i];
    __syncthreads();
    if (w == 0 && c < a.D) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int q = 1; q < W; ++q) acc[i] += sums[q][lane][i];
        if (c + i < a.D) static_cast<T*>(a.out)[(int64_t)v * a.D + c + i] = (T)(acc[i] * a.scale);
      }
    }
    __syncthreads();
  }
}

int threads_for(int nvec) {
  int tx = 8;
  while (tx < nvec && tx < kThreads) tx *= 2;
  return tx;
}

template <typename T>
void embed_typed(const EmbedArgs& a, hipStream_t s) {
  const int tx = threads_for((a.D + kVec<T> - 1) / kVec<T>);
  const int64_t rows = kThreads / tx * 4, need = (a.N + rows - 1) / rows;
  const unsigned grid = (unsigned)(need < kMaxBlocks ? need : kMaxBlocks);
  if (a.D < kVec<T>) embed_kernel<T, true><<<grid, kThreads, 0, s>>>(a, tx);
  else embed_kernel<T, false><<<grid, kThreads, 0, s>>>(a, tx);
}

template <typename T>
void embed_sum_typed(const EmbedArgs& a, int sorted, hipStream_t s) {
  const int nvec = (a.D + kVec<T> - 1) / kVec<T>, tx = threads_for(nvec), per = kThreads / tx;
  const int64_t tiles = (a.N + kTile - 1) / kTile, tile_blocks = (tiles + per - 1) / per;
  const dim3 grid((unsigned)(tile_blocks + (a.V + 63) / 64), (unsigned)((nvec + tx - 1) / tx));
  if (a.D < kVec<T>) embed_sum_kernel<T, true><<<grid, kThreads, 0, s>>>(a, tx, tile_blocks, sorted);
  else embed_sum_kernel<T, false><<<grid, kThreads, 0, s>>>(a, tx, tile_blocks, sorted);
  if (tiles > 1) {
    const dim3 join((unsigned)(tiles - 1 < 65536 ? tiles - 1 : 65536), (unsigned)((a.D + 255) / 256));
    if (a.D < 4) embed_join_kernel<T, true><<<join, kThreads, 0, s>>>(a, sorted);
    else embed_join_kernel<T, false><<<join, kThreads, 0, s>>>(a, sorted);
  }
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

int64_t embed_workspace_bytes(int64_t N, int64_t V, int D) {
  EmbedArgs a{};
  a.N = N; a.V = V; a.D = D;
  embed_workspace(a, nullptr);
  const int64_t tiles = (N + kTile - 1) / kTile;
  return reinterpret_cast<int64_t>(a.part) + align256(tiles * 2 * D * 4);
}

void embed_workspace(EmbedArgs& a, void* ws) {
  char* p = static_cast<char*>(ws);
  auto take = [&](auto*& at, int64_t bytes) {
    at = reinterpret_cast<std::decay_t<decltype(at)>>(p);
    p += align256(bytes);
  };
  const int64_t rpb = sort_rows(a.N), blocks = (a.N + rpb - 1) / rpb;
  const int bits = key_bits(a.V), passes = (bits + kMaxBits - 1) / kMaxBits, digit = (bits + passes - 1) / passes;
  for (int i = 0; i < 2; ++i) take(a.key[i], a.N * 4);
  for (int i = 0; i < 2; ++i) take(a.pos[i], a.N * 4);
  take(a.hist, blocks * (int64_t(1) << digit) * 4);
  take(a.totals, (int64_t(1) << digit) * 4);
  take(a.seen, a.V);
  a.part = reinterpret_cast<float*>(p);
}

void launch_embed(const EmbedArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) embed_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) embed_typed<__bf16>(a, s);
  else embed_typed<_Float16>(a, s);
}

void launch_embed_bwd(const EmbedArgs& a, hipStream_t s) {
  const int64_t rpb = sort_rows(a.N);
  const unsigned blocks = (unsigned)((a.N + rpb - 1) / rpb);
  const int all = key_bits(a.V), passes = (all + kMaxBits - 1) / kMaxBits, bits = (all + passes - 1) / passes;
  int from = -1;
  const int one = (all + kOneBits - 1) / kOneBits, one_bits = (all + one - 1) / one;
  if (a.N <= kOneRows && a.V <= kOneClear) {
    sort_one_kernel<<<1, kOneThreads, 0, s>>>(a, kOneRows, all, one_bits);
    from = 0;
  } else if (a.N <= kMergeRows && passes > 1) {
    const int parts = (int)((a.N + kPart - 1) / kPart);
    const int clear = (int)std::min<int64_t>(a.V / (kOneClear / 4), 256);
    sort_one_kernel<<<std::max(parts, clear), kOneThreads, 0, s>>>(a, kPart, all, one_bits);
    sort_merge_kernel<<<(unsigned)((a.N + kThreads - 1) / kThreads), kThreads, parts * kPart * 4, s>>>(a, parts);
    from = 1;
  } else {
    for (int p = 0; p < passes; ++p) {
      const int to = p & 1, bins = 1 << bits;
      const size_t lds = kSortThreads / 64 * bins * 4;
      sort_count_kernel<<<blocks, kSortThreads, bins * 4, s>>>(a, from, p * bits, bits, rpb);
      if ((int)blocks <= kFewBlocks) {
        sort_place_kernel<true><<<blocks, kSortThreads, lds, s>>>(a, from, to, p * bits, bits, rpb, p + 1 == passes);
      } else {
        sort_scan_kernel<<<(bins + kScanCols - 1) / kScanCols, kScanCols * kScanParts, 0, s>>>(a, bits, (int)blocks);
        sort_place_kernel<false><<<blocks, kSortThreads, lds, s>>>(a, from, to, p * bits, bits, rpb, p + 1 == passes);
      }
      from = to;
    }
  }
  if (a.elem == ELEM_F32) embed_sum_typed<float>(a, from, s);
  else if (a.elem == ELEM_BF16) embed_sum_typed<__bf16>(a, from, s);
  else embed_sum_typed<_Float16>(a, from, s);
}

}  // namespace gx::layer
