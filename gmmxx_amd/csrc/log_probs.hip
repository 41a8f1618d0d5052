// Log probabilities of given tokens under rows of scores, the rows' entropies, the best
// alternatives, and the gradient of all three.
//
// A row's candidates are its scores that are neither -inf nor NaN.  With m the largest,
// d = s - m, Z = Σ e^d and U = Σ e^d d over the candidates:
//   log p_t = d_t - log Z,   H = -Σ p log p = log Z - U / Z
// (both terms of H are non-negative: nothing cancels).  Of several +inf each has
// p = 1 / their number.  The gradient from g (chosen), h (entropy) and q (alternatives) is
//   ds_j = g [j = t] + Σ_i q_i [j = top_i] - p_j (g + Σ_i q_i + h (log p_j + H)).
//
// One pass over the scores: a thread keeps its own (m, Z, U), brought to a larger m where
// one comes up (once a 16-byte vector at most), and the threads' are merged at the end, in
// a fixed order.  Rows are cut into parts where there are too few for the card, and joined by
// a second kernel.
//
// Alternatives are found in the same pass.  A score's rank is a 64-bit number, its value
// above its complemented index, so no two are equal and ties go to the lower index.  The
// first scores give a bound that k of them reach; scores that reach the bound go to a list in LDS,
// which is cut back to its k largest when it may overflow (its k-th by bisection over the
// rank's bits) and raises the bound.  The list's order depends on the waves', what is kept of it
// does not.

#include <math.h>

#include "rows.hpp"
#include "tokens.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 1 << 20;

// exp(d) for d <= 0, which takes NaN and -inf to 0; `d` comes back as at least -110, where exp is 0.
__device__ __forceinline__ float exp_below(float& d) {
  d = fmaxf(d, -110.f);
  return fast_exp2(d * kLog2e);
}

// Scores seen: the largest, Σ e^(s - m), Σ e^(s - m) (s - m).  m = -inf: none yet.  A largest of +inf leaves sums
// that do not count (see finish).
struct Stats {
  float m = -INFINITY, z = 0.f, u = 0.f;
  __device__ __forceinline__ void raise(float to) {      // to >= m
    const float by = m - to;
    if (by == 0.f || m == to) return;
    const float f = m == -INFINITY ? 0.f : __expf(fmaxf(by, -110.f));
    u = f == 0.f ? 0.f : f * fmaf(z, by, u);
    z *= f;
    m = to;
  }
  template <int V>
  __device__ __forceinline__ void add(const float (&s)[V]) {
    float top = s[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = fmaxf(top, s[i]);
    if (top > m) raise(top);
    float zv = 0.f, uv = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float d = s[i] - m;
      const float e = exp_below(d);
      zv += e;
      uv = fmaf(e, d, uv);
    }
    z += zv;
    u += uv;
  }
};

__device__ __forceinline__ Stats merge(Stats a, Stats b) {
  const float to = fmaxf(a.m, b.m);
  a.raise(to);
  b.raise(to);
  a.z += b.z;
  a.u += b.u;
  return a;
}

// The statistics of G lanes' scores, in all of them.
template <int G>
__device__ __forceinline__ Stats lanes_merge(Stats s) {
  const float to = lanes_reduce<G>(s.m, [](float a, float b) { return fmaxf(a, b); });
  s.raise(to);
  s.z = lanes_sum<G>(s.z);
  s.u = lanes_sum<G>(s.u);
  return s;
}

// ... of a workgroup's; `red` takes three floats a wave.
__device__ __forceinline__ Stats block_merge(Stats s, float (*red)[3]) {
  s = lanes_merge<64>(s);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = s.m;
    red[threadIdx.x >> 6][1] = s.z;
    red[threadIdx.x >> 6][2] = s.u;
  }
  __syncthreads();
  Stats r;
  r.m = red[0][0], r.z = red[0][1], r.u = red[0][2];
  for (int w = 1; w < (int)blockDim.x / 64; ++w) {
    Stats o;
    o.m = red[w][0], o.z = red[w][1], o.u = red[w][2];
    r = merge(r, o);
  }
  return r;
}

__device__ __forceinline__ int64_t token_at(const LogpArgs& a, int64_t n) {
  const int64_t t = a.index64 ? static_cast<const int64_t*>(a.index)[n] : static_cast<const int32_t*>(a.index)[n];
  return (uint64_t)t < (uint64_t)a.V ? t : -1;
}

// log p of a score v in a row with largest m.
__device__ __forceinline__ float log_p(float v, float m, float logz) {
  return v > -INFINITY ? (v == m ? -logz : (v - m) - logz) : -INFINITY;
}

// A row's results, by one thread.
template <typename T>
__device__ __forceinline__ float2 finish(const LogpArgs& a, int64_t n, Stats s) {
  const bool some = s.m > -INFINITY;
  const float logz = some ? logf(s.z) : 0.f, h = some ? logz - s.u / s.z : 0.f;
  const int64_t t = token_at(a, n);
  a.chosen[n] = t < 0 ? 0.f : log_p(to_f32(static_cast<const T*>(a.scores)[n * a.lds + t]), s.m, logz);
  a.entropy[n] = h;
  if (a.stats) {
    a.stats[n * 3] = s.m;
    a.stats[n * 3 + 1] = logz;
    a.stats[n * 3 + 2] = h;
  }
  return make_float2(s.m, logz);
}

// How many of a row's scores are +inf, counted by G lanes (at a row whose largest is).
template <typename T, int G>
__device__ __forceinline__ Stats infinite(const LogpArgs& a, int64_t n, int lane) {
  float count = 0.f;
  for (int c = lane; c < a.V; c += G) count += to_f32(static_cast<const T*>(a.scores)[n * a.lds + c]) == INFINITY;
  Stats s;
  s.m = INFINITY;
  s.z = lanes_sum<(G < 64 ? G : 64)>(count);
  return s;
}

// --- no alternatives ------------------------------------------------------------

// G lanes share a row.
template <typename T, int G, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_rows_kernel(LogpArgs a) {
  constexpr int V = kVec<T>, U = 4, R = kThreads / G;
  const int lane = threadIdx.x % G;
  for (int64_t n = (int64_t)blockIdx.x * R + threadIdx.x / G; n < a.N; n += (int64_t)gridDim.x * R) {
    const T* row = static_cast<const T*>(a.scores) + n * a.lds;
    Stats s;
    for (int c0 = lane * V; c0 < a.V; c0 += G * V * U) {
      uint4 u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = c0 + j * G * V;
        u[j] = fetch16<SHORT>(row + (c < a.V ? c : 0), c < a.V ? a.V - c : a.V);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = c0 + j * G * V;
        if (c >= a.V) break;
        float v[V];
        unpack16<T>(keep16<SHORT, T>(u[j], a.V - c, a.V), v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c + i < a.V ? v[i] : -INFINITY;
        s.add(v);
      }
    }
    s = lanes_merge<G>(s);
    if (s.m == INFINITY) s = infinite<T, G>(a, n, lane);
    if (lane == 0) finish<T>(a, n, s);
  }
}

// --- ranks ------------------------------------------------------------------------

// A score's value in integer order; those of -inf and NaN (0) are no candidates.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t rank_of(uint32_t key, int index) { return (uint64_t)key << 32 | (uint32_t)~index; }

constexpr int kTopVectors = 2;                          // a thread's vectors between looks at the list's length
template <typename T>
constexpr int kListRoom = kThreads * kTopVectors * kVec<T>;      // that they may add
template <typename T>
constexpr int kListSize = kListRoom<T> + 1024;

// Keeps the k largest of list[0 .. count - 1] (count > k) in list[0 .. k - 1], in some order; returns the least of
// them.  Their bits are found from the highest: the largest number that at least k of the list reach.
template <int SIZE>
__device__ __forceinline__ uint64_t cut(uint64_t* list, int count, int k, int* scratch) {
  constexpr int PER = (SIZE + kThreads - 1) / kThreads, W = kThreads / 64;
  uint64_t mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kThreads + threadIdx.x;
    mine[i] = at < count ? list[at] : 0;
  }
  uint64_t bound = 0;
  int turn = 0;
  for (int b = 63; b >= 0; --b) {
    const uint64_t test = bound | 1ull << b;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(mine[i] >= test));
    int* slot = scratch + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) n += slot[w];
    if (n >= k) bound = test;
    if (n == k) break;
  }
  __syncthreads();
  if (threadIdx.x == 0) scratch[0] = 0;
  __syncthreads();
  uint64_t least = ~0ull;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (mine[i] >= bound) list[atomicAdd(&scratch[0], 1)] = mine[i];
  __syncthreads();
  for (int i = 0; i < k; ++i) least = list[i] < least ? list[i] : least;
  __syncthreads();
  return least;
}

// The k largest of the list in descending order to out[0 .. k - 1], zeros where there are fewer.
template <int SIZE>
__device__ __forceinline__ void sorted(uint64_t* list, int count, int k, int* scratch, uint64_t* out) {
  if (count > kThreads && count > k) {
    cut<SIZE>(list, count, k, scratch);
    count = k;
  }
  __syncthreads();
  if ((int)threadIdx.x < count) {
    const uint64_t mine = list[threadIdx.x];
    int above = 0;
    for (int i = 0; i < count; ++i) above += list[i] > mine;
    if (above < k) out[above] = mine;
  }
  if ((int)threadIdx.x >= count && (int)threadIdx.x < k) out[threadIdx.x] = 0;
  __syncthreads();
}

// Writes a row's alternatives from their sorted ranks.
__device__ __forceinline__ void write_top(const LogpArgs& a, int64_t n, const uint64_t* top, float2 row) {
  if ((int)threadIdx.x < a.k) {
    const uint64_t r = top[threadIdx.x];
    const float v = value_of((uint32_t)(r >> 32));
    a.top[n * a.k + threadIdx.x] = r ? log_p(v, row.x, row.y) : -INFINITY;
    a.top_index[n * a.k + threadIdx.x] = r ? (int32_t)~(uint32_t)r : -1;
  }
}

// A part of a row (x) of each row (y), with k alternatives (or none); one part: the row's results.
template <typename T, bool TOP, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_part_kernel(LogpArgs a) {
  constexpr int V = kVec<T>, U = TOP ? kTopVectors : 4;
  __shared__ uint64_t list[TOP ? kListSize<T> : 1];
  __shared__ uint64_t out[kLogpMaxK];
  __shared__ float red[kThreads / 64][3];
  __shared__ uint32_t tops[kThreads];
  __shared__ int scratch[2 * kThreads / 64], count, bound0;
  __shared__ float2 result;
  const int split = blockIdx.x;
  for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
    const T* row = static_cast<const T*>(a.scores) + n * a.lds;
    const int per = (int)((((int64_t)a.V + a.splits - 1) / a.splits + V - 1) / V * V);
    const int first = (int64_t)split * per < a.V ? split * per : a.V;
    const int last = first + (int64_t)per < a.V ? first + per : a.V;
    Stats s;
    uint64_t bound = 1;               // (0: no candidate)
    bool fresh = true;
    if (threadIdx.x == 0) count = 0, bound0 = 0;
    __syncthreads();
    for (int base = first; base < last; base += kThreads * V * U) {
      uint4 u[U];
      float v[U][V];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = base + (j * kThreads + (int)threadIdx.x) * V;
        u[j] = fetch16<SHORT>(row + (c < last ? c : 0), c < last ? a.V - c : a.V);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = base + (j * kThreads + (int)threadIdx.x) * V;
        unpack16<T>(keep16<SHORT, T>(u[j], c < last ? a.V - c : a.V, a.V), v[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = c + i < last ? v[j][i] : -INFINITY;
        s.add(v[j]);
      }
      if constexpr (!TOP) continue;
      if (fresh) {                    // a value that k threads' largest reach
        fresh = false;
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) mine = max(mine, key_of(v[j][i]));
        tops[threadIdx.x] = mine;
        __syncthreads();
        int reach = 0;
#pragma unroll 8
        for (int i = 0; i < kThreads; ++i) reach += tops[i] >= mine;
        if (reach >= a.k) atomicMax(reinterpret_cast<uint32_t*>(&bound0), mine);
        __syncthreads();
        const uint64_t b = (uint64_t)(uint32_t)bound0 << 32;
        bound = b > bound ? b : bound;
      }
      const float least = value_of((uint32_t)(bound >> 32));
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = base + (j * kThreads + (int)threadIdx.x) * V;
        float top = v[j][0];
#pragma unroll
        for (int i = 1; i < V; ++i) top = fmaxf(top, v[j][i]);
        if ((bound >> 32) == 0 ? top > -INFINITY : top >= least) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const uint64_t r = rank_of(key_of(v[j][i]), c + i);
            if ((r >> 32) != 0 && r >= bound) list[atomicAdd(&count, 1)] = r;
          }
        }
      }
      __syncthreads();
      const int have = count;
      if (have > kListSize<T> - kListRoom<T>) {
        bound = cut<kListSize<T>>(list, have, a.k, scratch);
        if (threadIdx.x == 0) count = a.k;
      }
      __syncthreads();
    }
    s = block_merge(s, red);
    if constexpr (TOP) sorted<kListSize<T>>(list, count, a.k, scratch, out);
    if (a.splits > 1) {
      const int64_t at = n * a.splits + split;
      if (threadIdx.x == 0) a.part[at * 3] = s.m, a.part[at * 3 + 1] = s.z, a.part[at * 3 + 2] = s.u;
      if (TOP && (int)threadIdx.x < a.k) a.part_top[at * a.k + threadIdx.x] = out[threadIdx.x];
    } else {
      if (s.m == INFINITY) {
        Stats mine = infinite<T, kThreads>(a, n, threadIdx.x);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][1] = mine.z;
        __syncthreads();
        s = Stats();
        s.m = INFINITY;
        for (int w = 0; w < kThreads / 64; ++w) s.z += red[w][1];
      }
      if (threadIdx.x == 0) result = finish<T>(a, n, s);
      __syncthreads();
      if constexpr (TOP) write_top(a, n, out, result);
    }
    __syncthreads();
  }
}

// The parts of a row.
constexpr int kMaxSplits = 64;
template <typename T>
__global__ __launch_bounds__(kThreads) void logp_join_kernel(LogpArgs a) {
  __shared__ uint64_t list[kMaxSplits * kLogpMaxK];
  __shared__ uint64_t out[kLogpMaxK];
  __shared__ float red[kThreads / 64][3];
  __shared__ int scratch[2 * kThreads / 64], count;
  __shared__ float2 result;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    Stats s;
    if ((int)threadIdx.x < a.splits) {
      const float* p = a.part + (n * a.splits + threadIdx.x) * 3;
      s.m = p[0], s.z = p[1], s.u = p[2];
    }
    s = block_merge(s, red);
    if (s.m == INFINITY) {
      Stats mine = infinite<T, kThreads>(a, n, threadIdx.x);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][1] = mine.z;
      __syncthreads();
      s = Stats();
      s.m = INFINITY;
      for (int w = 0; w < kThreads / 64; ++w) s.z += red[w][1];
    }
    if (threadIdx.x == 0) {
      result = finish<T>(a, n, s);
      count = 0;
    }
    __syncthreads();
    if (a.k) {
      // every part's list is sorted: no score below a part's last is among the row's k best
      const uint64_t* p = a.part_top + n * a.splits * a.k;
      uint64_t bound = 1;
      for (int i = 0; i < a.splits; ++i) {
        const uint64_t b = p[i * a.k + a.k - 1];
        bound = b > bound ? b : bound;
      }
      for (int i = threadIdx.x; i < a.splits * a.k; i += kThreads) {
        const uint64_t r = p[i];
        if (r >= bound) list[atomicAdd(&count, 1)] = r;
      }
      __syncthreads();
      sorted<kMaxSplits * kLogpMaxK>(list, count, a.k, scratch, out);
      write_top(a, n, out, result);
    }
    __syncthreads();
  }
}

// --- gradient ---------------------------------------------------------------------

// The factors of a row's p: ds = p (c + h (log p + H)) before what the chosen get.
struct Factors {
  float m, logz, entropy, c, h;
};

// Σ over the alternatives that exist.
__device__ __forceinline__ Factors factors_of(const LogpArgs& a, int64_t n, float dtop) {
  Factors f;
  f.m = a.stats[n * 3], f.logz = a.stats[n * 3 + 1], f.entropy = a.stats[n * 3 + 2];
  f.c = -(a.dchosen && token_at(a, n) >= 0 ? a.dchosen[n] : 0.f) - dtop;
  f.h = a.dentropy ? -a.dentropy[n] : 0.f;
  return f;
}

template <bool INF>
__device__ __forceinline__ float slope(const Factors& f, float s) {
  float d = s - f.m;
  if constexpr (INF) d = s == f.m ? 0.f : d;
  float lp = d - f.logz;
  const float p = exp_below(lp);
  return p * fmaf(f.h, lp + f.entropy, f.c);
}

// tx threads share a row's part: y counts parts of tx V U columns.
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_bwd_kernel(LogpArgs a, int tx) {
  constexpr int V = kVec<T>, U = 4;
  const int lane = threadIdx.x & (tx - 1), rpb = kThreads / tx;
  __shared__ float sums[kThreads / 4];
  for (int64_t n0 = (int64_t)blockIdx.x * rpb; n0 < a.N; n0 += (int64_t)gridDim.x * rpb) {
    const int64_t n = n0 + threadIdx.x / tx;
    const bool there = n < a.N;
    const int64_t r = there ? n : a.N - 1;
    const T* row = static_cast<const T*>(a.scores) + r * a.lds;
    T* out = static_cast<T*>(a.dscores) + r * a.V;
    const int first = (int)blockIdx.y * tx * V * U;
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int c = first + (j * tx + lane) * V;
      u[j] = fetch16<SHORT>(row + (c < a.V ? c : 0), c < a.V ? a.V - c : a.V);
    }
    float dtop = 0.f;
    if (a.dtop) {
      if (lane == 0)
        for (int i = 0; i < a.k; ++i)
          if (a.top_index[r * a.k + i] >= 0) dtop += a.dtop[r * a.k + i];
      if (lane == 0) sums[threadIdx.x / tx] = dtop;
      __syncthreads();
      dtop = sums[threadIdx.x / tx];
    }
    const Factors f = factors_of(a, r, dtop);
    const int64_t t = a.dchosen ? token_at(a, r) : -1;
    const float dc = t >= 0 ? a.dchosen[r] : 0.f;
    if (there) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = first + (j * tx + lane) * V;
        if (c >= a.V) break;
        float v[V];
        unpack16<T>(keep16<SHORT, T>(u[j], a.V - c, a.V), v);
        const int at = t >= c && t < c + V ? (int)(t - c) : -1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = v[i];
          v[i] = f.m == INFINITY ? slope<true>(f, s) : slope<false>(f, s);
          if (at == i && s > -INFINITY) v[i] += dc;
        }
        store_row(out + c, a.V - c, v);
      }
    }
    if (a.dtop) {
      // The alternatives' columns again, with what they get: after the row's part is written.
      __syncthreads();
      if (there) {
        for (int i = lane; i < a.k; i += tx) {
          const int32_t c = a.top_index[r * a.k + i];
          if (c < first || c >= first + tx * V * U) continue;
          const float s = to_f32(row[c]);
          float g = f.m == INFINITY ? slope<true>(f, s) : slope<false>(f, s);
          if (c == t) g += dc;
          out[c] = (T)(g + a.dtop[r * a.k + i]);
        }
      }
      __syncthreads();
    }
  }
}

// --- launches ---------------------------------------------------------------------

template <typename T, int G, bool SHORT>
void rows_grouped(const LogpArgs& a, hipStream_t s) {
  const int64_t need = (a.N + kThreads / G - 1) / (kThreads / G);
  logp_rows_kernel<T, G, SHORT><<<(unsigned)(need < kMaxBlocks ? need : kMaxBlocks), kThreads, 0, s>>>(a);
}

template <typename T>
void logp_typed(const LogpArgs& a, hipStream_t s) {
  if (a.k == 0 && a.V <= 2048) {
    if (a.V < kVec<T>) rows_grouped<T, 4, true>(a, s);
    else if (a.V <= 128) rows_grouped<T, 4, false>(a, s);
    else if (a.V <= 512) rows_grouped<T, 16, false>(a, s);
    else rows_grouped<T, 64, false>(a, s);
    return;
  }
  const dim3 grid((unsigned)a.splits, (unsigned)(a.N < 65535 ? a.N : 65535));
  if (a.k == 0) logp_part_kernel<T, false, false><<<grid, kThreads, 0, s>>>(a);      // (V > 2048)
  else if (a.V < kVec<T>) logp_part_kernel<T, true, true><<<grid, kThreads, 0, s>>>(a);
  else logp_part_kernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
  if (a.splits > 1) logp_join_kernel<T><<<(unsigned)(a.N < kMaxBlocks ? a.N : kMaxBlocks), kThreads, 0, s>>>(a);
}

template <typename T>
void logp_bwd_typed(const LogpArgs& a, hipStream_t s) {
  constexpr int V = kVec<T>;
  const int nvec = (a.V + V * 4 - 1) / (V * 4);
  int tx = 4;
  while (tx < nvec && tx < kThreads) tx *= 2;
  const int64_t need = (a.N + kThreads / tx - 1) / (kThreads / tx);
  const int64_t parts = (a.V + (int64_t)tx * V * 4 - 1) / ((int64_t)tx * V * 4);
  const dim3 grid((unsigned)(need < kMaxBlocks ? need : kMaxBlocks), (unsigned)parts);
  if (a.V < V) logp_bwd_kernel<T, true><<<grid, kThreads, 0, s>>>(a, tx);
  else logp_bwd_kernel<T, false><<<grid, kThreads, 0, s>>>(a, tx);
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

// Parts of a row: none with enough rows for the card, else parts of 4096 scores or more.
int logp_splits(int64_t N, int V, int k) {
  if (k == 0 && V <= 2048) return 1;
  int64_t parts = (1024 + N - 1) / (N > 0 ? N : 1);
  const int64_t most = (V + 4095) / 4096;
  if (parts > most) parts = most;
  return (int)(parts < 1 ? 1 : (parts < kMaxSplits ? parts : kMaxSplits));
}

int64_t logp_workspace_bytes(int64_t N, int V, int k) {
  const int64_t splits = logp_splits(N, V, k);
  return splits > 1 ? logp_top_offset(N, (int)splits) + align256(N * splits * k * 8) : 0;
}

int64_t logp_top_offset(int64_t N, int splits) { return align256(N * splits * 12); }

void launch_logp(const LogpArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) logp_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) logp_typed<__bf16>(a, s);
  else logp_typed<_Float16>(a, s);
}

void launch_logp_bwd(const LogpArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) logp_bwd_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) logp_bwd_typed<__bf16>(a, s);
  else logp_bwd_typed<_Float16>(a, s);
}

}  // namespace gx::layer
