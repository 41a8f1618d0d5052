// Log probabilities of given tokens under rows of scores, the rows' entropies, the best
// alternatives, and the gradient of all three.
//
// A row's candidates are its scores that are neither -inf nor NaN.  With m the largest,
// d = s - m, Z = Σ e^d and U = Σ e^d d over the candidates:
//   log p_t = d_t - log Z,   H = -Σ p log p = log Z - U / Z
// Both terms of H are non-negative then.  Sums beside a reference below m (see Lean) make log Z and -U / Z larger and
// smaller by what it lacks, at most 2.1: of rows with p near 1, log p and H, near 0, are good to some 1e-7, not to
// digits of their own (64 to 40000 normal scores and one with p = 0.98 or 0.9996: 3e-7 to 8e-7 at most).
// Of several +inf each has p = 1 / their number.  The gradient from g (chosen), h (entropy) and q (alternatives) is
//   ds_j = g [j = t] + Σ_i q_i [j = top_i] - p_j (g + Σ_i q_i + h (log p_j + H)).
//
// One pass over the scores: a thread keeps its own sums beside a reference, at first the largest of the first scores of
// its wave (or group of lanes), brought to a larger one where scores pass it by much (once a 16-byte vector at most), and
// the threads' are merged at the end, in a fixed order.  Rows are cut into parts where there are too few for the card,
// and joined by a second kernel.
//
// 8192 x 65536 bf16: 185 us call after call (1074 MB, 5.8 TB/s, some of it from caches), 228 behind a gradient whose writes
// are still in the caches, and the gradient 396 us (2147 MB, 5.4 TB/s): bytes.  100003 x 500 fp32: 44 and 73 us.  One row
// of 65536 with 5 alternatives 8.5 + 4.5 us: the chains of a part and of the join; 130 rows of 32001 with 20, 15 + 5
// us, 21 + 5 with rows of the type's lowest value alone, which are read twice.
//
// Alternatives are found in the same pass.  A score's rank is a 64-bit number, its value
// above its complemented index, so no two are equal and ties go to the lower index.  The
// first scores give a bound that k of them reach; scores that reach the bound go to a list in LDS,
// which is cut back to its k largest where it would overflow (its k-th by bisection over the
// rank's bits), which raises the bound.  The list's order depends on the waves', what is kept of it
// does not.

#include <float.h>
#include <math.h>

#include <algorithm>

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

// Scores taken in by one thread, as the slow form: the largest (`ref`), Σ e^(s - m), Σ e^(s - m) (s - m).  -inf: none yet.  A largest
// of +inf leaves sums that do not count (see resolve).
struct Plain {
  float ref = -INFINITY, z = 0.f, u = 0.f;
  __device__ __forceinline__ void raise(float to) {      // to >= ref
    const float by = ref - to;
    if (by == 0.f || ref == to) return;
    const float f = ref == -INFINITY ? 0.f : __expf(fmaxf(by, -110.f));
    u = f == 0.f ? 0.f : f * fmaf(z, by, u);
    z *= f;
    ref = to;
  }
  // (no s is +inf)
  template <int V>
  __device__ __forceinline__ void add(const float (&s)[V]) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, s[i]);
    if (top > ref) raise(top);
    float zv = 0.f, uv = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float d = s[i] - ref;
      const float e = exp_below(d);
      zv += e;
      uv = fmaf(e, d, uv);
    }
    z += zv;
    u += uv;
  }
};

// The same in half the instructions: sums of 2^l and 2^l l with l = s L - ref, L = log2(e) in fp32, where ref
// need not be the largest s L, only near it.  Where a vector's sum passes the number of its scores, which one of 3.02
// (fp32: 2.02) above ref does, and none without one above it, ref is raised to its largest, rounded: the largest
// score's own l is what the rounding left, at most 1/2 where |ref| < kNear, and 64 where |s| < kFar: 2^22 sums of 2^64
// still fit.  Below -kFar scores that differ do so by 64 at least, so what is no larger weighs nothing beside other
// scores and is left out.  A row whose ref ends past kNear, or that holds only scores left out, is taken in as Plain
// (see slowly).
constexpr float kNear = 0x1p24f, kFar = 0x1p30f;
struct Lean {
  float ref = -INFINITY, z = 0.f, u = 0.f;
  __device__ __forceinline__ void raise(float to) {
    const float by = ref - to;
    if (ref == to) return;
    const float f = ref == -INFINITY ? 0.f : fast_exp2(fmaxf(by, -160.f));
    u = f == 0.f ? 0.f : f * fmaf(z, by, u);
    z *= f;
    ref = to;
  }
  // `top`: the largest of some of the scores to come.
  __device__ __forceinline__ void begin(float top) {
    if (top > -kFar) ref = top < kFar ? top * kLog2e : INFINITY;
  }
  template <int V>
  __device__ __forceinline__ void sums(const float (&s)[V], float& zv, float& uv) const {
    zv = uv = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float l = fmaxf(fmaf(s[i], kLog2e, -ref), -160.f);      // (-inf and NaN too: 2^l is 0)
      const float e = fast_exp2(l);
      zv += e;
      uv = fmaf(e, l, uv);
    }
  }
  template <int V>
  __device__ __forceinline__ void add(const float (&s)[V]) {
    float zv, uv;
    sums(s, zv, uv);
    if (!(zv <= 1.01f * V)) {                         // (1.01: what ref's rounding leaves of equal scores)
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, s[i]);
      if (top <= -kFar) {                              // (beside any other score they weigh nothing)
        if (ref == -INFINITY && top > -INFINITY) z = 1.f;
        return;
      }
      raise(top < kFar ? fmaxf(ref, top * kLog2e) : INFINITY);
      sums(s, zv, uv);
    }
    z += zv;
    u += uv;
  }
};

template <typename S>
__device__ __forceinline__ S merge(S a, S b) {
  const float to = fmaxf(a.ref, b.ref);
  a.raise(to);
  b.raise(to);
  a.z += b.z;
  a.u += b.u;
  return a;
}

// What G lanes took in, in all of them.
template <int G, typename S>
__device__ __forceinline__ S lanes_merge(S s) {
  const float to = lanes_reduce<G>(s.ref, [](float a, float b) { return fmaxf(a, b); });
  s.raise(to);
  s.z = lanes_sum<G>(s.z);
  s.u = lanes_sum<G>(s.u);
  return s;
}

// ... what a workgroup did; `red` takes three floats a wave.
template <typename S>
__device__ __forceinline__ S block_merge(S s, float (*red)[3]) {
  s = lanes_merge<64>(s);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = s.ref;
    red[threadIdx.x >> 6][1] = s.z;
    red[threadIdx.x >> 6][2] = s.u;
  }
  __syncthreads();
  S r;
  r.ref = red[0][0], r.z = red[0][1], r.u = red[0][2];
  for (int w = 1; w < (int)blockDim.x / 64; ++w) {
    S o;
    o.ref = red[w][0], o.z = red[w][1], o.u = red[w][2];
    r = merge(r, o);
  }
  return r;
}

__device__ __forceinline__ int64_t token_at(const LogpArgs& a, int64_t n) {
  const int64_t t = a.index64 ? static_cast<const int64_t*>(a.index)[n] : static_cast<const int32_t*>(a.index)[n];
  return (uint64_t)t < (uint64_t)a.V ? t : -1;
}

// log p of a score v: m and log Z need not be the largest score's, only belong together.
__device__ __forceinline__ float log_p(float v, float m, float logz) {
  return v > -INFINITY ? fminf(v == m ? -logz : (v - m) - logz, 0.f) : -INFINITY;
}

struct Row { float m, logz, entropy; };

__device__ __forceinline__ Row resolved(Plain s) {
  if (!(s.ref > -INFINITY)) return Row{-INFINITY, 0.f, 0.f};
  const float logz = logf(s.z);
  return Row{s.ref, logz, fmaxf(logz - s.u / s.z, 0.f)};
}
// 2^ref = e^M exactly with M = ref / L: m is M in fp32, and what that rounds off goes to log Z.
__device__ __forceinline__ Row resolved(Lean s) {
  const double exact = (double)s.ref / (double)kLog2e;
  const float m = (float)exact, lz = logf(s.z);
  return Row{m, lz + (float)(exact - (double)m), fmaxf(lz - s.u / (s.z * kLog2e), 0.f)};
}

// Scores lo .. hi - 1 of a row (lo in whole vectors) by G lanes, or the workgroup's threads (G = kThreads), as Plain; of
// +inf each weighs 1.
template <typename T, int G, bool SHORT>
__device__ __forceinline__ Plain take_slowly(const LogpArgs& a, int64_t n, int lo, int hi, int lane, float (*red)[3]) {
  constexpr int V = kVec<T>, U = 8;    // vectors in flight
  const T* row = static_cast<const T*>(a.scores) + n * a.lds;
  Plain s;
  float infinite = 0.f;
  for (int c0 = lo + lane * V; c0 < hi; c0 += G * V * U) {
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int c = c0 + j * G * V;
      u[j] = fetch16<SHORT>(row + (c < hi ? c : 0), c < hi ? a.V - c : a.V);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int c = c0 + j * G * V;
      if (c >= hi) break;
      float v[V];
      unpack16<T>(keep16<SHORT, T>(u[j], a.V - c, a.V), v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool inf = c + i < hi && v[i] == INFINITY;
        infinite += inf ? 1.f : 0.f;
        v[i] = c + i < hi && !inf ? v[i] : -INFINITY;
      }
      s.add(v);
    }
  }
  if constexpr (G <= 64) {
    s = lanes_merge<G>(s);
    infinite = lanes_sum<G>(infinite);
  } else {
    __syncthreads();
    s = block_merge(s, red);
    infinite = lanes_sum<64>(infinite);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = infinite;
    __syncthreads();
    infinite = 0.f;
    for (int w = 0; w < kThreads / 64; ++w) infinite += red[w][0];
  }
  if (infinite > 0.f) {
    s = Plain();
    s.ref = INFINITY;
    s.z = infinite;
  }
  return s;
}
__device__ __forceinline__ bool only_low(Lean s) { return s.ref == -INFINITY && s.z > 0.f; }
__device__ __forceinline__ bool slowly(Lean s) {
  return s.ref == -INFINITY ? s.z > 0.f : !(fabsf(s.ref) < kNear);
}

template <typename T, int G, bool SHORT>
__device__ __forceinline__ Row resolve(const LogpArgs& a, int64_t n, int lane, float (*red)[3], Lean s) {
  if (slowly(s)) return resolved(take_slowly<T, G, SHORT>(a, n, 0, a.V, lane, red));
  return s.ref == -INFINITY ? Row{-INFINITY, 0.f, 0.f} : resolved(s);
}

// Writes a row's results, by one thread.
template <typename T>
__device__ __forceinline__ void finish(const LogpArgs& a, int64_t n, Row r) {
  const int64_t t = token_at(a, n);
  a.chosen[n] = t < 0 ? 0.f : log_p(to_f32(static_cast<const T*>(a.scores)[n * a.lds + t]), r.m, r.logz);
  a.entropy[n] = r.entropy;
  if (a.stats) {
    a.stats[n * 3] = r.m;
    a.stats[n * 3 + 1] = r.logz;
    a.stats[n * 3 + 2] = r.entropy;
  }
}

// --- no alternatives ------------------------------------------------------------

// G lanes share a row.
template <typename T, int G, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_rows_kernel(LogpArgs a) {
  constexpr int V = kVec<T>, U = 4, R = kThreads / G;
  const int lane = threadIdx.x % G;
  for (int64_t n = (int64_t)blockIdx.x * R + threadIdx.x / G; n < a.N; n += (int64_t)gridDim.x * R) {
    const T* row = static_cast<const T*>(a.scores) + n * a.lds;
    Lean s;
#pragma unroll 1                       // (a first pass peeled off takes registers: 65536 x 4096 bf16 107 us, not 93)
    for (int base = 0; base < a.V; base += G * V * U) {
      const int c0 = base + lane * V;
      uint4 u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = c0 + j * G * V;
        u[j] = fetch16<SHORT>(row + (c < a.V ? c : 0), c < a.V ? a.V - c : a.V);
      }
      if constexpr (!SHORT)          // (what fetch16 gives are scores of the row, in place or not)
        if (base == 0) {
          // all lanes begin at the largest of their first scores, which few later ones pass by much
          float v[V], top = -INFINITY;
          unpack16<T>(u[0], v);
#pragma unroll
          for (int i = 0; i < V; ++i) top = fmaxf(top, v[i]);
          s.begin(lanes_reduce<G>(top, [](float p, float q) { return fmaxf(p, q); }));
        }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = c0 + j * G * V;
        if (c >= a.V) break;
        float v[V];
        unpack16<T>(keep16<SHORT, T>(u[j], a.V - c, a.V), v);
        if (c + V > a.V) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = c + i < a.V ? v[i] : -INFINITY;
        }
        s.add(v);
      }
    }
    const Row r = resolve<T, G, SHORT>(a, n, lane, nullptr, lanes_merge<G>(s));
    if (lane == 0) finish<T>(a, n, r);
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

// Short rows: G lanes hold one, NV vectors of its scores each, as integers in their order (vector i of lane l holds the
// scores from (i G + l) V on).  Each alternative is the largest left, then the lowest index that has it; where a wave
// has few rows, a round passes over the vectors in which no row has its own.  33000 x 500 fp32 with 10 alternatives 45
// us, 160000 x 100 with 5 34 us, 8000 x 2000 bf16 with 20 44 us; a workgroup for each row took 308, 1213 and 90.
// Few rows with many alternatives wait for the rounds (4 x 2000, 20: 17 us) and take a workgroup each (9.6).
constexpr int kShort = 2048;
bool short_rows(int64_t N, int V, int k) { return V <= kShort && (V <= 256 || N > 512 || k <= 6); }
template <int G, typename F>
__device__ __forceinline__ uint32_t lanes_reduce_key(uint32_t v, F&& op) {
  return __float_as_uint(lanes_reduce<G>(__uint_as_float(v), [&](float a, float b) {
    return __uint_as_float(op(__float_as_uint(a), __float_as_uint(b)));
  }));
}
template <typename T, int G, int NV, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_rows_top_kernel(LogpArgs a) {
  constexpr int V = kVec<T>, R = kThreads / G;
  constexpr bool kSkip = G >= 16;
  const auto larger = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
  const auto smaller = [](uint32_t p, uint32_t q) { return p < q ? p : q; };
  const int lane = threadIdx.x % G;
  for (int64_t n0 = (int64_t)blockIdx.x * R; n0 < a.N; n0 += (int64_t)gridDim.x * R) {   // (groups exchange together)
    const bool there = n0 + threadIdx.x / G < a.N;
    const int64_t n = there ? n0 + threadIdx.x / G : a.N - 1;
    const T* row = static_cast<const T*>(a.scores) + n * a.lds;
    uint4 u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      u[i] = fetch16<SHORT>(row + (c < a.V ? c : 0), c < a.V ? a.V - c : a.V);
    }
    uint32_t v[NV][V], top[NV], best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + lane) * V;
      float s[V];
      unpack16<T>(keep16<SHORT, T>(u[i], a.V - c, a.V), s);
      top[i] = 0;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        v[i][q] = c + q < a.V ? key_of(s[q]) : 0;
        top[i] = larger(top[i], v[i][q]);
      }
      best = larger(best, top[i]);
    }
    best = lanes_reduce_key<G>(best, larger);
    const float m = best ? value_of(best) : -INFINITY;
    Plain sums;
    sums.ref = m;
    if (fabsf(m) < INFINITY) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int q = 0; q < V; ++q) {
          float d = value_of(v[i][q]) - m;              // (no candidate: NaN)
          const float e = exp_below(d);
          sums.z += e;
          sums.u = fmaf(e, d, sums.u);
        }
    } else {                                            // of +inf each weighs 1
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int q = 0; q < V; ++q) sums.z += v[i][q] == best ? 1.f : 0.f;
    }
    sums.z = lanes_sum<G>(sums.z);
    sums.u = lanes_sum<G>(sums.u);
    const Row r = resolved(sums);
    if (lane == 0 && there) finish<T>(a, n, r);
    float value = 0.f;                                  // the alternative that this lane writes
    int32_t index = 0;
    int mine = 0;                                       // the last one, as this lane's score 0 would be 0
    for (int j = 0; j < a.k; ++j) {
      if (j > 0) {
        best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!kSkip || __any((unsigned)(mine - i * G * V) < (unsigned)V)) {
            top[i] = 0;
#pragma unroll
            for (int q = 0; q < V; ++q) {
              v[i][q] = mine == i * G * V + q ? 0 : v[i][q];
              top[i] = larger(top[i], v[i][q]);
            }
          }
          best = larger(best, top[i]);
        }
        best = lanes_reduce_key<G>(best, larger);
      }
      uint32_t at = 0x7fffffff;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (!kSkip || __any(top[i] == best)) {
#pragma unroll
          for (int q = V - 1; q >= 0; --q) at = v[i][q] == best ? i * G * V + q : at;
        }
      at = lanes_reduce_key<G>(at == 0x7fffffff ? at : at + lane * V, smaller);
      mine = (int)at - lane * V;
      if (lane == j % G) {
        value = best ? log_p(value_of(best), r.m, r.logz) : -INFINITY;
        index = best ? (int32_t)at : -1;
      }
      if ((j % G == G - 1 || j == a.k - 1) && lane <= j % G && there) {
        a.top[n * a.k + j - j % G + lane] = value;
        a.top_index[n * a.k + j - j % G + lane] = index;
      }
    }
  }
}

constexpr int kTile = 4096;            // scores of a workgroup at a time
constexpr int kListSize = 1024;

// Keeps the k largest of list[0 .. count - 1] (count > k) in list[0 .. k - 1], in some order; returns the least of
// them.  Their bits are found from the highest in which the list's ranks differ: the largest number that at least k of
// them reach.
template <int SIZE>
__device__ __forceinline__ uint64_t cut(uint64_t* list, int count, int k, int* scratch) {
  constexpr int PER = (SIZE + kThreads - 1) / kThreads, W = kThreads / 64;
  uint64_t mine[PER], differ = 0;
  const uint64_t first = list[0];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * kThreads + threadIdx.x;
    mine[i] = at < count ? list[at] : 0;
    differ |= at < count ? mine[i] ^ first : 0;
  }
  int high = 63;                       // the highest bit that differs somewhere
  {
    uint32_t hi = (uint32_t)(differ >> 32), lo = (uint32_t)differ;
#pragma unroll
    for (int off = 32; off; off /= 2) hi |= __shfl_xor(hi, off), lo |= __shfl_xor(lo, off);
    if ((threadIdx.x & 63) == 0)
      scratch[threadIdx.x >> 6] = hi ? 63 - __clz((int)hi) : (lo ? 31 - __clz((int)lo) : 0);
    __syncthreads();
    high = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) high = max(high, scratch[w]);
  }
  uint64_t bound = high < 63 ? first >> (high + 1) << (high + 1) : 0;
  int turn = 1;
  for (int b = high; b >= 0; --b) {
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
#pragma unroll 8
  for (int i = 0; i < k; ++i) least = list[i] < least ? list[i] : least;
  __syncthreads();
  return least;
}

// The k largest of the list in descending order to out[0 .. k - 1], zeros where there are fewer.  The list has room for
// kAhead more.
constexpr int kAhead = 16;
template <int SIZE>
__device__ __forceinline__ void sorted(uint64_t* list, int count, int k, int* scratch, uint64_t* out) {
  if (count > kThreads && count > k) {
    cut<SIZE>(list, count, k, scratch);
    count = k;
  }
  if (threadIdx.x < kAhead) list[count + threadIdx.x] = 0;
  __syncthreads();
  if ((int)threadIdx.x < count) {
    const uint64_t mine = list[threadIdx.x];
    int above = 0;
    for (int i = 0; i < count; i += kAhead)
#pragma unroll
      for (int q = 0; q < kAhead; ++q) above += list[i + q] > mine;
    if (above < k) out[above] = mine;
  }
  if ((int)threadIdx.x >= count && (int)threadIdx.x < k) out[threadIdx.x] = 0;
  __syncthreads();
}

// Writes a row's alternatives from their sorted ranks.
__device__ __forceinline__ void write_top(const LogpArgs& a, int64_t n, const uint64_t* top, Row row) {
  if ((int)threadIdx.x < a.k) {
    const uint64_t r = top[threadIdx.x];
    const float v = value_of((uint32_t)(r >> 32));
    a.top[n * a.k + threadIdx.x] = r ? log_p(v, row.m, row.logz) : -INFINITY;
    a.top_index[n * a.k + threadIdx.x] = r ? (int32_t)~(uint32_t)r : -1;
  }
}

// The k-th largest of the threads' ranks, or a number that is no larger and that k of them reach: its bits from the
// highest, by every wave for itself.
__device__ __forceinline__ uint64_t reached(uint64_t mine, int k, uint64_t* ranks) {
  constexpr int PER = kThreads / 64;
  ranks[threadIdx.x] = mine;
  __syncthreads();
  uint64_t rank[PER], bound = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) rank[i] = ranks[i * 64 + (threadIdx.x & 63)];
  for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
    const uint64_t test = bound | bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += __popcll(__ballot(rank[i] >= test));
    if (n >= k) bound = test;
    if (n == k) break;
  }
  return bound;
}

// The scores of a row's part from c on, c + V G ..., U vectors of a thread.
template <typename T, int U>
struct Vectors {
  static constexpr int V = kVec<T>;
  uint4 u[U];
  // (a whole tile, as most are, takes no thought of the row's end: 9.3 instructions a score where it took 12.5)
  static __device__ __forceinline__ bool whole(int base, int last) { return base + kThreads * V * U <= last; }
  __device__ __forceinline__ void fetch(const T* row, int base, int last, int length) {
    if (whole(base, last)) {
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = ld16_any(row + base + (j * kThreads + threadIdx.x) * V);
      return;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int c = base + (j * kThreads + (int)threadIdx.x) * V;
      u[j] = fetch16<false>(row + (c < last ? c : 0), c < last ? length - c : length);
    }
  }
  // -inf past the part.
  __device__ __forceinline__ void unpack(int j, int base, int last, int length, float (&v)[V]) const {
    if (whole(base, last)) return unpack16<T>(u[j], v);
    const int c = base + (j * kThreads + (int)threadIdx.x) * V;
    unpack16<T>(keep16<false, T>(u[j], c < last ? length - c : length, length), v);
    if (c + V > last) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = c + i < last ? v[i] : -INFINITY;
    }
  }
};

// A part of a row (x) of each row (y), with k alternatives (or none); one part: the row's results.  The next
// scores are in flight while those at hand are taken in.  (Four waves a SIMD: the slow form's code would take registers
// for two.)
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads, 4) void logp_part_kernel(LogpArgs a) {
  constexpr int V = kVec<T>, U = kTile / kThreads / V;
  __shared__ __align__(16) uint64_t list[TOP ? kListSize + kAhead : 1];
  __shared__ uint64_t out[kLogpMaxK];
  __shared__ float red[kThreads / 64][3];
  __shared__ uint64_t ranks[TOP ? kThreads : 1];
  __shared__ int scratch[2 * kThreads / 64], count;
  const int split = blockIdx.x;
  for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
    const T* row = static_cast<const T*>(a.scores) + n * a.lds;
    const int per = (int)((((int64_t)a.V + a.splits - 1) / a.splits + V - 1) / V * V);
    const int first = (int64_t)split * per < a.V ? split * per : a.V;
    const int last = first + (int64_t)per < a.V ? first + per : a.V;
    Lean s;
    uint64_t bound = 1;               // (0: no candidate)
    if (threadIdx.x == 0) count = 0;
    Vectors<T, U> next;
    next.fetch(row, first, last, a.V);
#pragma unroll 1
    for (int base = first; base < last; base += kTile) {
      const Vectors<T, U> now = next;
      if (base + kTile < last) next.fetch(row, base + kTile, last, a.V);
      float v[U][V], most = -INFINITY;        // (also where all of a thread's are NaN)
#pragma unroll
      for (int j = 0; j < U; ++j) now.unpack(j, base, last, a.V, v[j]);
      if (TOP || base == first) {
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) most = fmaxf(most, v[j][i]);
      }
      // (a wave begins at the largest of its first scores, which few later ones pass by much)
      if (base == first) s.begin(lanes_reduce<64>(most, [](float p, float q) { return fmaxf(p, q); }));
#pragma unroll
      for (int j = 0; j < U; ++j) s.add(v[j]);
      if constexpr (TOP) {
        if (base == first) {
          int at = 0;                  // the first place of a thread's largest
#pragma unroll
          for (int j = U - 1; j >= 0; --j)
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
              at = v[j][i] == most ? base + (j * kThreads + (int)threadIdx.x) * V + i : at;
          const uint32_t key = key_of(most);
          bound = max(bound, reached(key ? rank_of(key, at) : 0, a.k, ranks));
        }
        // Each thread's scores that reach the bound, as bits; what the list has no room for waits until the list is
        // cut and the bound is higher.
        const auto reach = [&](int j, int i) {
          const int c = base + (j * kThreads + (int)threadIdx.x) * V;
          return rank_of(key_of(v[j][i]), c + i);
        };
        const float least = (bound >> 32) != 0 ? value_of((uint32_t)(bound >> 32)) : -FLT_MAX;
        uint32_t waiting = 0;
        if (most >= least) {
#pragma unroll
          for (int j = 0; j < U; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) waiting |= v[j][i] >= least ? 1u << (j * V + i) : 0;
        }
        for (;;) {
          if ((uint32_t)bound > 1 && __any(waiting)) {   // (a bound with an index: equal scores after it do not reach it)
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
              for (int i = 0; i < V; ++i)
                if (reach(j, i) < bound) waiting &= ~(1u << (j * V + i));
          }
          // places in the list: a wave's share of it, in which a lane's scores follow those of the lanes before it
          if (__any(waiting)) {
            const int mine = __popc(waiting), before = lanes_scan(mine, [](int p, int q) { return p + q; });
            const int all = __builtin_amdgcn_readlane(before, 63);
            int at = 0;
            if ((threadIdx.x & 63) == 0) at = atomicAdd(&count, all);
            at = __builtin_amdgcn_readfirstlane(at) + before - mine;
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
              for (int i = 0; i < V; ++i)
                if (waiting >> (j * V + i) & 1) {
                  if (at < kListSize) {
                    list[at] = reach(j, i);
                    waiting &= ~(1u << (j * V + i));
                  }
                  ++at;
                }
          }
          __syncthreads();
          const int have = count;
          __syncthreads();
          if (have <= kListSize) break;
          bound = cut<kListSize>(list, kListSize, a.k, scratch);
          if (threadIdx.x == 0) count = a.k;
          __syncthreads();
        }
      }
    }
    s = block_merge(s, red);
    if constexpr (TOP) sorted<kListSize>(list, count, a.k, scratch, out);
    if (a.splits > 1) {
      const int64_t at = n * a.splits + split;
      // (a part of low scores alone, as a fully masked row has them, is left as Plain, marked by a negative sum)
      if (only_low(s)) {
        const Plain low = take_slowly<T, kThreads, false>(a, n, first, last, threadIdx.x, red);
        s.ref = low.ref, s.z = -low.z, s.u = low.u;
      }
      if (threadIdx.x == 0) a.part[at * 3] = s.ref, a.part[at * 3 + 1] = s.z, a.part[at * 3 + 2] = s.u;
      if (TOP && (int)threadIdx.x < a.k) a.part_top[at * a.k + threadIdx.x] = out[threadIdx.x];
    } else {
      const Row r = resolve<T, kThreads, false>(a, n, threadIdx.x, red, s);
      if (threadIdx.x == 0) finish<T>(a, n, r);
      if constexpr (TOP) write_top(a, n, out, r);
    }
    __syncthreads();
  }
}

// The parts of a row.
constexpr int kMaxSplits = 64;
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_join_kernel(LogpArgs a) {
  __shared__ __align__(16) uint64_t list[TOP ? kMaxSplits * kLogpMaxK + kAhead : 1];
  __shared__ uint64_t out[kLogpMaxK];
  __shared__ float red[kThreads / 64][3];
  __shared__ int scratch[2 * kThreads / 64], count;
  __shared__ uint64_t lowest;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    Lean s;
    Plain low;
    const uint64_t* p = a.part_top + n * a.splits * a.k;
    uint64_t bound = 1;
    if ((int)threadIdx.x < a.splits) {
      const float* q = a.part + (n * a.splits + threadIdx.x) * 3;
      s.ref = q[0], s.z = q[1], s.u = q[2];
      if (s.z < 0.f) {
        low.ref = s.ref, low.z = -s.z, low.u = s.u;
        s = Lean();
        s.z = 1.f;
      }
      // every part's list is sorted: no score below a part's last is among the row's k best
      if (TOP) bound = max(bound, p[threadIdx.x * a.k + a.k - 1]);
    }
    const int all = a.splits * a.k;
    constexpr int PER = 4;             // of them in flight before the bound is known
    uint64_t mine[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = i * kThreads + threadIdx.x;
      mine[i] = at < all ? p[at] : 0;
    }
    if constexpr (TOP) {                         // (the parts are the first wave's)
#pragma unroll
      for (int off = 32; off; off /= 2) {
        const uint64_t o = (uint64_t)__shfl_xor((int)(bound >> 32), off) << 32 | (uint32_t)__shfl_xor((int)bound, off);
        bound = max(bound, o);
      }
      if (threadIdx.x == 0) lowest = bound, count = 0;
    }
    s = block_merge(s, red);
    Row r;
    if (only_low(s)) {
      __syncthreads();
      r = resolved(block_merge(low, red));
    } else {
      r = resolve<T, kThreads, false>(a, n, threadIdx.x, red, s);
    }
    if constexpr (TOP) {
      bound = lowest;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (mine[i] >= bound) list[atomicAdd(&count, 1)] = mine[i];
      for (int at = PER * kThreads + threadIdx.x; at < all; at += kThreads) {
        const uint64_t o = p[at];
        if (o >= bound) list[atomicAdd(&count, 1)] = o;
      }
    }
    if (threadIdx.x == 0) finish<T>(a, n, r);
    __syncthreads();
    if constexpr (TOP) {
      sorted<kMaxSplits * kLogpMaxK>(list, count, a.k, scratch, out);
      write_top(a, n, out, r);
    }
    __syncthreads();
  }
}

// --- gradient ---------------------------------------------------------------------

// What a row's gradient is made of: ds = p (c + h (log p + H)) before what the chosen get.
struct Factors {
  float m, logz, entropy, c, h;
};

// (dtop: the sum over the alternatives that exist)
__device__ __forceinline__ Factors factors_of(const LogpArgs& a, int64_t n, float dtop) {
  Factors f;
  f.m = a.stats[n * 3], f.logz = a.stats[n * 3 + 1], f.entropy = a.stats[n * 3 + 2];
  f.c = -(a.dchosen && token_at(a, n) >= 0 ? a.dchosen[n] : 0.f) - dtop;
  f.h = a.dentropy ? -a.dentropy[n] : 0.f;
  return f;
}

// The gradient of score s, of any row.
__device__ __forceinline__ float slope(const Factors& f, float s) {
  const float d = s == f.m ? 0.f : s - f.m;
  float lp = d - f.logz;
  const float p = exp_below(lp);
  return s > -INFINITY ? p * fmaf(f.h, lp + f.entropy, f.c) : 0.f;
}

// The same in fewer instructions, where |m| < kNear and the row's gradients are finite: with l = s L - k, L = log2(e) in
// fp32 and k = m L + log2 Z rounded to fp32, p = 2^(l - off) by what k's rounding left, off (at most 2 there), and so
// ds = 2^l (c' + h' l).
struct Quick {
  float k, c, h;
  __device__ __forceinline__ explicit Quick(const Factors& f) {
#pragma clang fp contract(off)      // (what roundings leave is taken from rounded values)
    const float m = f.m > -INFINITY ? f.m : 0.f;                // (an empty row: every 2^l is 0)
    const float a = m * kLog2e, b = f.logz * kLog2e;
    k = a + b;
    const float bb = k - a;                                     // (a + b = k + ((a - (k - bb)) + (b - bb)) exactly)
    const float off = fmaf(m, kLog2e, -a) + fmaf(f.logz, kLog2e, -b) + f.logz * 1.925963033500e-8f +
                      ((a - (k - bb)) + (b - bb));              // (log2(e) = kLog2e + 1.926e-8)
    const float back = fast_exp2(-off);
    c = fmaf(f.h, f.entropy - off * kLn2, f.c) * back;
    h = f.h * kLn2 * back;
  }
  // (what is no candidate is multiplied by 2^-160, which is 0, and has no other look at it)
  __device__ __forceinline__ bool finite() const { return fmaf(fabsf(h), 160.f, fabsf(c)) < INFINITY; }
  __device__ __forceinline__ float slope(float s) const {
    const float l = fmaxf(fmaf(s, kLog2e, -k), -160.f);
    return fast_exp2(l) * fmaf(h, l, c);
  }
};

// WHOLE: a workgroup takes `tiles` times kThreads V U columns of a row (y counts such parts), the next scores in flight.
// Otherwise tx threads share a row of at most tx V U columns.
template <typename T, bool WHOLE, bool SHORT>
__global__ __launch_bounds__(kThreads) void logp_bwd_kernel(LogpArgs a, int tx_, int tiles) {
  constexpr int V = kVec<T>, U = WHOLE ? 2 : 4;
  const int tx = WHOLE ? kThreads : tx_;
  const int lane = threadIdx.x & (tx - 1), rpb = kThreads / tx;
  __shared__ float sums[kThreads / 4];
  for (int64_t n0 = (int64_t)blockIdx.x * rpb; n0 < a.N; n0 += (int64_t)gridDim.x * rpb) {
    const int64_t n = WHOLE ? n0 : n0 + threadIdx.x / tx;
    const bool there = WHOLE || n < a.N;
    const int64_t r = there ? n : a.N - 1;
    const T* row = static_cast<const T*>(a.scores) + r * a.lds;
    T* out = static_cast<T*>(a.dscores) + r * a.V;
    const int span = tx * V * U, first = WHOLE ? (int)blockIdx.y * tiles * span : 0;
    const int last = WHOLE ? min(first + tiles * span, a.V) : a.V;
    uint4 next[U];
    const auto fetch = [&](int base) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int c = base + (j * tx + lane) * V;
        next[j] = fetch16<SHORT>(row + (c < a.V ? c : 0), c < a.V ? a.V - c : a.V);
      }
    };
    fetch(first);
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
    const int t = a.dchosen ? (int)token_at(a, r) : -1;
    const float dc = t >= 0 ? a.dchosen[r] : 0.f;
    const Quick q(f);
    const bool quick = (fabsf(f.m) < kNear || f.m == -INFINITY) && q.finite();
    if (there) {
      for (int base = first; base < last; base += span) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = next[j];
        if (WHOLE && base + span < last) fetch(base + span);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int c = base + (j * tx + lane) * V;
          if (c >= a.V) break;
          float v[V], o[V];
          unpack16<T>(keep16<SHORT, T>(u[j], a.V - c, a.V), v);
          if (quick) {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = q.slope(v[i]);
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = slope(f, v[i]);
          }
          const int at = t - c;
          if ((unsigned)at < (unsigned)V) {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] += at == i && v[i] > -INFINITY ? dc : 0.f;
          }
          store_row(out + c, a.V - c, o);
        }
      }
    }
    if (a.dtop) {
      // The alternatives' columns again, with what they get: after the row's part is written.
      __syncthreads();
      if (there) {
        for (int i = lane; i < a.k; i += tx) {
          const int32_t c = a.top_index[r * a.k + i];
          if (c < first || c >= last) continue;
          const float s = to_f32(row[c]);
          float g = quick ? q.slope(s) : slope(f, s);
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

// Without alternatives a wave takes a whole row also where rows enough fill the card: it waits for no other and has no
// barrier.  us a call by waves and by workgroups, for 128, 1000, 2500, 4096 and 10000 rows of V scores:
//    3001 bf16  7.4  7.7   7.6  7.8   7.7 10.8    8.3 15.7   16  34      fp32  7.4  7.3   7.7  7.6   8.4 11.9    11  17   22  37
//    9001       9.8 10.0   9.3 14.1  14.0 16.6   17   24     33  50           13   10    14   16    19   21      26  30   65  72
//   12288      12   10    11   14    17   16     20   22     41  45           17   10    17   18    23   22      33  32   89  81
//   32001      22   10    25   20    37   31     46   46    120 133           35   10    39   27    58   52      93  92  222 210
//   32768      22   10    25   19    37   30     52   44    131 114           34   10    39   26    65   55     101  94  238 215
// At 8192 x 65536 bf16 a workgroup is ahead, 185 against 212.  The type has no part in the rule, since the
// workspace's size, which callers ask for without one, goes by it too.
bool rows_by_wave(int64_t N, int V) { return V <= kShort || (V <= 9216 && N >= 1000) || (V <= 32768 && N >= 4096); }

template <typename T, int G, int NV, bool SHORT>
void rows_top(const LogpArgs& a, hipStream_t s) {
  const int64_t need = (a.N + kThreads / G - 1) / (kThreads / G);
  logp_rows_top_kernel<T, G, NV, SHORT><<<(unsigned)(need < kMaxBlocks ? need : kMaxBlocks), kThreads, 0, s>>>(a);
}

template <typename T>
void logp_typed(const LogpArgs& a, hipStream_t s) {
  if (a.k > 0 && short_rows(a.N, a.V, a.k)) {
    constexpr int N8 = 8 / kVec<T>;      // vectors of 8 scores
    if (a.V < kVec<T>) rows_top<T, 4, N8, true>(a, s);
    else if (a.V <= 32) rows_top<T, 4, N8, false>(a, s);
    else if (a.V <= 64) rows_top<T, 4, 2 * N8, false>(a, s);
    else if (a.V <= 128) rows_top<T, 8, 2 * N8, false>(a, s);
    else if (a.V <= 256) rows_top<T, 8, 4 * N8, false>(a, s);
    else if (a.V <= 512) rows_top<T, 16, 4 * N8, false>(a, s);
    else if (a.V <= 1024) rows_top<T, 32, 4 * N8, false>(a, s);
    else rows_top<T, 64, 4 * N8, false>(a, s);
    return;
  }
  if (a.k == 0 && rows_by_wave(a.N, a.V)) {
    if (a.V < kVec<T>) rows_grouped<T, 4, true>(a, s);
    else if (a.V <= 128) rows_grouped<T, 4, false>(a, s);
    else if (a.V <= 512) rows_grouped<T, 16, false>(a, s);
    else rows_grouped<T, 64, false>(a, s);
    return;
  }
  const dim3 grid((unsigned)a.splits, (unsigned)(a.N < 65535 ? a.N : 65535));
  if (a.k == 0) logp_part_kernel<T, false><<<grid, kThreads, 0, s>>>(a);             // (V > kShort)
  else logp_part_kernel<T, true><<<grid, kThreads, 0, s>>>(a);                        // (V > 256)
  if (a.splits == 1) return;
  const unsigned rows = (unsigned)(a.N < kMaxBlocks ? a.N : kMaxBlocks);
  if (a.k == 0) logp_join_kernel<T, false><<<rows, kThreads, 0, s>>>(a);
  else logp_join_kernel<T, true><<<rows, kThreads, 0, s>>>(a);
}

template <typename T>
void logp_bwd_typed(const LogpArgs& a, hipStream_t s) {
  constexpr int V = kVec<T>;
  const int nvec = (a.V + V * 4 - 1) / (V * 4);
  const auto grid = [](int64_t need) { return (unsigned)(need < kMaxBlocks ? need : kMaxBlocks); };
  if (nvec > kThreads / 2) {
    // parts of a row as long as 4096 workgroups allow
    const int64_t spans = (a.V + (int64_t)kThreads * V * 2 - 1) / (kThreads * V * 2);
    const int64_t parts = std::min(spans, std::max<int64_t>(1, 4096 / a.N)), tiles = (spans + parts - 1) / parts;
    const dim3 blocks(grid(a.N), (unsigned)((spans + tiles - 1) / tiles));
    logp_bwd_kernel<T, true, false><<<blocks, kThreads, 0, s>>>(a, kThreads, (int)tiles);
    return;
  }
  int tx = 4;
  while (tx < nvec) tx *= 2;
  const unsigned blocks = grid((a.N + kThreads / tx - 1) / (kThreads / tx));
  if (a.V < V) logp_bwd_kernel<T, false, true><<<blocks, kThreads, 0, s>>>(a, tx, 1);
  else logp_bwd_kernel<T, false, false><<<blocks, kThreads, 0, s>>>(a, tx, 1);
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

// Parts of a row: none with enough rows for the card, else parts of 4096 scores or more.
int logp_splits(int64_t N, int V, int k) {
  if (V <= kShort || (k == 0 && rows_by_wave(N, V))) return 1;
  const int64_t blocks = k ? 512 : 1024;
  int64_t parts = (blocks + N - 1) / (N > 0 ? N : 1);
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
