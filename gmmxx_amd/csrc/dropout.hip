// Dropout by a counter-based generator: the mask is a function of (seed, offset, element)
// and is computed wherever it is needed, never stored.
//
//   word(i) = word i % 4 of Philox 4x32-10 at counter (i / 4, offset), key seed
//   y_i = [word(i) >= border] x_i scale + residual_i,   dx_i = [word(i) >= border] dy_i scale
// with border = round(p 2^32) and scale = 1 / (1 - p).  (Generator: Salmon, Moraes, Dror
// and Shaw, Parallel random numbers: as easy as 1, 2, 3, 2011.)  Words belong to elements
// in the order of the tensor's shape, whatever its type, so both directions and both
// 16-bit types see one mask.  A dropped element is zero whatever x holds.
//
// A thread takes 16 bytes of x: one or two counters, whose words are all used.  Bound by bytes: 16384 x 4096
// bf16 with a residual 71 us (403 MB, 5.7 TB/s), the gradient 55 us (268 MB, 4.9 TB/s); eight elements take 195
// instructions, most of them the rounds', somewhat more than half of what the card issues in that time.

#include "rows.hpp"
#include "tokens.hpp"

namespace gx::layer {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)0xD2511F53u * c.x, q = (uint64_t)0xCD9E8D57u * c.z;
    c = make_uint4((uint32_t)(q >> 32) ^ c.y ^ k0, (uint32_t)q, (uint32_t)(p >> 32) ^ c.w ^ k1, (uint32_t)p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

template <typename T, bool RESIDUAL>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a) {
  constexpr int V = kVec<T>;
  const uint64_t seed = a.seed_at ? (uint64_t)*a.seed_at : a.seed;
  const int64_t vectors = (a.n + V - 1) / V;
  for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < vectors; g += (int64_t)gridDim.x * kThreads) {
    const int64_t i = g * V;
    const int valid = a.n - i < V ? (int)(a.n - i) : V;
    float v[V], r[V];
    uint4 u, w;
    // (a vector that ends past the last element is read element by element)
    if (valid == V) {
      u = ld16_any(static_cast<const T*>(a.x) + i);
      if constexpr (RESIDUAL) w = ld16_any(static_cast<const T*>(a.residual) + i);
    } else {
      u = fetch16<true>(static_cast<const T*>(a.x) + i, valid);
      if constexpr (RESIDUAL) w = fetch16<true>(static_cast<const T*>(a.residual) + i, valid);
    }
    unpack16<T>(u, v);
    if constexpr (RESIDUAL) unpack16<T>(w, r);
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      const uint64_t c = (uint64_t)g * (V / 4) + h;
      const uint4 p = philox(make_uint4((uint32_t)c, (uint32_t)(c >> 32), (uint32_t)a.offset,
                                        (uint32_t)(a.offset >> 32)), (uint32_t)seed, (uint32_t)(seed >> 32));
      const uint32_t word[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * h + j;
        v[e] = word[j] >= a.border && !a.none ? (RESIDUAL ? fmaf(v[e], a.scale, r[e]) : v[e] * a.scale)
                                              : (RESIDUAL ? r[e] : 0.f);
      }
    }
    store_row(static_cast<T*>(a.out) + i, valid, v);
  }
}

template <typename T>
void dropout_typed(const DropArgs& a, hipStream_t s) {
  const int64_t blocks = ((a.n + kVec<T> - 1) / kVec<T> + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
  if (a.residual) dropout_kernel<T, true><<<grid, kThreads, 0, s>>>(a);
  else dropout_kernel<T, false><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

void launch_dropout(const DropArgs& a, hipStream_t s) {
  if (a.elem == ELEM_F32) dropout_typed<float>(a, s);
  else if (a.elem == ELEM_BF16) dropout_typed<__bf16>(a, s);
  else dropout_typed<_Float16>(a, s);
}

}  // namespace gx::layer
