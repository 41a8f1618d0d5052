// Argument blocks and launchers of the token operators: embedding, dropout, log
// probabilities and products in 8-bit integers (entry points in tokens_abi.hip).
#pragma once

#include "experts.hpp"

namespace gx::layer {

constexpr int64_t kEmbedMaxV = int64_t(1) << 24;
struct EmbedArgs {
  const void* table; int64_t ldt;        // forward: V rows of D elements, row stride in elements
  const void* index; int index64;        // N tokens, int32 or int64; outside 0 .. V-1: none
  const void* dy; int64_t lddy;          // backward: N rows of D elements
  void* out;                             // contiguous: forward [N][D], backward [V][D]
  int64_t N, V;
  int D, elem;
  float scale;
  // backward's workspace: tokens and positions in two buffers each, the blocks' counts, the tiles' partial sums
  uint32_t* key[2];
  int32_t* pos[2];
  int32_t* hist;
  int32_t* totals;
  uint8_t* seen;                         // [V] whether a token has a place
  float* part;
};
int64_t embed_workspace_bytes(int64_t N, int64_t V, int D);
void embed_workspace(EmbedArgs& a, void* ws);      // sets the workspace's pointers
void launch_embed(const EmbedArgs& a, hipStream_t s);
void launch_embed_bwd(const EmbedArgs& a, hipStream_t s);

struct DropArgs {
  const void* x;                         // n elements
  const void* residual;                  // n elements, or null
  void* out;
  const int64_t* seed_at;                // read by the kernel, or null: seed
  uint64_t seed, offset;
  int64_t n;
  uint32_t border;                       // words below it are dropped
  int none;                              // every element is dropped
  float scale;
  int elem;
};
void launch_dropout(const DropArgs& a, hipStream_t s);

constexpr int kLogpMaxK = 64;
constexpr int64_t kLogpMaxV = int64_t(1) << 22;
struct LogpArgs {
  const void* scores; int64_t lds;       // N rows of V scores
  const void* index; int index64;        // N tokens
  int64_t N;
  int V, k, elem;
  float* chosen;                         // N
  float* entropy;                        // N
  float* top;                            // [N][k]
  int32_t* top_index;                    // [N][k], -1: no candidate was left
  float* stats;                          // [N][3]: largest candidate, log sum, entropy (or null)
  const float* dchosen; const float* dentropy; const float* dtop;   // backward: N, N, [N][k] (or null)
  void* dscores;                         // backward: [N][V]
  float* part;                           // workspace: [N][splits][3]
  uint64_t* part_top;                    // workspace: [N][splits][k]
  int splits;
};
int logp_splits(int64_t N, int V, int k);
int64_t logp_workspace_bytes(int64_t N, int V, int k);
int64_t logp_top_offset(int64_t N, int splits);      // of `part_top` in the workspace
void launch_logp(const LogpArgs& a, hipStream_t s);
void launch_logp_bwd(const LogpArgs& a, hipStream_t s);

constexpr int kQuantMaxD = 1 << 17;      // sums of D products of two values from -128 to 127 lie above -2^31 and up to 2^31
constexpr int kQuantPad = 128;           // rows of 8-bit values are padded to whole cache lines
struct QuantArgs {
  const void* x; int64_t ldx;            // N rows of D elements
  int64_t N;
  int D, elem;
  int8_t* values; int64_t ldv;           // rows of D values, zeros up to the next multiple of 16
  float* scales;                         // N
};
void launch_quantize(const QuantArgs& a, hipStream_t s);

struct QuantMatmulArgs {
  const int8_t* x; int64_t ldx;          // N rows of D values, readable in whole 16 bytes
  const float* xs;                       // N
  const int8_t* w; int64_t ldw;          // F rows of D values, likewise
  const float* ws;                       // F
  const void* bias;                      // F of `elem`, or null
  void* out;                             // [N][F]
  int64_t N, F;
  int D, elem;
};
void launch_quant_matmul(const QuantMatmulArgs& a, hipStream_t s);
// The two one after the other (x.values is a.x), or one kernel without x.values and x.scales.
bool quant_linear_at_once(int64_t N, int D, int elem);
void launch_quant_linear(const QuantArgs& x, const QuantMatmulArgs& a, hipStream_t s);

}  // namespace gx::layer
