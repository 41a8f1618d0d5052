// Argument blocks and launchers of the sparsely gated layer: layer norm, row routing,
// grouped products and the combination of the experts' results (entry points in
// experts_abi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gx::layer {

enum Elem { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };   // enum gmmxx_dtype

constexpr int kNormMaxD = 65536;
constexpr int kNormMaxBlocks = 512;     // row slices of the backward pass
struct NormArgs {
  const void* x;  int64_t ldx;           // rows of D elements, row stride in elements
  const void* dy; int64_t lddy;
  const void* weight;                    // D, or null (ones)
  const void* bias;                      // D, or null (zeros)
  void* y;                               // contiguous rows (forward: y, backward: dx)
  float* mean;                           // N
  float* rstd;                           // N
  float* part;                           // backward: [blocks][2][D] partial sums of dw, db
  void* dweight; void* dbias;            // D, or null
  int64_t N;
  int D;
  int x_elem, w_elem;
  float eps;
};
int norm_blocks(int64_t N, int D);
void launch_norm_fwd(const NormArgs& a, hipStream_t s);
void launch_norm_bwd(const NormArgs& a, hipStream_t s);

constexpr int kRouteMaxE = 4096;
constexpr int kRouteMaxK = 64;
struct RouteArgs {
  const void* scores; int64_t lds;       // rows of E scores
  int64_t N;
  int E, k, elem, renormalize;
  int32_t* experts;                      // [N][k]
  float* gates;                          // [N][k]
  int32_t* offsets;                      // [E + 1]
  int32_t* rows;                         // [N k]
  int32_t* slots;                        // [N][k]
  float2* norm;                          // [N] largest candidate, 1 / sum (or null)
  int32_t* hist;                         // workspace: [blocks][E + 1] counts, then their exclusive prefixes
  int32_t* totals;                       // workspace: [E + 1]
  const float* dgates;                   // backward: [N][k]
  void* dscores;                         // backward: [N][E]
};
int64_t route_workspace_bytes(int64_t N, int E);
int64_t route_totals_offset(int64_t N, int E);   // of `totals` in the workspace, after `hist`
void launch_route(const RouteArgs& a, hipStream_t s);
void launch_route_bwd(const RouteArgs& a, hipStream_t s);

constexpr int kGroupedMaxE = 4096;
struct GroupedArgs {
  const void* x; int64_t ldx;            // rows of K elements
  const int32_t* rows;                   // source row of each of the M positions, or null (position p is row p)
  int64_t Nx;                            // rows of x
  const void* w; int64_t we, wk, wn;     // weight element (e, k, n) at e we + k wk + n wn; wk or wn is 1
  const void* bias;                      // [E][Nn], or null
  const void* offsets; int off64;        // [E + 1] int32 or int64
  const void* dy; int64_t lddy;          // weight gradient: M rows of Nn elements
  void* out;                             // [M][Nn], or [E][K][Nn] for the weight gradient
  void* dbias;                           // [E][Nn], or null
  float* part;                           // weight gradient in parts: [splits][E][K][Nn]
  float* bias_part;                      // the bias's in parts: [splits][E][Nn]
  int64_t M;
  int E, K, Nn, elem;
  int out_f32;                           // out is fp32 whatever the elements are
};
void launch_grouped(const GroupedArgs& a, hipStream_t s);
void launch_grouped_dw(const GroupedArgs& a, hipStream_t s);
int64_t grouped_workspace_bytes(int64_t M, int64_t E, int64_t K, int64_t N);
// Whole, aligned 16-byte chunks, which the tiles load straight into LDS.
bool grouped_direct(const GroupedArgs& a);
// Few rows for each expert (grouped_few.hip).
bool grouped_few_better(const GroupedArgs& a);
void launch_grouped_few(const GroupedArgs& a, hipStream_t s);

constexpr int kCombineMaxK = 64;
struct CombineArgs {
  const void* y; int64_t ldy;            // M rows of F elements
  const float* gates;                    // [N][k], or null (ones)
  const int32_t* slots;                  // [N][k]
  const int32_t* offsets; int E;         // positions from offsets[E] on belong to no expert
  const void* dout; int64_t lddout;      // backward: N rows of F elements
  void* out;                             // forward: [N][F]; backward: dy [M][F]
  float* dgates;                         // backward: [N][k]
  int64_t N, M;
  int F, k, elem;                        // elem: of out (and dout)
  int y_f32;                             // y is fp32 whatever elem is (forward)
};
void launch_combine(const CombineArgs& a, hipStream_t s);
void launch_combine_bwd(const CombineArgs& a, hipStream_t s);

}  // namespace gx::layer
