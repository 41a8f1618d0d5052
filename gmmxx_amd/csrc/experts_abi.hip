// C-ABI entry points of the sparsely gated layer (declared in include/gmmxx_hip.h):
// arguments are checked against what the kernels and their grids assume, then the
// launches are enqueued on the caller's stream.

#include <stdint.h>

#include "engine.hpp"
#include "experts.hpp"
#include "gmmxx_hip.h"

namespace {

using namespace gx;
using namespace gx::layer;

constexpr int64_t kMaxPositions = int64_t(1) << 30;
constexpr int64_t kMaxDim = int64_t(1) << 22;

int invalid(const char* msg) { return set_error(GMMXX_ERR_INVALID_ARGUMENT, msg); }
int unsupported(const char* msg) { return set_error(GMMXX_ERR_UNSUPPORTED, msg); }

bool is_elem(int e) { return e == GMMXX_F32 || e == GMMXX_BF16 || e == GMMXX_F16; }

int check_workspace(const void* ws, int64_t have, int64_t need) {
  if (!ws) return set_error(GMMXX_ERR_WORKSPACE, "workspace is NULL");
  if (have < need) return set_error(GMMXX_ERR_WORKSPACE, "workspace too small");
  if ((uintptr_t)ws % 256 != 0) return set_error(GMMXX_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return GMMXX_OK;
}

int check_norm(int elem, int param_elem, int64_t N, int64_t D) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (param_elem != elem && param_elem != GMMXX_F32) return invalid("param_elem must be elem or GMMXX_F32");
  if (N < 0 || D <= 0) return invalid("N must be non-negative and D positive");
  if (D > kNormMaxD) return unsupported("D > 65536");
  return GMMXX_OK;
}

int check_route(int elem, int64_t N, int64_t E, int64_t k) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || E <= 0) return invalid("N must be non-negative and E positive");
  if (k < 1 || k > E) return invalid("k must satisfy 1 <= k <= E");
  if (E > kRouteMaxE) return unsupported("E > 4096");
  if (k > kRouteMaxK) return unsupported("k > 64");
  if (N >= kMaxPositions / k) return unsupported("N k >= 2^30");
  return GMMXX_OK;
}

int check_grouped(int elem, int64_t M, int64_t Nx, int64_t E, int64_t K, int64_t N, int offset_bits) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (M < 0 || E <= 0 || K <= 0 || N <= 0) return invalid("M must be non-negative and E, K and N positive");
  if (M > 0 && Nx <= 0) return invalid("x has no rows");
  if (offset_bits != 32 && offset_bits != 64) return invalid("offset_bits must be 32 or 64");
  if (E > kGroupedMaxE) return unsupported("E > 4096");
  if (M >= kMaxPositions) return unsupported("M >= 2^30");
  if (Nx > INT32_MAX) return unsupported("Nx >= 2^31");
  if (K > kMaxDim || N > kMaxDim) return unsupported("K or N > 2^22");
  return GMMXX_OK;
}

int check_combine(int elem, int64_t N, int64_t k, int64_t E, int64_t F) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || k <= 0 || E <= 0 || F <= 0) return invalid("N must be non-negative and k, E and F positive");
  if (k > kCombineMaxK) return unsupported("k > 64");
  if (E > INT32_MAX - 1) return unsupported("E too large");
  if (N >= kMaxPositions / k) return unsupported("N k >= 2^30");
  if (F > kMaxDim) return unsupported("F > 2^22");
  return GMMXX_OK;
}

GroupedArgs grouped_args(int elem, int64_t M, int64_t Nx, int64_t E, int64_t K, int64_t N, const void* x, int64_t ldx,
                         const int32_t* rows, const void* offsets, int offset_bits) {
  GroupedArgs a{};
  a.elem = elem; a.M = M; a.Nx = Nx; a.E = (int)E; a.K = (int)K; a.Nn = (int)N;
  a.x = x; a.ldx = ldx; a.rows = rows; a.offsets = offsets; a.off64 = offset_bits == 64;
  return a;
}

}  // namespace

extern "C" {

int gmmxx_hip_layer_norm(int elem, int param_elem, int64_t N, int64_t D, const void* x, int64_t ldx,
                         const void* weight, const void* bias, double eps, void* y, float* mean, float* rstd,
                         void* stream) {
  if (int rc = check_norm(elem, param_elem, N, D)) return rc;
  if (!(eps >= 0.0)) return invalid("eps must be non-negative");
  if (N == 0) return GMMXX_OK;
  if (!x || !y || !mean != !rstd) return invalid("NULL buffer");
  if (ldx < 0) return invalid("row strides must be non-negative");
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.N = N; a.D = (int)D; a.x_elem = elem; a.w_elem = param_elem; a.eps = (float)eps;
  launch_norm_fwd(a, (hipStream_t)stream);
  return launch_status("layer_norm");
}

int64_t gmmxx_hip_layer_norm_workspace_bytes(int64_t N, int64_t D) {
  if (check_norm(GMMXX_F32, GMMXX_F32, N, D)) return -1;
  return (int64_t)norm_blocks(N, (int)D) * 2 * D * 4;
}

int gmmxx_hip_layer_norm_backward(int elem, int param_elem, int64_t N, int64_t D, const void* x, int64_t ldx,
                                  const void* dy, int64_t lddy, const void* weight, const float* mean,
                                  const float* rstd, void* dx, void* dweight, void* dbias, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (int rc = check_norm(elem, param_elem, N, D)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!x || !dy || !mean || !rstd || !dx) return invalid("NULL buffer");
  if (ldx < 0 || lddy < 0) return invalid("row strides must be non-negative");
  const bool params = dweight || dbias;
  if (params)
    if (int rc = check_workspace(workspace, workspace_bytes, gmmxx_hip_layer_norm_workspace_bytes(N, D))) return rc;
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.weight = weight; a.y = dx;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.part = params ? static_cast<float*>(workspace) : nullptr; a.dweight = dweight; a.dbias = dbias;
  a.N = N; a.D = (int)D; a.x_elem = elem; a.w_elem = param_elem;
  launch_norm_bwd(a, (hipStream_t)stream);
  return launch_status("layer_norm_backward");
}

int64_t gmmxx_hip_route_workspace_bytes(int64_t N, int64_t E, int64_t k) {
  if (check_route(GMMXX_F32, N, E, k)) return -1;
  return route_workspace_bytes(N, (int)E);
}

int gmmxx_hip_route(int elem, int64_t N, int64_t E, int64_t k, int renormalize, const void* scores, int64_t ld,
                    int32_t* experts, float* gates, int32_t* offsets, int32_t* rows, int32_t* slots, float* norm,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_route(elem, N, E, k)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!scores || !experts || !gates || !offsets || !rows || !slots) return invalid("NULL buffer");
  if (ld < 0) return invalid("row strides must be non-negative");
  if (int rc = check_workspace(workspace, workspace_bytes, route_workspace_bytes(N, (int)E))) return rc;
  RouteArgs a{};
  a.scores = scores; a.lds = ld; a.N = N; a.E = (int)E; a.k = (int)k; a.elem = elem; a.renormalize = renormalize != 0;
  a.experts = experts; a.gates = gates; a.offsets = offsets; a.rows = rows; a.slots = slots;
  a.norm = reinterpret_cast<float2*>(norm);
  a.hist = static_cast<int32_t*>(workspace);
  a.totals = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + route_totals_offset(N, (int)E));
  launch_route(a, (hipStream_t)stream);
  return launch_status("route");
}

int gmmxx_hip_route_backward(int elem, int64_t N, int64_t E, int64_t k, int renormalize, const void* scores,
                             int64_t ld, const int32_t* experts, const float* gates, const float* norm,
                             const float* dgates, void* dscores, void* stream) {
  if (int rc = check_route(elem, N, E, k)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!experts || !gates || !dgates || !dscores) return invalid("NULL buffer");
  if (!renormalize && (!scores || !norm)) return invalid("gates over all candidates need scores and norm");
  if (ld < 0) return invalid("row strides must be non-negative");
  RouteArgs a{};
  a.scores = scores; a.lds = ld; a.N = N; a.E = (int)E; a.k = (int)k; a.elem = elem; a.renormalize = renormalize != 0;
  a.experts = const_cast<int32_t*>(experts); a.gates = const_cast<float*>(gates);
  a.norm = reinterpret_cast<float2*>(const_cast<float*>(norm)); a.dgates = dgates; a.dscores = dscores;
  launch_route_bwd(a, (hipStream_t)stream);
  return launch_status("route_backward");
}

int gmmxx_hip_grouped_matmul(int elem, int64_t M, int64_t Nx, int64_t E, int64_t K, int64_t N, const void* x,
                             int64_t ldx, const int32_t* rows, const void* w, int64_t we, int64_t wk, int64_t wn,
                             const void* bias, const void* offsets, int offset_bits, void* out, int out_elem,
                             void* stream) {
  if (int rc = check_grouped(elem, M, Nx, E, K, N, offset_bits)) return rc;
  if (out_elem != elem && out_elem != GMMXX_F32) return invalid("out_elem must be elem or GMMXX_F32");
  if (M == 0) return GMMXX_OK;
  if (!x || !w || !offsets || !out) return invalid("NULL buffer");
  if (ldx < 0 || we < 0 || wk < 0 || wn < 0) return invalid("strides must be non-negative");
  if (wk != 1 && wn != 1) return invalid("wk or wn must be 1");
  if (!rows && Nx < M) return invalid("x has fewer rows than there are positions");
  GroupedArgs a = grouped_args(elem, M, Nx, E, K, N, x, ldx, rows, offsets, offset_bits);
  a.w = w; a.we = we; a.wk = wk; a.wn = wn; a.bias = bias; a.out = out; a.out_f32 = out_elem != elem;
  launch_grouped(a, (hipStream_t)stream);
  return launch_status("grouped_matmul");
}

int64_t gmmxx_hip_grouped_workspace_bytes(int64_t M, int64_t E, int64_t K, int64_t N) {
  if (check_grouped(GMMXX_F32, M, 1, E, K, N, 32)) return -1;
  return grouped_workspace_bytes(M, E, K, N);
}

int gmmxx_hip_grouped_weight_grad(int elem, int64_t M, int64_t Nx, int64_t E, int64_t K, int64_t N, const void* x,
                                  int64_t ldx, const int32_t* rows, const void* dy, int64_t lddy,
                                  const void* offsets, int offset_bits, void* dw, void* dbias, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (int rc = check_grouped(elem, M, Nx, E, K, N, offset_bits)) return rc;
  if (M == 0) return GMMXX_OK;
  if (!x || !dy || !offsets || (!dw && !dbias)) return invalid("NULL buffer");
  if (ldx < 0 || lddy < 0) return invalid("strides must be non-negative");
  if (!rows && Nx < M) return invalid("x has fewer rows than there are positions");
  if (const int64_t need = gmmxx_hip_grouped_workspace_bytes(M, E, K, N))
    if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  GroupedArgs a = grouped_args(elem, M, Nx, E, K, N, x, ldx, rows, offsets, offset_bits);
  a.dy = dy; a.lddy = lddy; a.out = dw; a.dbias = dbias; a.part = static_cast<float*>(workspace);
  launch_grouped_dw(a, (hipStream_t)stream);
  return launch_status("grouped_weight_grad");
}

int gmmxx_hip_combine(int elem, int64_t N, int64_t k, int64_t E, int64_t F, const void* y, int y_elem, int64_t ldy,
                      const float* gates, const int32_t* slots, const int32_t* offsets, void* out, void* stream) {
  if (int rc = check_combine(elem, N, k, E, F)) return rc;
  if (y_elem != elem && y_elem != GMMXX_F32) return invalid("y_elem must be elem or GMMXX_F32");
  if (N == 0) return GMMXX_OK;
  if (!y || !slots || !offsets || !out) return invalid("NULL buffer");
  if (ldy < 0) return invalid("row strides must be non-negative");
  CombineArgs a{};
  a.y = y; a.ldy = ldy; a.gates = gates; a.slots = slots; a.offsets = offsets; a.E = (int)E; a.out = out;
  a.N = N; a.M = N * k; a.F = (int)F; a.k = (int)k; a.elem = elem; a.y_f32 = y_elem != elem;
  launch_combine(a, (hipStream_t)stream);
  return launch_status("combine");
}

int gmmxx_hip_combine_backward(int elem, int64_t N, int64_t k, int64_t E, int64_t F, const void* y, int64_t ldy,
                               const float* gates, const int32_t* slots, const int32_t* offsets, const void* dout,
                               int64_t lddout, void* dy, float* dgates, void* stream) {
  if (int rc = check_combine(elem, N, k, E, F)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!y || !gates || !slots || !offsets || !dout || !dy || !dgates) return invalid("NULL buffer");
  if (ldy < 0 || lddout < 0) return invalid("row strides must be non-negative");
  CombineArgs a{};
  a.y = y; a.ldy = ldy; a.gates = gates; a.slots = slots; a.offsets = offsets; a.E = (int)E;
  a.dout = dout; a.lddout = lddout; a.out = dy; a.dgates = dgates;
  a.N = N; a.M = N * k; a.F = (int)F; a.k = (int)k; a.elem = elem;
  launch_combine_bwd(a, (hipStream_t)stream);
  return launch_status("combine_backward");
}

}  // extern "C"
