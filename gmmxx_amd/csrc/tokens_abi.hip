// C-ABI entry points of the token operators (declared in include/gmmxx_hip.h): arguments
// are checked against what the kernels and their grids assume, then the launches are
// enqueued on the caller's stream.

#include <math.h>
#include <stdint.h>

#include "engine.hpp"
#include "gmmxx_hip.h"
#include "tokens.hpp"

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

int check_embed(int elem, int64_t N, int64_t V, int64_t D, int index_bits, double scale) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || V <= 0 || D <= 0) return invalid("N must be non-negative and V and D positive");
  if (index_bits != 32 && index_bits != 64) return invalid("index_bits must be 32 or 64");
  if (!(fabs(scale) <= 3.4028234663852886e38)) return invalid("scale must be finite in fp32");
  if (V > kEmbedMaxV) return unsupported("V > 2^24");
  if (D > kMaxDim) return unsupported("D > 2^22");
  if (N >= kMaxPositions) return unsupported("N >= 2^30");
  if (N > (int64_t(1) << 40) / D || V > (int64_t(1) << 40) / D) return unsupported("N D or V D > 2^40");
  return GMMXX_OK;
}

int check_logp(int elem, int64_t N, int64_t V, int64_t k, int index_bits) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || V <= 0) return invalid("N must be non-negative and V positive");
  if (index_bits != 32 && index_bits != 64) return invalid("index_bits must be 32 or 64");
  if (k < 0 || k > V) return invalid("k must satisfy 0 <= k <= V");
  if (k > kLogpMaxK) return unsupported("k > 64");
  if (V > kLogpMaxV) return unsupported("V > 2^22");
  if (N >= kMaxPositions) return unsupported("N >= 2^30");
  return GMMXX_OK;
}

int check_quant(int elem, int64_t N, int64_t F, int64_t D) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || F <= 0 || D <= 0) return invalid("N must be non-negative and F and D positive");
  if (D > kQuantMaxD) return unsupported("D > 131072");
  if (F > kMaxDim) return unsupported("F > 2^22");
  if (N >= kMaxPositions) return unsupported("N >= 2^30");
  return GMMXX_OK;
}

int check_values(const int8_t* values, int64_t ld) {
  if (ld % 16 != 0 || ld < 0 || (uintptr_t)values % 16 != 0)
    return invalid("x and w must lie in rows of whole, aligned 16 bytes");
  if (ld > (1 << 23)) return unsupported("row strides > 2^23");
  return GMMXX_OK;
}

int64_t values_row(int64_t D) { return (D + kQuantPad - 1) / kQuantPad * kQuantPad; }
int64_t values_bytes(int64_t N, int64_t D) { return (N * values_row(D) + 255) / 256 * 256; }

}  // namespace

extern "C" {

int gmmxx_hip_embed(int elem, int64_t N, int64_t V, int64_t D, const void* table, int64_t ldt, const void* index,
                    int index_bits, double scale, void* out, void* stream) {
  if (int rc = check_embed(elem, N, V, D, index_bits, scale)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!table || !index || !out) return invalid("NULL buffer");
  if (ldt < 0) return invalid("row strides must be non-negative");
  EmbedArgs a{};
  a.table = table; a.ldt = ldt; a.index = index; a.index64 = index_bits == 64; a.out = out;
  a.N = N; a.V = V; a.D = (int)D; a.elem = elem; a.scale = (float)scale;
  launch_embed(a, (hipStream_t)stream);
  return launch_status("embed");
}

int64_t gmmxx_hip_embed_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  if (check_embed(GMMXX_F32, N, V, D, 32, 1.0)) return -1;
  return N ? embed_workspace_bytes(N, V, (int)D) : 0;
}

int gmmxx_hip_embed_backward(int elem, int64_t N, int64_t V, int64_t D, const void* dy, int64_t lddy,
                             const void* index, int index_bits, double scale, void* dtable, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (int rc = check_embed(elem, N, V, D, index_bits, scale)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!dy || !index || !dtable) return invalid("NULL buffer");
  if (lddy < 0) return invalid("row strides must be non-negative");
  if (int rc = check_workspace(workspace, workspace_bytes, embed_workspace_bytes(N, V, (int)D))) return rc;
  EmbedArgs a{};
  a.dy = dy; a.lddy = lddy; a.index = index; a.index64 = index_bits == 64; a.out = dtable;
  a.N = N; a.V = V; a.D = (int)D; a.elem = elem; a.scale = (float)scale;
  embed_workspace(a, workspace);
  launch_embed_bwd(a, (hipStream_t)stream);
  return launch_status("embed_backward");
}

int gmmxx_hip_dropout(int elem, int64_t n, double p, uint64_t seed, const int64_t* seed_at, uint64_t offset,
                      const void* x, const void* residual, void* out, void* stream) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (n < 0) return invalid("n must be non-negative");
  if (!(p >= 0.0 && p <= 1.0)) return invalid("p must satisfy 0 <= p <= 1");
  if (n > (int64_t(1) << 40)) return unsupported("n > 2^40");
  if (n == 0) return GMMXX_OK;
  if (!x || !out) return invalid("NULL buffer");
  DropArgs a{};
  const uint64_t border = (uint64_t)llrint(p * 4294967296.0);
  a.none = border >> 32 != 0;
  a.border = a.none ? 0xffffffffu : (uint32_t)border;
  a.scale = a.none ? 0.f : (float)(1.0 / (1.0 - p));
  a.x = x; a.residual = residual; a.out = out; a.seed = seed; a.seed_at = seed_at; a.offset = offset;
  a.n = n; a.elem = elem;
  launch_dropout(a, (hipStream_t)stream);
  return launch_status("dropout");
}

int64_t gmmxx_hip_log_probs_workspace_bytes(int64_t N, int64_t V, int64_t k) {
  if (check_logp(GMMXX_F32, N, V, k, 32)) return -1;
  return N ? logp_workspace_bytes(N, (int)V, (int)k) : 0;
}

int gmmxx_hip_log_probs(int elem, int64_t N, int64_t V, int64_t k, const void* scores, int64_t ld, const void* index,
                        int index_bits, float* chosen, float* entropy, float* top, int32_t* top_index, float* stats,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_logp(elem, N, V, k, index_bits)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!scores || !index || !chosen || !entropy || (k && (!top || !top_index))) return invalid("NULL buffer");
  if (ld < 0) return invalid("row strides must be non-negative");
  const int64_t need = logp_workspace_bytes(N, (int)V, (int)k);
  if (need)
    if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  LogpArgs a{};
  a.scores = scores; a.lds = ld; a.index = index; a.index64 = index_bits == 64;
  a.N = N; a.V = (int)V; a.k = (int)k; a.elem = elem;
  a.chosen = chosen; a.entropy = entropy; a.top = top; a.top_index = top_index; a.stats = stats;
  a.splits = logp_splits(N, (int)V, (int)k);
  a.part = static_cast<float*>(workspace);
  a.part_top = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + logp_top_offset(N, a.splits));
  launch_logp(a, (hipStream_t)stream);
  return launch_status("log_probs");
}

int gmmxx_hip_log_probs_backward(int elem, int64_t N, int64_t V, int64_t k, const void* scores, int64_t ld,
                                 const void* index, int index_bits, const int32_t* top_index, const float* stats,
                                 const float* dchosen, const float* dentropy, const float* dtop, void* dscores,
                                 void* stream) {
  if (int rc = check_logp(elem, N, V, k, index_bits)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!scores || !index || !stats || !dscores || (dtop && !top_index)) return invalid("NULL buffer");
  if (ld < 0) return invalid("row strides must be non-negative");
  LogpArgs a{};
  a.scores = scores; a.lds = ld; a.index = index; a.index64 = index_bits == 64;
  a.N = N; a.V = (int)V; a.k = (int)k; a.elem = elem;
  a.top_index = const_cast<int32_t*>(top_index); a.stats = const_cast<float*>(stats);
  a.dchosen = dchosen; a.dentropy = dentropy; a.dtop = k ? dtop : nullptr; a.dscores = dscores;
  launch_logp_bwd(a, (hipStream_t)stream);
  return launch_status("log_probs_backward");
}

int gmmxx_hip_quantize(int elem, int64_t N, int64_t D, const void* x, int64_t ldx, int8_t* values, int64_t ldv,
                       float* scales, void* stream) {
  if (!is_elem(elem)) return invalid("elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N < 0 || D <= 0) return invalid("N must be non-negative and D positive");
  if (D > kQuantMaxD) return unsupported("D > 131072");
  if (N >= kMaxPositions) return unsupported("N >= 2^30");
  if (N == 0) return GMMXX_OK;
  if (!x || !values || !scales) return invalid("NULL buffer");
  if (ldx < 0) return invalid("row strides must be non-negative");
  if (ldv % 16 != 0 || ldv < D || (uintptr_t)values % 16 != 0)
    return invalid("values must lie in rows of whole, aligned 16 bytes");
  QuantArgs a{};
  a.x = x; a.ldx = ldx; a.N = N; a.D = (int)D; a.elem = elem; a.values = values; a.ldv = ldv; a.scales = scales;
  launch_quantize(a, (hipStream_t)stream);
  return launch_status("quantize");
}

int gmmxx_hip_quantized_matmul(int elem, int64_t N, int64_t F, int64_t D, const int8_t* x, int64_t ldx,
                               const float* xscales, const int8_t* w, int64_t ldw, const float* wscales,
                               const void* bias, void* out, void* stream) {
  if (int rc = check_quant(elem, N, F, D)) return rc;
  if (N == 0) return GMMXX_OK;
  if (!x || !xscales || !w || !wscales || !out) return invalid("NULL buffer");
  if (int rc = check_values(x, ldx)) return rc;
  if (int rc = check_values(w, ldw)) return rc;
  QuantMatmulArgs a{};
  a.x = x; a.ldx = ldx; a.xs = xscales; a.w = w; a.ldw = ldw; a.ws = wscales; a.bias = bias; a.out = out;
  a.N = N; a.F = F; a.D = (int)D; a.elem = elem;
  launch_quant_matmul(a, (hipStream_t)stream);
  return launch_status("quantized_matmul");
}

int64_t gmmxx_hip_quantized_linear_workspace_bytes(int elem, int64_t N, int64_t D) {
  if (check_quant(elem, N, 1, D)) return -1;
  if (N == 0 || quant_linear_at_once(N, (int)D, elem)) return 0;
  return values_bytes(N, D) + (N * 4 + 255) / 256 * 256;
}

int gmmxx_hip_quantized_linear(int elem, int out_elem, int64_t N, int64_t F, int64_t D, const void* x, int64_t ldx,
                               const int8_t* w, int64_t ldw, const float* wscales, const void* bias, void* out,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_quant(elem, N, F, D)) return rc;
  if (!is_elem(out_elem)) return invalid("out_elem must be GMMXX_F32, GMMXX_BF16 or GMMXX_F16");
  if (N == 0) return GMMXX_OK;
  if (!x || !w || !wscales || !out) return invalid("NULL buffer");
  if (ldx < 0) return invalid("row strides must be non-negative");
  if (int rc = check_values(w, ldw)) return rc;
  if (const int64_t need = gmmxx_hip_quantized_linear_workspace_bytes(elem, N, D))
    if (int rc = check_workspace(workspace, workspace_bytes, need)) return rc;
  QuantArgs q{};
  q.x = x; q.ldx = ldx; q.N = N; q.D = (int)D; q.elem = elem;
  q.values = static_cast<int8_t*>(workspace); q.ldv = values_row(D);
  q.scales = reinterpret_cast<float*>(static_cast<char*>(workspace) + values_bytes(N, D));
  QuantMatmulArgs a{};
  a.x = q.values; a.ldx = q.ldv; a.xs = q.scales; a.w = w; a.ldw = ldw; a.ws = wscales; a.bias = bias; a.out = out;
  a.N = N; a.F = F; a.D = (int)D; a.elem = out_elem;
  launch_quant_linear(q, a, (hipStream_t)stream);
  return launch_status("quantized_linear");
}

}  // extern "C"
