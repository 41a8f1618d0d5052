// What the autograd functions share: the library's entry points, the device and stream of a
// call, and what is refused.
#pragma once

#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <string>
#include <tuple>
#include <unordered_map>

#include "gmmxx_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&gmmxx_hip_last_error) last_error = nullptr;
  decltype(&gmmxx_hip_layer_norm) layer_norm = nullptr;
  decltype(&gmmxx_hip_layer_norm_workspace_bytes) layer_norm_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_layer_norm_backward) layer_norm_backward = nullptr;
  decltype(&gmmxx_hip_route_workspace_bytes) route_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_route) route = nullptr;
  decltype(&gmmxx_hip_route_backward) route_backward = nullptr;
  decltype(&gmmxx_hip_grouped_matmul) grouped_matmul = nullptr;
  decltype(&gmmxx_hip_grouped_workspace_bytes) grouped_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_grouped_weight_grad) grouped_weight_grad = nullptr;
  decltype(&gmmxx_hip_combine) combine = nullptr;
  decltype(&gmmxx_hip_combine_backward) combine_backward = nullptr;
  decltype(&gmmxx_hip_embed) embed = nullptr;
  decltype(&gmmxx_hip_embed_workspace_bytes) embed_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_embed_backward) embed_backward = nullptr;
  decltype(&gmmxx_hip_dropout) dropout = nullptr;
  decltype(&gmmxx_hip_log_probs_workspace_bytes) log_probs_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_log_probs) log_probs = nullptr;
  decltype(&gmmxx_hip_log_probs_backward) log_probs_backward = nullptr;
  decltype(&gmmxx_hip_quantize) quantize = nullptr;
  decltype(&gmmxx_hip_quantized_matmul) quantized_matmul = nullptr;
  decltype(&gmmxx_hip_quantized_linear_workspace_bytes) quantized_linear_workspace_bytes = nullptr;
  decltype(&gmmxx_hip_quantized_linear) quantized_linear = nullptr;
} lib;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
  auto take = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name));
  };
  take(lib.last_error, "last_error");
  take(lib.layer_norm, "layer_norm");
  take(lib.layer_norm_workspace_bytes, "layer_norm_workspace_bytes");
  take(lib.layer_norm_backward, "layer_norm_backward");
  take(lib.route_workspace_bytes, "route_workspace_bytes");
  take(lib.route, "route");
  take(lib.route_backward, "route_backward");
  take(lib.grouped_matmul, "grouped_matmul");
  take(lib.grouped_workspace_bytes, "grouped_workspace_bytes");
  take(lib.grouped_weight_grad, "grouped_weight_grad");
  take(lib.combine, "combine");
  take(lib.combine_backward, "combine_backward");
  take(lib.embed, "embed");
  take(lib.embed_workspace_bytes, "embed_workspace_bytes");
  take(lib.embed_backward, "embed_backward");
  take(lib.dropout, "dropout");
  take(lib.log_probs_workspace_bytes, "log_probs_workspace_bytes");
  take(lib.log_probs, "log_probs");
  take(lib.log_probs_backward, "log_probs_backward");
  take(lib.quantize, "quantize");
  take(lib.quantized_matmul, "quantized_matmul");
  take(lib.quantized_linear_workspace_bytes, "quantized_linear_workspace_bytes");
  take(lib.quantized_linear, "quantized_linear");
}

// The device of a call: current while it lives, with its current stream.
class On {
 public:
  explicit On(const Tensor& t) : guard_(t.device()), stream_(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
  void* stream() const { return stream_; }

 private:
  c10::DeviceGuard guard_;
  void* stream_;
};

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "gmmxx_hip_", what, " failed (status ", rc, "): ", lib.last_error());
}

int elem(at::ScalarType t) { return t == at::kFloat ? GMMXX_F32 : t == at::kBFloat16 ? GMMXX_BF16 : GMMXX_F16; }
int elem(const Tensor& t) { return elem(t.scalar_type()); }

// A tensor that stands for values without holding them (a fake or functional tensor, torch's efficient zeros) gives
// a null pointer, which the library takes for an operand that is not there.
void* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.data_ptr();
  TORCH_CHECK_NOT_IMPLEMENTED(p || t.numel() == 0, "gmmxx_amd operators need tensors that hold their values");
  return p;
}
float* floats(const Tensor& t) { return static_cast<float*>(ptr(t)); }
int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(ptr(t)); }

// A tensor whose memory holds its values: a view may stand for the negatives of them (the imaginary part of a
// conjugate), which data_ptr() does not tell.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// A matrix whose rows' elements are adjacent.
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? plain(t) : plain(t).contiguous(); }

Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// What no result would show is refused: the operators have no forward-mode derivative, and a result without a
// tangent would pass for a constant; a trace would record the results' allocation but not the launch that writes
// them.
void refuse(std::initializer_list<const Tensor*> ts) {
  using c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() && !(TorchDispatchModeTLS::any_modes_set() &&
                                            TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY)),
      "gmmxx_amd operators cannot be traced");
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "gmmxx_amd operators have no forward-mode derivative");
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  refuse(ts);
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients asked for with a graph of their own: an error where that graph is used.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list fake;
  for (const Tensor& g : grads)
    if (g.defined()) fake.push_back(g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a gmmxx_amd operator, whose gradient has none", (int)fake.size());
  variable_list out = (*error)(std::move(fake));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
std::optional<Tensor> plain(const std::optional<Tensor>& t) { return t.has_value() ? std::optional(plain(*t)) : t; }

}  // namespace
