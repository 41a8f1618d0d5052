// The sparsely gated layer's operators as autograd functions: tensors in, tensors out,
// with the library's C ABI (include/gmmxx_hip.h) in between.
//
// The backward pass of a Python autograd function takes the interpreter's lock on the
// engine's own thread; at small sizes that and the interpreter cost several times what
// the kernels do: the norm of one row takes 6 us a call where it took 11, of 100003 x
// 100 with its gradients 70 us where it took 118 (46 us of them kernels).  Here both
// directions run without the interpreter.  The entry points are those of the library
// that the package loaded: their addresses are handed over once (bind), so there is one
// library whatever its path.
//
// Arguments have been checked by the caller (gmmxx_amd/experts.py): matrices with
// adjacent row elements, matching shapes, types and devices.

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

// --- layer norm ---------------------------------------------------------------

Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, float* stats) {
  const int64_t n = x.size(0), d = x.size(1);
  Tensor y = at::empty({n, d}, x.options());
  if (n == 0) return y;
  On on(x);
  const int param = w.defined() ? elem(w) : b.defined() ? elem(b) : elem(x);
  check(lib.layer_norm(elem(x), param, n, d, ptr(x), x.stride(0), ptr(w), ptr(b), eps, ptr(y), stats,
                       stats ? stats + n : nullptr, on.stream()),
        "layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    const Tensor w = or_none(weight), b = or_none(bias);
    Tensor stats = at::empty({2 * x.size(0)}, x.options().dtype(at::kFloat));
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["bias"] = (int64_t)(b.defined() ? (int)b.scalar_type() : -1);
    return norm_forward(x, w, b, eps, floats(stats));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t n = x.size(0), d = x.size(1), bias = ctx->saved_data["bias"].toInt();
    const at::ScalarType param = w.defined() ? w.scalar_type() : bias >= 0 ? (at::ScalarType)bias : x.scalar_type();
    size_t edge = 1;
    const bool need_w = w.defined() && ctx->needs_input_grad(edge++);
    const bool need_b = bias >= 0 && ctx->needs_input_grad(edge);
    const auto options = x.options().dtype(param);
    Tensor dx = at::empty({n, d}, x.options()), dw, db;
    if (need_w) dw = n ? at::empty({d}, options) : at::zeros({d}, options);
    if (need_b) db = n ? at::empty({d}, options) : at::zeros({d}, options);
    if (n) {
      const Tensor dy = rows_of(grads[0]);
      On on(x);
      const int64_t need = need_w || need_b ? lib.layer_norm_workspace_bytes(n, d) : 0;
      const Tensor ws = need ? bytes(need, x) : Tensor();
      check(lib.layer_norm_backward(elem(x), elem(param), n, d, ptr(x), x.stride(0), ptr(dy), dy.stride(0), ptr(w),
                                    floats(stats), floats(stats) + n, ptr(dx), ptr(dw), ptr(db), ptr(ws), need,
                                    on.stream()),
            "layer_norm_backward");
    }
    return once({dx, dw, db, Tensor()});
  }
};

Tensor layer_norm(const Tensor& x0, const std::optional<Tensor>& weight0, const std::optional<Tensor>& bias0,
                  double eps) {
  const Tensor x = plain(x0);
  const std::optional<Tensor> weight = plain(weight0), bias = plain(bias0);
  const Tensor w = or_none(weight), b = or_none(bias);
  if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, weight, bias, eps);
  return norm_forward(x, w, b, eps, nullptr);
}

// --- routing --------------------------------------------------------------------

// experts, gates, offsets, rows, slots and, if wanted, the rows' normalisers.
variable_list route_forward(const Tensor& scores, int64_t k, bool renormalize, bool want_norm) {
  const int64_t n = scores.size(0), e = scores.size(1), m = n * k;
  const auto options = scores.options();
  Tensor experts = at::empty({n, k}, options.dtype(at::kInt)), gates = at::empty({n, k}, options.dtype(at::kFloat));
  Tensor offsets = n ? at::empty({e + 1}, options.dtype(at::kInt)) : at::zeros({e + 1}, options.dtype(at::kInt));
  Tensor rows = at::empty({m}, options.dtype(at::kInt)), slots = at::empty({n, k}, options.dtype(at::kInt));
  Tensor norm = want_norm ? at::empty({n, 2}, options.dtype(at::kFloat)) : Tensor();
  if (n) {
    On on(scores);
    const int64_t need = lib.route_workspace_bytes(n, e, k);
    const Tensor ws = bytes(need, scores);
    check(lib.route(elem(scores), n, e, k, renormalize, ptr(scores), scores.stride(0), ints(experts), floats(gates),
                    ints(offsets), ints(rows), ints(slots), floats(norm), ptr(ws), need, on.stream()),
          "route");
  }
  return {experts, gates, offsets, rows, slots, norm};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& scores, int64_t k, bool renormalize) {
    variable_list out = route_forward(scores, k, renormalize, !renormalize);
    ctx->save_for_backward({out[0], out[1], renormalize ? Tensor() : scores, out[5]});
    ctx->saved_data["renormalize"] = renormalize;
    ctx->saved_data["e"] = scores.size(1);
    ctx->saved_data["type"] = (int64_t)scores.scalar_type();
    out.pop_back();
    ctx->mark_non_differentiable({out[0], out[2], out[3], out[4]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[1]});
    if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &experts = saved[0], &gates = saved[1], &scores = saved[2], &norm = saved[3];
    const bool renormalize = ctx->saved_data["renormalize"].toBool();
    const int64_t n = gates.size(0), k = gates.size(1), e = ctx->saved_data["e"].toInt();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    Tensor ds = at::empty({n, e}, gates.options().dtype(type));
    if (n) {
      const Tensor dg = plain(grads[1]).contiguous();
      On on(gates);
      check(lib.route_backward(elem(type), n, e, k, renormalize, ptr(scores), scores.defined() ? scores.stride(0) : 0,
                               ints(experts), floats(gates), floats(norm), floats(dg), ptr(ds), on.stream()),
            "route_backward");
    }
    return once({ds, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route(const Tensor& scores0, int64_t k, bool renormalize) {
  const Tensor scores = plain(scores0);
  const variable_list r =
      wants_grad({&scores}) ? Route::apply(scores, k, renormalize) : route_forward(scores, k, renormalize, false);
  return {r[0], r[1], r[2], r[3], r[4]};
}

// --- grouped products -----------------------------------------------------------

// out (M, w.size(out_dim)): rows of x by w's matrices, summed over reduce_dim.  A dimension of one element counts
// as adjacent where the other is not.
Tensor grouped_forward(const Tensor& x, const Tensor& w, int reduce_dim, int out_dim, const Tensor& bias,
                       const Tensor& offsets, const Tensor& rows, int64_t m, at::ScalarType out_type) {
  Tensor out = at::empty({m, w.size(out_dim)}, x.options().dtype(out_type));
  if (m == 0) return out;
  int64_t wk = w.stride(reduce_dim), wn = w.stride(out_dim);
  if (wk != 1 && wn != 1) (w.size(reduce_dim) == 1 ? wk : wn) = 1;
  On on(x);
  check(lib.grouped_matmul(elem(x), m, x.size(0), w.size(0), w.size(reduce_dim), w.size(out_dim), ptr(x), x.stride(0),
                           ints(rows), ptr(w), w.stride(0), wk, wn, ptr(bias), ptr(offsets),
                           8 * (int)offsets.element_size(), ptr(out), elem(out_type), on.stream()),
        "grouped_matmul");
  return out;
}

Tensor combine_forward(const Tensor& y, const Tensor& gates, const Tensor& slots, const Tensor& offsets,
                       at::ScalarType type) {
  const int64_t n = slots.size(0), k = slots.size(1);
  Tensor out = at::empty({n, y.size(1)}, y.options().dtype(type));
  if (n == 0) return out;
  On on(y);
  check(lib.combine(elem(type), n, k, offsets.size(0) - 1, y.size(1), ptr(y), elem(y), y.stride(0), floats(gates),
                    ints(slots), ints(offsets), ptr(out), on.stream()),
        "combine");
  return out;
}

struct Grouped : torch::autograd::Function<Grouped> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                        const Tensor& offsets, const std::optional<Tensor>& rows, const std::optional<Tensor>& slots) {
    const Tensor r = or_none(rows);
    ctx->save_for_backward({x, w, offsets, r, or_none(slots)});
    ctx->saved_data["bias"] = bias.has_value();
    return grouped_forward(x, w, 1, 2, or_none(bias), offsets, r, r.defined() ? r.size(0) : x.size(0), x.scalar_type());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &offsets = saved[2], &rows = saved[3], &slots = saved[4];
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    const Tensor dy = rows_of(grads[0]);
    const int64_t m = dy.size(0), f = dy.size(1), e = w.size(0), d = w.size(1);
    Tensor dx, dw, db;
    if (need_x && !rows.defined()) {
      dx = grouped_forward(dy, w, 2, 1, Tensor(), offsets, Tensor(), m, x.scalar_type());
    } else if (need_x) {
      // A row's choices are added in fp32 and rounded once; a single choice needs no sum.
      const auto type = slots.size(1) == 1 ? x.scalar_type() : at::kFloat;
      const Tensor parts = grouped_forward(dy, w, 2, 1, Tensor(), offsets, Tensor(), m, type);
      dx = combine_forward(parts, Tensor(), slots, offsets, x.scalar_type());
    }
    if (need_w || need_b) {
      if (need_w) dw = m ? at::empty({e, d, f}, x.options()) : at::zeros({e, d, f}, x.options());
      if (need_b) db = m ? at::empty({e, f}, x.options()) : at::zeros({e, f}, x.options());
      if (m) {
        On on(x);
        const int64_t need = lib.grouped_workspace_bytes(m, e, d, f);
        const Tensor ws = need ? bytes(need, x) : Tensor();
        check(lib.grouped_weight_grad(elem(x), m, x.size(0), e, d, f, ptr(x), x.stride(0), ints(rows), ptr(dy),
                                      dy.stride(0), ptr(offsets), 8 * (int)offsets.element_size(), ptr(dw), ptr(db),
                                      ptr(ws), need, on.stream()),
              "grouped_weight_grad");
      }
    }
    return once({dx, dw, db, Tensor(), Tensor(), Tensor()});
  }
};

Tensor grouped(const Tensor& x0, const Tensor& w0, const std::optional<Tensor>& bias0, const Tensor& offsets,
               const std::optional<Tensor>& rows, const std::optional<Tensor>& slots) {
  const Tensor x = plain(x0), w = plain(w0);
  const std::optional<Tensor> bias = plain(bias0);
  const Tensor b = or_none(bias), r = or_none(rows);
  if (wants_grad({&x, &w, &b})) return Grouped::apply(x, w, bias, offsets, rows, slots);
  return grouped_forward(x, w, 1, 2, b, offsets, r, r.defined() ? r.size(0) : x.size(0), x.scalar_type());
}

// --- combination ----------------------------------------------------------------

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& gates, const Tensor& slots,
                        const Tensor& offsets) {
    ctx->save_for_backward({y, gates, slots, offsets});
    return combine_forward(y, gates, slots, offsets, y.scalar_type());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &y = saved[0], &gates = saved[1], &slots = saved[2], &offsets = saved[3];
    const int64_t n = slots.size(0), k = slots.size(1);
    Tensor dy = at::empty(y.sizes(), y.options()), dg = at::empty({n, k}, gates.options());
    if (n) {
      const Tensor dout = rows_of(grads[0]);
      On on(y);
      check(lib.combine_backward(elem(y), n, k, offsets.size(0) - 1, y.size(1), ptr(y), y.stride(0), floats(gates),
                                 ints(slots), ints(offsets), ptr(dout), dout.stride(0), ptr(dy), floats(dg),
                                 on.stream()),
            "combine_backward");
    }
    if (!ctx->needs_input_grad(0)) dy = Tensor();
    if (!ctx->needs_input_grad(1)) dg = Tensor();
    return once({dy, dg, Tensor(), Tensor()});
  }
};

Tensor combine(const Tensor& y0, const Tensor& gates0, const Tensor& slots, const Tensor& offsets) {
  const Tensor y = plain(y0), gates = plain(gates0);
  if (wants_grad({&y, &gates})) return Combine::apply(y, gates, slots, offsets);
  return combine_forward(y, gates, slots, offsets, y.scalar_type());
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("bind", &bind);
  m.def("layer_norm", &layer_norm);
  m.def("route", &route);
  m.def("grouped", &grouped);
  m.def("combine", &combine);
}
