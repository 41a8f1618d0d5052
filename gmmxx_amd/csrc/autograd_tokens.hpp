// The token operators' autograd functions (see autograd.cpp).  Arguments have been checked by
// gmmxx_amd/tokens.py: matrices with adjacent row elements, matching shapes, types and devices.
#pragma once

#include "autograd.hpp"

namespace {

int index_bits(const Tensor& index) { return 8 * (int)index.element_size(); }

// --- embedding ------------------------------------------------------------------

Tensor embed_forward(const Tensor& table, const Tensor& index, double scale) {
  const int64_t n = index.size(0), v = table.size(0), d = table.size(1);
  Tensor out = at::empty({n, d}, table.options());
  if (n == 0) return out;
  On on(table);
  check(lib.embed(elem(table), n, v, d, ptr(table), table.stride(0), ptr(index), index_bits(index), scale, ptr(out),
                  on.stream()),
        "embed");
  return out;
}

struct Embed : torch::autograd::Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& index, double scale) {
    ctx->save_for_backward({index});
    ctx->saved_data["v"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    return embed_forward(table, index, scale);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor& index = saved[0];
    const Tensor dy = rows_of(grads[0]);
    const int64_t n = dy.size(0), d = dy.size(1), v = ctx->saved_data["v"].toInt();
    Tensor dtable = n ? at::empty({v, d}, dy.options()) : at::zeros({v, d}, dy.options());
    if (n) {
      On on(dy);
      const int64_t need = lib.embed_workspace_bytes(n, v, d);
      const Tensor ws = bytes(need, dy);
      check(lib.embed_backward(elem(dy), n, v, d, ptr(dy), dy.stride(0), ptr(index), index_bits(index),
                               ctx->saved_data["scale"].toDouble(), ptr(dtable), ptr(ws), need, on.stream()),
            "embed_backward");
    }
    return once({dtable, Tensor(), Tensor()});
  }
};

Tensor embed(const Tensor& table0, const Tensor& index, double scale) {
  const Tensor table = plain(table0);
  if (wants_grad({&table})) return Embed::apply(table, index, scale);
  return embed_forward(table, index, scale);
}

// --- dropout --------------------------------------------------------------------

Tensor drop(const Tensor& x, const Tensor& residual, double p, int64_t seed, const Tensor& seed_at, int64_t offset) {
  Tensor out = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return out;
  On on(x);
  check(lib.dropout(elem(x), x.numel(), p, (uint64_t)seed, static_cast<int64_t*>(ptr(seed_at)), (uint64_t)offset,
                    ptr(x), ptr(residual), ptr(out), on.stream()),
        "dropout");
  return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual, double p,
                        int64_t seed, const std::optional<Tensor>& seed_at, int64_t offset) {
    ctx->save_for_backward({or_none(seed_at)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = residual.has_value();
    return drop(x, or_none(residual), p, seed, or_none(seed_at), offset);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    Tensor dx, dresidual;
    if (ctx->needs_input_grad(0))
      dx = drop(plain(grads[0]).contiguous(), Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                saved[0], ctx->saved_data["offset"].toInt());
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) dresidual = grads[0];
    return once({dx, dresidual, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor& x0, const std::optional<Tensor>& residual0, double p, int64_t seed,
               const std::optional<Tensor>& seed_at, int64_t offset) {
  const Tensor x = plain(x0);
  const std::optional<Tensor> residual = plain(residual0);
  const Tensor r = or_none(residual);
  if (wants_grad({&x, &r})) return Dropout::apply(x, residual, p, seed, seed_at, offset);
  return drop(x, r, p, seed, or_none(seed_at), offset);
}

// --- log probabilities ----------------------------------------------------------

// chosen, entropy, top, top_index and, if wanted, what the backward pass reads.
variable_list log_probs_forward(const Tensor& scores, const Tensor& index, int64_t k, bool want_stats) {
  const int64_t n = scores.size(0), v = scores.size(1);
  const auto f32 = scores.options().dtype(at::kFloat);
  Tensor chosen = at::empty({n}, f32), entropy = at::empty({n}, f32), top = at::empty({n, k}, f32);
  Tensor top_index = at::empty({n, k}, scores.options().dtype(at::kInt));
  Tensor stats = want_stats ? at::empty({n, 3}, f32) : Tensor();
  if (n) {
    On on(scores);
    const int64_t need = lib.log_probs_workspace_bytes(n, v, k);
    const Tensor ws = need ? bytes(need, scores) : Tensor();
    check(lib.log_probs(elem(scores), n, v, k, ptr(scores), scores.stride(0), ptr(index), index_bits(index),
                        floats(chosen), floats(entropy), floats(top), ints(top_index), floats(stats), ptr(ws), need,
                        on.stream()),
          "log_probs");
  }
  return {chosen, entropy, top, top_index, stats};
}

struct LogProbs : torch::autograd::Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& scores, const Tensor& index, int64_t k) {
    variable_list out = log_probs_forward(scores, index, k, true);
    ctx->save_for_backward({scores, index, out[3], out[4]});
    out.pop_back();
    ctx->mark_non_differentiable({out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse({&grads[0], &grads[1], &grads[2]});
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &scores = saved[0], &index = saved[1], &top_index = saved[2], &stats = saved[3];
    const int64_t n = scores.size(0), v = scores.size(1);
    Tensor ds = at::empty({n, v}, scores.options()), g[3];
    if (n) {
      for (int i = 0; i < 3; ++i)
        if (grads[i].defined()) g[i] = plain(grads[i]).contiguous();
      On on(scores);
      check(lib.log_probs_backward(elem(scores), n, v, top_index.size(1), ptr(scores), scores.stride(0), ptr(index),
                                   index_bits(index), ints(top_index), floats(stats), floats(g[0]), floats(g[1]),
                                   floats(g[2]), ptr(ds), on.stream()),
            "log_probs_backward");
    }
    return once({ds, Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> log_probs(const Tensor& scores0, const Tensor& index, int64_t k) {
  const Tensor scores = plain(scores0);
  const variable_list r =
      wants_grad({&scores}) ? LogProbs::apply(scores, index, k) : log_probs_forward(scores, index, k, false);
  return {r[0], r[1], r[2], r[3]};
}

// --- products in 8-bit integers ---------------------------------------------------

constexpr int64_t kPad = 128;      // rows of values take whole cache lines

void no_gradient(std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad(ts), "gmmxx_amd's 8-bit products have no gradient: call them under "
                                               "torch.no_grad() or on detached tensors");
}

std::tuple<Tensor, Tensor> quantize_forward(const Tensor& x) {
  const int64_t n = x.size(0), d = x.size(1), room = (d + kPad - 1) / kPad * kPad;
  const Tensor values = at::empty({n, room}, x.options().dtype(at::kChar));
  const Tensor scales = at::empty({n}, x.options().dtype(at::kFloat));
  if (n) {
    On on(x);
    check(lib.quantize(elem(x), n, d, ptr(x), x.stride(0), static_cast<int8_t*>(ptr(values)), room, floats(scales),
                       on.stream()),
          "quantize");
  }
  return {values.narrow(1, 0, d), scales};
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x0) {
  const Tensor x = plain(x0);
  no_gradient({&x});
  return quantize_forward(x);
}

// A matrix of values as the product reads it: rows of whole, aligned 16 bytes; itself or a copy.
Tensor whole_rows(const Tensor& t) {
  const int64_t n = t.size(0), d = t.size(1), whole = (d + 15) / 16 * 16;
  const int64_t ld = n > 1 ? t.stride(0) : whole;
  const int64_t room = (int64_t)t.storage().nbytes() - t.storage_offset();
  if ((d == 1 || t.stride(1) == 1) && ld % 16 == 0 && ld <= (1 << 23) && reinterpret_cast<uintptr_t>(ptr(t)) % 16 == 0 &&
      (n - 1) * ld + whole <= room)
    return t;
  Tensor copy = at::empty({n, (d + kPad - 1) / kPad * kPad}, t.options()).narrow(1, 0, d);
  copy.copy_(t);
  return copy;
}

Tensor quantized_matmul(const Tensor& x0, const std::optional<Tensor>& xscales, const Tensor& w0, const Tensor& wscales,
                        const std::optional<Tensor>& bias0, at::ScalarType type) {
  const Tensor x = plain(x0), xs0 = or_none(xscales), bias = or_none(plain(bias0));
  no_gradient({&x, &xs0, &wscales, &bias});
  const int64_t n = x.size(0), d = x.size(1), f = w0.size(0);
  Tensor out = at::empty({n, f}, x.options().dtype(type));
  if (n == 0) return out;
  On on(x);
  const Tensor w = whole_rows(w0);
  const int64_t whole = (d + 15) / 16 * 16, ldw = f > 1 ? w.stride(0) : whole;
  const int8_t* wp = static_cast<int8_t*>(ptr(w));
  if (!xs0.defined()) {
    const int64_t need = lib.quantized_linear_workspace_bytes(elem(x), n, d);
    const Tensor ws = need ? bytes(need, x) : Tensor();
    check(lib.quantized_linear(elem(x), elem(type), n, f, d, ptr(x), x.stride(0), wp, ldw, floats(plain(wscales)),
                               ptr(bias), ptr(out), ptr(ws), need, on.stream()),
          "quantized_linear");
    return out;
  }
  const Tensor values = whole_rows(x);
  check(lib.quantized_matmul(elem(type), n, f, d, static_cast<int8_t*>(ptr(values)), n > 1 ? values.stride(0) : whole,
                             floats(plain(xs0)), wp, ldw, floats(plain(wscales)), ptr(bias), ptr(out), on.stream()),
        "quantized_matmul");
  return out;
}

}  // namespace
