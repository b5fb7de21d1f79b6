// The operators around the attention as PyTorch sees them (layer norm, the gated feed-forward block, dropout
// with the residual sum): schema, CUDA implementations and autograd.  Checks arguments, allocates outputs
// and workspaces and calls the C ABI, as torch_ops.cpp does for the attention.

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>

#include "torch_common.h"

namespace {

using at::Tensor;
using std::optional;
using trifast_torch::check_rc;
using trifast_torch::dtype_code;
using trifast_torch::raise_if_device_gave_up;
using trifast_torch::refuse_tangents;

// ------------------------------------------------------------------ arguments
void check_like(const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), " but x is on ", x.device(),
                    ": every tensor must live on the same CUDA device");
}
void check_cuda(const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "trifast_b200 runs on CUDA devices only (there is no CPU path)");
}

bool whole(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// A dense tensor on a 16-byte boundary.
Tensor dense(const Tensor& t) {
  return t.is_contiguous() && whole(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// All leading dimensions as one: rows at one distance, each contiguous, on a 16-byte boundary; anything
// else is copied.
struct Rows {
  Tensor t;
  int64_t rows, ld;
};
Rows dense_rows(const Tensor& t) {
  return {t.clone(at::MemoryFormat::Contiguous), t.numel() / t.size(-1), t.size(-1)};
}
Rows as_rows(const Tensor& t) {
  const int64_t width = t.size(-1), rows = t.numel() / width;
  int64_t ld = width, next = -1;   // next: what the stride of the next dimension outwards must be
  bool ok = whole(t) && (width == 1 || t.stride(-1) == 1);
  for (int64_t d = t.dim() - 2; d >= 0 && ok; --d) {
    if (t.size(d) == 1) continue;
    if (next < 0)
      ld = t.stride(d);
    else
      ok = t.stride(d) == next;
    next = t.stride(d) * t.size(d);
  }
  return ok && ld >= width ? Rows{t, rows, ld} : dense_rows(t);
}
// The same for layer norm, whose rows lie a multiple of 16 bytes beyond their width.
Rows as_norm_rows(const Tensor& t) {
  const Rows r = as_rows(t);
  return (r.ld - t.size(-1)) * t.element_size() % 16 == 0 ? r : dense_rows(t);
}

void* ptr(const Tensor& t) { return t.defined() ? const_cast<void*>(t.const_data_ptr()) : nullptr; }

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

template <typename Sig>
c10::TypedOperatorHandle<Sig> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor value(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

// ------------------------------------------------------------------ layer norm
trifast_norm check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be (..., width); got ", x.sizes());
  const int64_t width = x.size(-1);
  // (before it is held in 32 bits)
  TORCH_CHECK_VALUE(width <= 1 << 20, "width must be at most 1048576; got ", width);
  for (const auto& [name, t] : {std::pair{"weight", &weight}, std::pair{"bias", &bias}}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == width, name, " must be [", width, "]; got ", t->sizes());
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, name,
                     " must be float32 or of x's type");
    check_like(name, *t, x);
  }
  TORCH_CHECK_VALUE(!bias.defined() || weight.defined(), "a bias needs a weight");
  if (bias.defined())
    TORCH_CHECK_TYPE(bias.scalar_type() == weight.scalar_type(), "weight and bias must share one dtype");
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative; got ", eps);
  const int32_t dt = dtype_code(x.scalar_type());
  return {0, width, width, (int32_t)width, dt, weight.defined() ? dtype_code(weight.scalar_type()) : dt, (float)eps};
}

Tensor layer_norm_cuda(const Tensor& x, const optional<Tensor>& weight_, const optional<Tensor>& bias_, double eps) {
  Tensor weight = value(weight_), bias = value(bias_);
  trifast_norm n = check_norm(x, weight, bias, eps);
  check_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  raise_if_device_gave_up(x.device().index(), stream);
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return y;
  const Rows r = as_norm_rows(x);
  n.rows = r.rows;
  n.ld_x = r.ld;
  if (weight.defined()) weight = dense(weight);
  if (bias.defined()) bias = dense(bias);
  check_rc(trifast_layer_norm(&n, ptr(r.t), ptr(weight), ptr(bias), ptr(y), stream), "trifast_layer_norm");
  return y;
}

void check_upstream(const Tensor& dy, const Tensor& x, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(dy.sizes() == shape && dy.scalar_type() == x.scalar_type(), "dy must be ", shape, " ",
                    x.scalar_type(), "; got ", dy.sizes(), " ", dy.scalar_type());
  check_like("dy", dy, x);
}

// (a gradient that is not wanted comes back empty)
std::tuple<Tensor, Tensor, Tensor> layer_norm_grads_cuda(const Tensor& dy, const Tensor& x, const optional<Tensor>& weight_,
                                                         double eps, bool want_x, bool want_weight, bool want_bias) {
  Tensor weight = value(weight_);
  trifast_norm n = check_norm(x, weight, Tensor(), eps);
  check_upstream(dy, x, x.sizes());
  TORCH_CHECK_VALUE(weight.defined() || !(want_weight || want_bias), "without a weight there is no gradient for it");
  check_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  raise_if_device_gave_up(x.device().index(), stream);
  Tensor dx, dw, db;
  if (want_x) dx = at::empty(x.sizes(), x.options());
  if (want_weight) dw = at::empty({n.width}, weight.options());
  if (want_bias) db = at::empty({n.width}, weight.options());
  Rows rx{x, 0, n.width}, rdy{dy, 0, n.width};
  if (x.numel() != 0) {
    rx = as_norm_rows(x);
    rdy = as_norm_rows(dy);
  }
  n.rows = rx.rows;
  n.ld_x = rx.ld;
  n.ld_dy = rdy.ld;
  if (weight.defined()) weight = dense(weight);
  const size_t bytes = want_weight || want_bias ? trifast_layer_norm_workspace_bytes(&n) : 0;
  const Tensor ws = workspace(bytes, x);
  check_rc(trifast_layer_norm_backward(&n, ptr(rdy.t), ptr(rx.t), ptr(weight), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream),
           "trifast_layer_norm_backward");
  const auto out = [&](const Tensor& t) { return t.defined() ? t : at::empty({0}, x.options()); };
  return {out(dx), out(dw), out(db)};
}

using NormSig = Tensor(const Tensor&, const optional<Tensor>&, const optional<Tensor>&, double);
using NormGradsSig = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const optional<Tensor>&, double, bool, bool, bool);

Tensor call_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  static auto op = find_op<NormSig>("trifast_b200::layer_norm");
  return op.call(x, weight, bias, eps);
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, value(weight)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["bias"] = value(bias).defined();
    return call_norm(x, weight, bias, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = find_op<NormGradsSig>("trifast_b200::layer_norm_grads");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool has_w = s[1].defined(), has_b = ctx->saved_data["bias"].toBool();
    const bool wx = ctx->needs_input_grad(0), ww = has_w && ctx->needs_input_grad(1), wb = has_b && ctx->needs_input_grad(2);
    auto [dx, dw, db] = op.call(grads[0], s[0], maybe(s[1]), ctx->saved_data["eps"].toDouble(), wx, ww, wb);
    return {wx ? dx : Tensor(), ww ? dw : Tensor(), wb ? db : Tensor(), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  const Tensor w = value(weight), b = value(bias);
  refuse_tangents("layer_norm", {&x, &w, &b});
  if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, weight, bias, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm(x, weight, bias, eps);
}

// The gradients have no gradient of their own: asking for one is an error when it is reached.
class NormOnce : public torch::autograd::Function<NormOnce> {
 public:
  static variable_list forward(AutogradContext*, const Tensor& dy, const Tensor& x, const optional<Tensor>& weight, double eps,
                               bool wx, bool ww, bool wb) {
    static auto op = find_op<NormGradsSig>("trifast_b200::layer_norm_grads");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dx, dw, db] = op.call(dy, x, weight, eps, wx, ww, wb);
    return {dx, dw, db};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "trifast_b200::layer_norm_grads has no gradient formula: layer_norm can be differentiated once");
  }
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_grads_autograd(const Tensor& dy, const Tensor& x, const optional<Tensor>& weight,
                                                             double eps, bool wx, bool ww, bool wb) {
  static auto op = find_op<NormGradsSig>("trifast_b200::layer_norm_grads");
  const Tensor w = value(weight);
  refuse_tangents("layer_norm_grads", {&dy, &x, &w});
  if (wants_grad({&dy, &x, &w})) {
    const variable_list r = NormOnce::apply(dy, x, weight, eps, wx, ww, wb);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(dy, x, weight, eps, wx, ww, wb);
}

// ------------------------------------------------------------------ gated feed-forward block
trifast_ff check_ff(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be (..., width); got ", x.sizes());
  const int64_t width = x.size(-1);
  TORCH_CHECK_VALUE(wg.dim() == 2 && wg.size(1) == width && wg.size(0) >= 1, "w_gate must be (hidden, ", width, "); got ", wg.sizes());
  const int64_t hidden = wg.size(0);
  TORCH_CHECK_VALUE(wu.sizes() == wg.sizes(), "w_up must be ", wg.sizes(), "; got ", wu.sizes());
  TORCH_CHECK_VALUE(wd.dim() == 2 && wd.size(1) == hidden && wd.size(0) >= 1, "w_down must be (width_out, ", hidden, "); got ", wd.sizes());
  const auto dt = x.scalar_type();
  TORCH_CHECK_TYPE(wg.scalar_type() == dt && wu.scalar_type() == dt && wd.scalar_type() == dt,
                   "x, w_gate, w_up and w_down must share one dtype");
  for (const auto& [name, t] : {std::pair{"w_gate", &wg}, std::pair{"w_up", &wu}, std::pair{"w_down", &wd}})
    check_like(name, *t, x);
  const int32_t code = dtype_code(dt);
  TORCH_CHECK_VALUE(width <= 65536 && hidden <= 65536 && wd.size(0) <= 65536, "width, hidden and width_out must be at most 65536");
  return {0, width, wd.size(0), (int32_t)width, (int32_t)hidden, (int32_t)wd.size(0), code};
}

std::vector<int64_t> out_shape(const Tensor& x, int64_t width) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = width;
  return s;
}

Tensor feed_forward_cuda(const Tensor& x, const Tensor& wg_, const Tensor& wu_, const Tensor& wd_) {
  trifast_ff f = check_ff(x, wg_, wu_, wd_);
  check_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  raise_if_device_gave_up(x.device().index(), stream);
  Tensor y = at::empty(out_shape(x, f.width_out), x.options());
  if (x.numel() == 0) return y;
  const Rows r = as_rows(x);
  f.rows = r.rows;
  f.ld_x = r.ld;
  const Tensor wg = dense(wg_), wu = dense(wu_), wd = dense(wd_);
  const size_t bytes = trifast_feed_forward_workspace_bytes(&f);
  const Tensor ws = workspace(bytes, x);
  check_rc(trifast_feed_forward(&f, ptr(r.t), ptr(wg), ptr(wu), ptr(wd), ptr(y), ptr(ws), bytes, stream), "trifast_feed_forward");
  return y;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> feed_forward_grads_cuda(const Tensor& dy, const Tensor& x, const Tensor& wg_, const Tensor& wu_,
                                                                   const Tensor& wd_, bool want_x, bool want_weights) {
  trifast_ff f = check_ff(x, wg_, wu_, wd_);
  check_upstream(dy, x, out_shape(x, f.width_out));
  check_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  raise_if_device_gave_up(x.device().index(), stream);
  Tensor dx, dg, du, dd;
  if (want_x) dx = at::empty(x.sizes(), x.options());
  if (want_weights) {
    dg = at::empty(wg_.sizes(), x.options());
    du = at::empty(wu_.sizes(), x.options());
    dd = at::empty(wd_.sizes(), x.options());
  }
  Rows rx{x, 0, f.width}, rdy{dy, 0, f.width_out};
  if (x.numel() != 0) {
    rx = as_rows(x);
    rdy = as_rows(dy);
  }
  f.rows = rx.rows;
  f.ld_x = rx.ld;
  f.ld_dy = rdy.ld;
  const Tensor wg = dense(wg_), wu = dense(wu_), wd = dense(wd_);
  const size_t bytes = f.rows ? trifast_feed_forward_backward_workspace_bytes(&f) : 0;
  const Tensor ws = workspace(bytes, x);
  check_rc(trifast_feed_forward_backward(&f, ptr(rdy.t), ptr(rx.t), ptr(wg), ptr(wu), ptr(wd), ptr(dx), ptr(dg), ptr(du), ptr(dd),
                                         ptr(ws), bytes, stream),
           "trifast_feed_forward_backward");
  const auto out = [&](const Tensor& t) { return t.defined() ? t : at::empty({0}, x.options()); };
  return {out(dx), out(dg), out(du), out(dd)};
}

using FfSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&);
using FfGradsSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool, bool);

Tensor call_ff(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
  static auto op = find_op<FfSig>("trifast_b200::gated_feed_forward");
  return op.call(x, wg, wu, wd);
}

class FeedForward : public torch::autograd::Function<FeedForward> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, wg, wu, wd});
    return call_ff(x, wg, wu, wd);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static auto op = find_op<FfGradsSig>("trifast_b200::gated_feed_forward_grads");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool wx = ctx->needs_input_grad(0);
    const bool w[3] = {ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)};
    auto [dx, dg, du, dd] = op.call(grads[0], s[0], s[1], s[2], s[3], wx, w[0] || w[1] || w[2]);
    return {wx ? dx : Tensor(), w[0] ? dg : Tensor(), w[1] ? du : Tensor(), w[2] ? dd : Tensor()};
  }
};

Tensor feed_forward_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
  refuse_tangents("gated_feed_forward", {&x, &wg, &wu, &wd});
  if (wants_grad({&x, &wg, &wu, &wd})) return FeedForward::apply(x, wg, wu, wd);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_ff(x, wg, wu, wd);
}

class FfOnce : public torch::autograd::Function<FfOnce> {
 public:
  static variable_list forward(AutogradContext*, const Tensor& dy, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                               bool wx, bool ww) {
    static auto op = find_op<FfGradsSig>("trifast_b200::gated_feed_forward_grads");
    at::AutoDispatchBelowADInplaceOrView below;
    auto [a, b, c, d] = op.call(dy, x, wg, wu, wd, wx, ww);
    return {a, b, c, d};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "trifast_b200::gated_feed_forward_grads has no gradient formula: gated_feed_forward can be differentiated once");
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> feed_forward_grads_autograd(const Tensor& dy, const Tensor& x, const Tensor& wg, const Tensor& wu,
                                                                       const Tensor& wd, bool wx, bool ww) {
  static auto op = find_op<FfGradsSig>("trifast_b200::gated_feed_forward_grads");
  refuse_tangents("gated_feed_forward_grads", {&dy, &x, &wg, &wu, &wd});
  if (wants_grad({&dy, &x, &wg, &wu, &wd})) {
    const variable_list r = FfOnce::apply(dy, x, wg, wu, wd, wx, ww);
    return {r[0], r[1], r[2], r[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(dy, x, wg, wu, wd, wx, ww);
}

// ------------------------------------------------------------------ dropout with the residual sum
Tensor dropout_add_cuda(const Tensor& x_, const optional<Tensor>& residual_, double p, int64_t seed, int64_t offset,
                        const optional<Tensor>& seed_tensor_, optional<int64_t> shared_dim) {
  const Tensor residual0 = value(residual_), seed_tensor = value(seed_tensor_);
  TORCH_CHECK_VALUE(p >= 0 && p <= 1, "p must be in [0, 1]; got ", p);
  trifast_dropout d = {1, 1, x_.numel(), dtype_code(x_.scalar_type()), (uint64_t)seed, (uint64_t)offset, p};
  if (shared_dim.has_value()) {
    const int64_t nd = x_.dim(), at = *shared_dim < 0 ? *shared_dim + nd : *shared_dim;
    TORCH_CHECK_VALUE(at >= 0 && at < nd, "shared_dim ", *shared_dim, " is not a dimension of x, which has ", nd);
    d.inner = 1;
    for (int64_t i = 0; i < nd; ++i) (i < at ? d.outer : i == at ? d.mid : d.inner) *= x_.size(i);
  }
  if (residual0.defined()) {
    TORCH_CHECK_VALUE(residual0.sizes() == x_.sizes(), "residual must be ", x_.sizes(), "; got ", residual0.sizes());
    TORCH_CHECK_TYPE(residual0.scalar_type() == x_.scalar_type(), "x and residual must share one dtype");
    check_like("residual", residual0, x_);
  }
  if (seed_tensor.defined()) {
    TORCH_CHECK_TYPE(seed_tensor.scalar_type() == at::kLong, "a seed tensor must be int64");
    TORCH_CHECK_VALUE(seed_tensor.numel() == 1, "a seed tensor must have one element; got ", seed_tensor.sizes());
    check_like("seed", seed_tensor, x_);
  }
  check_cuda(x_);
  const c10::cuda::CUDAGuard guard(x_.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  raise_if_device_gave_up(x_.device().index(), stream);
  Tensor y = at::empty(x_.sizes(), x_.options());
  if (x_.numel() == 0) return y;
  const Tensor x = dense(x_), residual = residual0.defined() ? dense(residual0) : residual0;
  check_rc(trifast_dropout_add(&d, static_cast<const int64_t*>(ptr(seed_tensor)), ptr(x), ptr(residual), ptr(y), stream), "trifast_dropout_add");
  return y;
}

using DropoutSig = Tensor(const Tensor&, const optional<Tensor>&, double, int64_t, int64_t, const optional<Tensor>&, optional<int64_t>);

Tensor call_dropout(const Tensor& x, const optional<Tensor>& residual, double p, int64_t seed, int64_t offset,
                    const optional<Tensor>& seed_tensor, optional<int64_t> shared_dim) {
  static auto op = find_op<DropoutSig>("trifast_b200::dropout_add");
  return op.call(x, residual, p, seed, offset, seed_tensor, shared_dim);
}

class DropoutAdd : public torch::autograd::Function<DropoutAdd> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& residual, double p, int64_t seed, int64_t offset,
                        const optional<Tensor>& seed_tensor, optional<int64_t> shared_dim) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({value(seed_tensor)});
    ctx->saved_data["residual"] = value(residual).defined();
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["shared_dim"] = shared_dim;
    return call_dropout(x, residual, p, seed, offset, seed_tensor, shared_dim);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    // dx is the same operator on dy (and has itself as its gradient); the residual's gradient is dy
    if (ctx->needs_input_grad(0))
      out[0] = call_dropout(grads[0], std::nullopt, ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                            ctx->saved_data["offset"].toInt(), maybe(ctx->get_saved_variables()[0]),
                            ctx->saved_data["shared_dim"].toOptional<int64_t>());
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) out[1] = grads[0];
    return out;
  }
};

Tensor dropout_add_autograd(const Tensor& x, const optional<Tensor>& residual, double p, int64_t seed, int64_t offset,
                            const optional<Tensor>& seed_tensor, optional<int64_t> shared_dim) {
  const Tensor r = value(residual);
  refuse_tangents("dropout_add", {&x, &r});
  if (wants_grad({&x, &r})) return DropoutAdd::apply(x, residual, p, seed, offset, seed_tensor, shared_dim);
  at::AutoDispatchBelowADInplaceOrView below;
  return call_dropout(x, residual, p, seed, offset, seed_tensor, shared_dim);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(trifast_b200, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", {at::Tag::pt2_compliant_tag});
  m.def(
      "layer_norm_grads(Tensor dy, Tensor x, Tensor? weight, float eps, bool want_x, bool want_weight, bool want_bias) "
      "-> (Tensor, Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def("gated_feed_forward(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down) -> Tensor", {at::Tag::pt2_compliant_tag});
  m.def(
      "gated_feed_forward_grads(Tensor dy, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, bool want_x, bool want_weights) "
      "-> (Tensor, Tensor, Tensor, Tensor)",
      {at::Tag::pt2_compliant_tag});
  m.def(
      "dropout_add(Tensor x, Tensor? residual, float p, int seed, int offset, Tensor? seed_tensor, int? shared_dim) -> Tensor",
      {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(trifast_b200, CUDA, m) {
  m.impl("layer_norm", &layer_norm_cuda);
  m.impl("layer_norm_grads", &layer_norm_grads_cuda);
  m.impl("gated_feed_forward", &feed_forward_cuda);
  m.impl("gated_feed_forward_grads", &feed_forward_grads_cuda);
  m.impl("dropout_add", &dropout_add_cuda);
}
TORCH_LIBRARY_IMPL(trifast_b200, Autograd, m) {
  m.impl("layer_norm", &layer_norm_autograd);
  m.impl("layer_norm_grads", &layer_norm_grads_autograd);
  m.impl("gated_feed_forward", &feed_forward_autograd);
  m.impl("gated_feed_forward_grads", &feed_forward_grads_autograd);
  m.impl("dropout_add", &dropout_add_autograd);
}
