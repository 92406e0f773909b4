// lact_b200::group_norm_fwd / _bwd (group norm with an activation, channels last).
#include "common.h"

namespace lact_torch {
namespace {

// [n, s, C] with adjacent channels, rows that do not overlap, and strides and base that whole accesses of up to 16 bytes fit; anything
// else is copied
Tensor rows_of(const Tensor& t) {
  int64_t w = 16 / t.element_size();
  while (t.size(2) % w) w /= 2;
  const bool spots = t.size(1) > 1, samples = t.size(0) > 1;
  if (t.stride(2) == 1 && !(spots && (t.stride(1) < t.size(2) || t.stride(1) % w)) && !(samples && (t.stride(0) < t.size(2) || t.stride(0) % w)) &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % (w * t.element_size()) == 0)
    return t;
  Tensor c = t.contiguous();   // (a contiguous view off its alignment is returned as it is)
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
Tensor weights_of(const OptTensor& t) { return given(t) ? t->to(at::kFloat).contiguous() : Tensor(); }
const float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

lact_group_norm_config config(const Tensor& x, int64_t groups, double eps, bool silu) {
  lact_group_norm_config c{};
  c.n = x.size(0); c.s = x.size(1); c.channels = x.size(2); c.groups = groups;
  c.x_ns = c.n > 1 ? x.stride(0) : 0; c.x_ss = c.s > 1 ? x.stride(1) : 0;
  c.dtype = dtype_code(x);
  c.silu = silu;
  c.eps = static_cast<float>(eps);
  return c;
}

// [n, ..., C] as [n, s, C]
Tensor three(const Tensor& t) { return t.dim() == 3 ? t : t.dim() == 2 ? t.unsqueeze(1) : t.flatten(1, -2); }

// y and the statistics
std::vector<Tensor> fwd(const Tensor& x_, const OptTensor& w_, const OptTensor& b_, int64_t groups, double eps, bool silu) {
  const c10::cuda::CUDAGuard guard(x_.device());
  Tensor y = empty(x_.sizes(), x_.scalar_type(), x_), stats = empty({x_.size(0), groups, 2}, at::kFloat, x_);
  if (x_.numel() == 0) return {y, stats.zero_()};
  const Tensor x = rows_of(three(x_)), w = weights_of(w_), b = weights_of(b_);
  const lact_group_norm_config c = config(x, groups, eps, silu);
  size_t need = 0;
  check(lact_group_norm_workspace_bytes(&c, 0, &need), "lact_group_norm_workspace_bytes");
  Tensor room;
  if (need > 0) room = bytes(need, x);
  poll_status(x);
  check(lact_group_norm_fwd(&c, ptr(x), f32(w), f32(b), ptr(y), stats.data_ptr<float>(), need > 0 ? ptr(room) : nullptr, need, stream_of(x)),
        "lact_group_norm_fwd");
  return {y, stats};
}

// dx, dw, db
std::vector<Tensor> bwd(const Tensor& x_, const OptTensor& w_, const OptTensor& b_, const Tensor& stats_, const Tensor& dy_, int64_t groups,
                        double eps, bool silu) {
  const c10::cuda::CUDAGuard guard(x_.device());
  Tensor dx = empty(x_.sizes(), x_.scalar_type(), x_), dw = empty({x_.size(-1)}, at::kFloat, x_), db = at::empty_like(dw);
  if (x_.numel() == 0) return {dx, dw.zero_(), db.zero_()};
  const Tensor x = rows_of(three(x_)), dy = rows_of(three(dy_.to(x_.scalar_type()))), w = weights_of(w_), b = weights_of(b_), stats = stats_.contiguous();
  lact_group_norm_config c = config(x, groups, eps, silu);
  c.dy_ns = c.n > 1 ? dy.stride(0) : 0;
  c.dy_ss = c.s > 1 ? dy.stride(1) : 0;
  size_t need = 0;
  check(lact_group_norm_workspace_bytes(&c, 1, &need), "lact_group_norm_workspace_bytes");
  Tensor room;
  if (need > 0) room = bytes(need, x);
  poll_status(x);
  check(lact_group_norm_bwd(&c, ptr(x), f32(w), f32(b), stats.data_ptr<float>(), ptr(dy), ptr(dx), dw.data_ptr<float>(),
                            db.data_ptr<float>(), need > 0 ? ptr(room) : nullptr, need, stream_of(x)),
        "lact_group_norm_bwd");
  settle(x);
  return {dx, dw, db};
}

using FwdSig = std::vector<Tensor>(const Tensor&, const OptTensor&, const OptTensor&, int64_t, double, bool);
using BwdSig = std::vector<Tensor>(const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, int64_t, double, bool);
const auto& fwd_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::group_norm_fwd", "").typed<FwdSig>();
  return o;
}
const auto& bwd_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::group_norm_bwd", "").typed<BwdSig>();
  return o;
}

class NormFunction : public torch::autograd::Function<NormFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t groups, double eps,
                               bool silu) {
    at::AutoDispatchBelowADInplaceOrView guard;
    variable_list r = fwd_op().call(x, w, b, groups, eps, silu);
    ctx->save_for_backward({x, value(w), value(b), r[1]});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r[1]});
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(6);
    const auto r = bwd_op().call(t[0], opt(t[1]), opt(t[2]), t[3], g[0], ctx->saved_data["groups"].toInt(),
                                 ctx->saved_data["eps"].toDouble(), ctx->saved_data["silu"].toBool());
    auto as = [&](const Tensor& like, const Tensor& g) { return like.defined() ? g.to(like.scalar_type()) : Tensor(); };
    return {r[0], as(t[1], r[1]), as(t[2], r[2]), Tensor(), Tensor(), Tensor()};
  }
};
std::vector<Tensor> norm_autograd(const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t groups, double eps, bool silu) {
  const Tensor weight = value(w), bias = value(b);
  no_tangents("group_norm", {&x, &weight, &bias});
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || bias.requires_grad()))
    return NormFunction::apply(x, w, b, groups, eps, silu);
  at::AutoDispatchBelowADInplaceOrView guard;
  return fwd_op().call(x, w, b, groups, eps, silu);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lact_b200, m) {
  m.def("group_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, int groups, float eps, bool silu) -> Tensor[]");
  m.def("group_norm_bwd(Tensor x, Tensor? weight, Tensor? bias, Tensor stats, Tensor dy, int groups, float eps, bool silu) -> Tensor[]");
}
TORCH_LIBRARY_IMPL(lact_b200, CUDA, m) {
  m.impl("group_norm_fwd", &fwd);
  m.impl("group_norm_bwd", &bwd);
}
TORCH_LIBRARY_IMPL(lact_b200, Autograd, m) {
  m.impl("group_norm_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("group_norm_fwd", &norm_autograd);
}

}  // namespace lact_torch
