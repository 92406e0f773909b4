// lact_b200::linear_attention_fwd / _bwd / _step (linear attention with a decay per head).
#include "common.h"

namespace lact_torch {
namespace {

// [b, l, h, d] with heads adjacent within a token and 16-byte aligned token / batch strides; anything else is copied
Tensor head_view(const Tensor& t) {
  const int64_t h = t.size(2), d = t.size(3);
  if (t.stride(3) != 1 || t.stride(2) != d || t.stride(1) % 8 || t.stride(0) % 8 || t.stride(1) < h * d ||
      (t.stride(0) == 0 && t.size(0) > 1) || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
    return plain(t);
  return t;
}

// [b, h, d] likewise
Tensor token_view(const Tensor& t) {
  if (t.stride(2) != 1 || t.stride(1) != t.size(2) || t.stride(0) % 8 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return plain(t);
  return t;
}

const float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
Tensor whole(const OptTensor& t) {
  if (!given(t)) return Tensor();
  Tensor c = t->contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

lact_linear_config config(const Tensor& q, const Tensor& k, const Tensor& v, double scale, const OptTensor& cu) {
  lact_linear_config c{};
  c.batch = q.size(0); c.tokens = q.size(1); c.heads = q.size(2); c.kv_heads = k.size(2);
  c.dk = q.size(3); c.dv = v.size(3);
  c.sequences = given(cu) ? cu->numel() - 1 : 0;
  c.q_ts = q.stride(1); c.q_bs = q.stride(0);
  c.k_ts = k.stride(1); c.k_bs = k.stride(0);
  c.v_ts = v.stride(1); c.v_bs = v.stride(0);
  c.scale = static_cast<float>(scale);
  return c;
}
int64_t states_of(const Tensor& q, const OptTensor& cu) { return given(cu) ? cu->numel() - 1 : q.size(0); }

// o, the last state with `want_state`, and with `keep` what the backward takes over of this call's workspace (the states that its
// pieces of sequences begin with)
std::vector<Tensor> fwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, double scale, const OptTensor& state_,
                        const OptTensor& cu, bool want_state, bool keep) {
  const c10::cuda::CUDAGuard guard(q_.device());
  const int64_t b = q_.size(0), l = q_.size(1), h = q_.size(2), dk = q_.size(3), dv = v_.size(3), n = states_of(q_, cu);
  const Tensor g = g_.contiguous(), state = whole(state_);
  Tensor o = empty({b, l, h, dv}, at::kBFloat16, q_), last, room;
  if (want_state) last = empty({n, h, dk, dv}, at::kFloat, q_);
  if (b * l == 0 || n == 0) {   // no tokens: the state stays what it was
    o.zero_();
    if (want_state) state.defined() ? last.copy_(state) : last.zero_();
  } else {
    const Tensor q = head_view(q_), k = head_view(k_), v = head_view(v_);
    const lact_linear_config c = config(q, k, v, scale, cu);
    size_t need = 0;
    check(lact_linear_attention_workspace_bytes(&c, 0, &need), "lact_linear_attention_workspace_bytes");
    if (need > 0) room = bytes(need, q);
    check(lact_linear_attention_fwd(&c, ptr(q), ptr(k), ptr(v), f32(g), static_cast<const int32_t*>(ptr(cu)), f32(state),
                                    want_state ? last.data_ptr<float>() : nullptr, ptr(o), need > 0 ? ptr(room) : nullptr, need,
                                    status_word(q), stream_of(q)),
          "lact_linear_attention_fwd");
  }
  std::vector<Tensor> r{o};
  if (want_state) r.push_back(last);
  if (keep) r.push_back(room.defined() ? room : empty({0}, at::kByte, q_));
  return r;
}

// dq, dk, dv, and the first state's gradient where there is a first state
std::vector<Tensor> bwd(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, double scale, const OptTensor& state_,
                        const OptTensor& cu, const Tensor& kept, const OptTensor& dout_, const OptTensor& dlast_) {
  const c10::cuda::CUDAGuard guard(q_.device());
  const int64_t b = q_.size(0), l = q_.size(1), h = q_.size(2), n = states_of(q_, cu);
  const Tensor g = g_.contiguous(), state = whole(state_);
  Tensor dlast;
  if (given(dlast_)) dlast = whole(dlast_->to(at::kFloat));
  Tensor dq = empty(q_.sizes(), at::kBFloat16, q_), dk = empty(k_.sizes(), at::kBFloat16, q_), dv = empty(v_.sizes(), at::kBFloat16, q_);
  std::vector<Tensor> r{dq, dk, dv};
  if (state.defined()) r.push_back(empty({n, h, q_.size(3), v_.size(3)}, at::kFloat, q_));
  if (b * l == 0 || n == 0) {
    for (int i = 0; i < 3; ++i) r[i].zero_();
    if (state.defined()) dlast.defined() ? r[3].copy_(dlast) : r[3].zero_();
    return r;
  }
  const Tensor q = head_view(q_), k = head_view(k_), v = head_view(v_);
  const Tensor dout = given(dout_) ? head_view(dout_->to(at::kBFloat16)) : at::zeros({b, l, h, v.size(3)}, dq.options());
  lact_linear_config c = config(q, k, v, scale, cu);
  c.do_ts = dout.stride(1); c.do_bs = dout.stride(0);
  size_t need = 0;
  check(lact_linear_attention_workspace_bytes(&c, 1, &need), "lact_linear_attention_workspace_bytes");
  Tensor room;
  if (need > 0) room = bytes(need, q);
  check(lact_linear_attention_bwd(&c, ptr(q), ptr(k), ptr(v), f32(g), static_cast<const int32_t*>(ptr(cu)), f32(state),
                                  kept.numel() > 0 ? ptr(kept) : nullptr, static_cast<size_t>(kept.numel()), ptr(dout), f32(dlast), ptr(dq), ptr(dk), ptr(dv), state.defined() ? r[3].data_ptr<float>() : nullptr,
                                  need > 0 ? ptr(room) : nullptr, need, status_word(q), stream_of(q)),
        "lact_linear_attention_bwd");
  settle(q);
  return r;
}

// One token of every sequence; `new_state` is `state` itself or an array apart from it.
Tensor step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, double scale, const Tensor& state, const Tensor& new_state) {
  const c10::cuda::CUDAGuard guard(q_.device());
  const char *from = static_cast<const char*>(ptr(state)), *to = static_cast<const char*>(ptr(new_state));
  const int64_t size = state.numel() * 4;
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(from) % 16 == 0 && reinterpret_cast<uintptr_t>(to) % 16 == 0,
                    "state and new_state must start on 16-byte boundaries");
  TORCH_CHECK_VALUE(from == to || from + size <= to || to + size <= from, "new_state overlaps state without being the same array");
  Tensor o = empty({q_.size(0), q_.size(1), v_.size(2)}, at::kBFloat16, q_);
  if (q_.size(0) == 0) return o;
  const Tensor q = token_view(q_), k = token_view(k_), v = token_view(v_), g = g_.contiguous();
  lact_linear_config c{};
  c.batch = q.size(0); c.tokens = 1; c.heads = q.size(1); c.kv_heads = k.size(1); c.dk = q.size(2); c.dv = v.size(2);
  c.q_bs = q.stride(0); c.q_ts = c.heads * c.dk;
  c.k_bs = k.stride(0); c.k_ts = c.kv_heads * c.dk;
  c.v_bs = v.stride(0); c.v_ts = c.kv_heads * c.dv;
  c.scale = static_cast<float>(scale);
  poll_status(q);
  check(lact_linear_attention_step(&c, ptr(q), ptr(k), ptr(v), f32(g), state.data_ptr<float>(), new_state.data_ptr<float>(), ptr(o),
                                   stream_of(q)),
        "lact_linear_attention_step");
  return o;
}

// The step as autograd sees it.  `new_state` gets a new version, so that a backward that has saved it (linear_attention saves its first
// state) raises in place of reading what is there now.  (PyTorch's own fallback for operators without a backward goes past the key that
// does this.  Tensors of inference mode have no version, and no backward can have saved them.)
using StepSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, double, const Tensor&, const Tensor&);
const auto& step_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::linear_attention_step", "").typed<StepSig>();
  return o;
}
Tensor step_versioned(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double scale,
                      const Tensor& state, const Tensor& new_state) {
  Tensor o;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    o = step_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, q, k, v, g, scale, state, new_state);
  }
  if (!new_state.is_inference()) torch::autograd::impl::bump_version(new_state);
  return o;
}
Tensor step_autograd(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double scale,
                     const Tensor& state, const Tensor& new_state) {
  no_tangents("linear_attention_step", {&q, &k, &v, &g, &state, &new_state});
  for (const Tensor* t : {&q, &k, &v, &g, &state, &new_state})
    TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t->requires_grad()), "linear_attention_step has no backward: use linear_attention");
  at::AutoDispatchBelowAutograd guard;
  return step_op().redispatch(keys & c10::after_autograd_keyset, q, k, v, g, scale, state, new_state);
}

using FwdSig = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, double, const OptTensor&, const OptTensor&, bool,
                                   bool);
using BwdSig = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, double, const OptTensor&, const OptTensor&,
                                   const Tensor&, const OptTensor&, const OptTensor&);
const auto& fwd_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::linear_attention_fwd", "").typed<FwdSig>();
  return o;
}
const auto& bwd_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::linear_attention_bwd", "").typed<BwdSig>();
  return o;
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double scale,
                               const OptTensor& state, const OptTensor& cu, bool want_state) {
    at::AutoDispatchBelowADInplaceOrView guard;
    variable_list r = fwd_op().call(q, k, v, g, scale, state, cu, want_state, true);
    ctx->save_for_backward({q, k, v, g, value(state), value(cu), r.back()});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    r.pop_back();
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    g.resize(2);
    if (!g[0].defined() && !g[1].defined()) return variable_list(8);
    const variable_list r = bwd_op().call(t[0], t[1], t[2], t[3], ctx->saved_data["scale"].toDouble(), opt(t[4]), opt(t[5]), t[6], opt(g[0]), opt(g[1]));
    return {r[0], r[1], r[2], Tensor(), Tensor(), r.size() > 3 ? r[3] : Tensor(), Tensor(), Tensor()};
  }
};
std::vector<Tensor> linear_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, double scale, const OptTensor& state,
                                    const OptTensor& cu, bool want_state, bool keep) {
  const Tensor first = value(state);
  no_tangents("linear_attention", {&q, &k, &v, &g, &first});
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK_NOT_IMPLEMENTED(!g.requires_grad(), "linear_attention has no gradient for log_decay");
    if (q.requires_grad() || k.requires_grad() || v.requires_grad() || first.requires_grad())
      return LinearFunction::apply(q, k, v, g, scale, state, cu, want_state);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return fwd_op().call(q, k, v, g, scale, state, cu, want_state, keep);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lact_b200, m) {
  m.def("linear_attention_fwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale, Tensor? state, Tensor? cu_seqlens, "
        "bool want_state, bool keep=False) -> Tensor[]");
  m.def("linear_attention_bwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale, Tensor? state, Tensor? cu_seqlens, "
        "Tensor kept, Tensor? dout, Tensor? dlast) -> Tensor[]");
  m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale, Tensor state, Tensor(a!) new_state) -> Tensor");
}
TORCH_LIBRARY_IMPL(lact_b200, CUDA, m) {
  m.impl("linear_attention_fwd", &fwd);
  m.impl("linear_attention_bwd", &bwd);
  m.impl("linear_attention_step", &step);
}
TORCH_LIBRARY_IMPL(lact_b200, ADInplaceOrView, m) { m.impl("linear_attention_step", &step_versioned); }
TORCH_LIBRARY_IMPL(lact_b200, Autograd, m) {
  m.impl("linear_attention_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_attention_step", &step_autograd);
  m.impl("linear_attention_fwd", &linear_autograd);
}

}  // namespace lact_torch
