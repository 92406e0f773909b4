// lact_b200::rotary_axes (rotary positions with several axes for queries and keys).
#include "common.h"

namespace lact_torch {
namespace {

// q and, if given, k are [batch, tokens, heads, d] or [tokens, heads, d]
void check_args(const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq, at::IntArrayRef sections) {
  const int64_t dims = q.dim();
  TORCH_CHECK_VALUE(dims == 3 || dims == 4, "q: [batch, tokens, heads, head_dim] or [tokens, heads, head_dim]");
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat, "q: bf16 or float32");
  const int64_t d = q.size(dims - 1);
  TORCH_CHECK_VALUE(d >= 2 && d % 2 == 0 && d <= 512, "head_dim must be even, 512 at most");
  TORCH_CHECK_VALUE(q.size(dims - 2) > 0, "q has no heads");
  if (given(k)) {
    TORCH_CHECK_TYPE(k->scalar_type() == q.scalar_type(), "q and k must have the same dtype");
    TORCH_CHECK_VALUE(k->dim() == dims && k->size(dims - 1) == d && k->size(0) == q.size(0) && (dims == 3 || k->size(1) == q.size(1)) && k->size(dims - 2) > 0,
                      "k: as q but for the number of heads");
    TORCH_CHECK_VALUE(k->device() == q.device(), "all tensors must be on the same device");
  }
  TORCH_CHECK_VALUE(!sections.empty() && sections.size() <= LACT_ROTARY_AXES, "sections: pairs of each axis, ", LACT_ROTARY_AXES, " axes at most");
  int64_t pairs = 0;
  for (int64_t n : sections) {
    TORCH_CHECK_VALUE(n >= 0 && n <= d, "sections must not be negative, and not above half of head_dim together");
    pairs += n;
  }
  TORCH_CHECK_VALUE(pairs >= 1 && 2 * pairs <= d, "sections must have a pair, and not above half of head_dim together");
  TORCH_CHECK_TYPE(freq.scalar_type() == at::kDouble, "frequencies: float64");
  TORCH_CHECK_VALUE(freq.dim() == 1 && freq.size(0) == pairs, "frequencies: one for each pair of the sections");
  TORCH_CHECK_TYPE(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong, "positions: int32 or int64");
  const int64_t axes = static_cast<int64_t>(sections.size()), tokens = q.size(dims - 3);
  TORCH_CHECK_VALUE((pos.dim() == 2 || (pos.dim() == 3 && dims == 4 && (pos.size(0) == q.size(0) || pos.size(0) == 1))) && pos.size(-1) == axes &&
                        pos.size(-2) == tokens,
                    "positions: [tokens, axes], or [batch, tokens, axes] where q has a batch");
  TORCH_CHECK_VALUE(pos.device() == q.device() && freq.device() == q.device(), "all tensors must be on the same device");
}

std::vector<Tensor> turn(const Tensor& q_, const OptTensor& k_, const Tensor& pos, const Tensor& freq_, at::IntArrayRef sections, bool interleaved,
                         bool backwards) {
  check_args(q_, k_, pos, freq_, sections);
  const c10::cuda::CUDAGuard guard(q_.device());
  const int64_t dims = q_.dim();
  const bool pair = given(k_);
  std::vector<Tensor> out{empty(q_.sizes(), q_.scalar_type(), q_)};
  if (pair) out.push_back(empty(k_->sizes(), q_.scalar_type(), q_));
  if (q_.numel() == 0) return out;
  const Tensor q = q_.stride(dims - 1) == 1 ? q_ : q_.contiguous(), k = !pair ? Tensor() : k_->stride(dims - 1) == 1 ? *k_ : k_->contiguous();
  const Tensor freq = freq_.contiguous();
  lact_rotary_config c{};
  c.batch = dims == 4 ? q.size(0) : 1;
  c.tokens = q.size(dims - 3);
  c.head_dim = q.size(dims - 1);
  c.q_heads = q.size(dims - 2);
  c.q_bs = dims == 4 ? q.stride(0) : 0; c.q_ts = q.stride(dims - 3); c.q_hs = q.stride(dims - 2);
  if (pair) {
    c.k_heads = k.size(dims - 2);
    c.k_bs = dims == 4 ? k.stride(0) : 0; c.k_ts = k.stride(dims - 3); c.k_hs = k.stride(dims - 2);
  }
  c.position_bs = pos.dim() == 3 && pos.size(0) > 1 ? pos.stride(0) : 0;
  c.position_ts = pos.stride(-2); c.position_as = pos.stride(-1);
  c.position_bytes = static_cast<int32_t>(pos.element_size());
  c.axes = static_cast<int32_t>(sections.size());
  for (size_t i = 0; i < sections.size(); ++i) c.sections[i] = sections[i];
  c.dtype = dtype_code(q);
  c.interleaved = interleaved;
  c.backwards = backwards;
  poll_status(q);
  check(lact_rotary_axes(&c, ptr(q), pair ? ptr(k) : nullptr, ptr(pos), freq.data_ptr<double>(), ptr(out[0]), pair ? ptr(out[1]) : nullptr, stream_of(q)),
        "lact_rotary_axes");
  if (backwards) settle(q);
  return out;
}
std::vector<Tensor> turn_cpu(const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq, at::IntArrayRef sections, bool, bool) {
  check_args(q, k, pos, freq, sections);
  TORCH_CHECK_VALUE(false, "rotary_axes needs CUDA tensors (there is no CPU implementation)");
}

using Sig = std::vector<Tensor>(const Tensor&, const OptTensor&, const Tensor&, const Tensor&, at::IntArrayRef, bool, bool);
const auto& op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::rotary_axes", "").typed<Sig>();
  return o;
}

// The gradient is the same operator turning the other way, so it has gradients in its turn.
class RotaryFunction : public torch::autograd::Function<RotaryFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq,
                               std::vector<int64_t> sections, bool interleaved, bool backwards) {
    at::AutoDispatchBelowADInplaceOrView guard;
    variable_list r = op().call(q, k, pos, freq, sections, interleaved, backwards);
    ctx->save_for_backward({pos, freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["backwards"] = backwards;
    ctx->saved_data["dtype"] = static_cast<int64_t>(q.scalar_type());
    ctx->set_materialize_grads(false);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto t = ctx->get_saved_variables();
    variable_list out(7);
    const auto dtype = static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt());
    std::vector<int> which;
    for (int i = 0; i < 2; ++i)
      if (i < static_cast<int>(g.size()) && g[i].defined() && ctx->needs_input_grad(i)) which.push_back(i);
    if (which.empty()) return out;
    const Tensor first = g[which[0]].to(dtype);
    const OptTensor second = which.size() > 1 ? OptTensor(g[which[1]].to(dtype)) : OptTensor();
    const auto r = op().call(first, second, t[0], t[1], ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(),
                             !ctx->saved_data["backwards"].toBool());
    for (size_t i = 0; i < which.size(); ++i) out[which[i]] = r[i];
    return out;
  }
};
std::vector<Tensor> turn_autograd(const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq, at::IntArrayRef sections, bool interleaved,
                                  bool backwards) {
  const Tensor key = value(k);
  no_tangents("rotary_axes", {&q, &key, &freq});
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK_NOT_IMPLEMENTED(!freq.requires_grad(), "rotary_axes has no gradient for the frequencies");
    if (q.requires_grad() || (key.defined() && key.requires_grad())) return RotaryFunction::apply(q, k, pos, freq, sections.vec(), interleaved, backwards);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  return op().call(q, k, pos, freq, sections, interleaved, backwards);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lact_b200, m) {
  m.def("rotary_axes(Tensor q, Tensor? k, Tensor positions, Tensor frequencies, int[] sections, bool interleaved, bool backwards=False) -> Tensor[]");
}
TORCH_LIBRARY_IMPL(lact_b200, CUDA, m) { m.impl("rotary_axes", &turn); }
TORCH_LIBRARY_IMPL(lact_b200, CPU, m) { m.impl("rotary_axes", &turn_cpu); }
TORCH_LIBRARY_IMPL(lact_b200, Autograd, m) { m.impl("rotary_axes", &turn_autograd); }

}  // namespace lact_torch
