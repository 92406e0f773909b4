// lact_b200::paged_cache_write / paged_cache_read / paged_attention_step (a paged cache of keys and values).
#include "common.h"

namespace lact_torch {
namespace {

bool whole_number(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

// [pages, heads, page_size, ..]: pages contiguous in themselves (axes of one entry may have any stride)
bool whole_pages(const Tensor& t) {
  int64_t n = 1;
  for (int64_t i = t.dim() - 1; i > 0; --i) {
    if (t.size(i) > 1 && t.stride(i) != n) return false;
    n *= t.size(i);
  }
  return t.size(0) <= 1 || t.stride(0) >= n;
}

void check_cache(const char* what, const Tensor& k, const Tensor& v, const OptTensor& ke, const OptTensor& ve, const Tensor& table, const Tensor& lengths) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(), "the cache's k and v: [pages, kv_heads, page_size, head_dim] both");
  TORCH_CHECK_VALUE(given(ke) == given(ve), "exponents: of k and of v, or of neither");
  const auto type = given(ke) ? at::kFloat8_e4m3fn : at::kBFloat16;
  TORCH_CHECK_TYPE(k.scalar_type() == type && v.scalar_type() == type, "the cache's k and v: bf16, or float8_e4m3fn with exponents");
  TORCH_CHECK_VALUE(k.size(3) == 64 || k.size(3) == 128, "head_dim must be 64 or 128");
  const int64_t page = k.size(2);
  TORCH_CHECK_VALUE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256");
  TORCH_CHECK_VALUE(k.size(0) > 0 && k.size(1) > 0, "the cache has no pages or no heads");
  TORCH_CHECK_VALUE(whole_pages(k) && whole_pages(v), "the cache's pages must be contiguous: they are read and written where they lie");
  if (given(ke)) {
    for (const Tensor* t : {&*ke, &*ve}) {
      TORCH_CHECK_TYPE(t->scalar_type() == at::kByte, "exponents: uint8");
      TORCH_CHECK_VALUE(t->dim() == 3 && t->sizes() == k.sizes().slice(0, 3) && whole_pages(*t), "exponents: [pages, kv_heads, page_size], pages contiguous");
      TORCH_CHECK_VALUE(t->device() == k.device(), "all tensors must be on the same device");
    }
  }
  TORCH_CHECK_TYPE(whole_number(table) && whole_number(lengths), "page_table, lengths: whole numbers (int32)");
  TORCH_CHECK_VALUE(table.dim() == 2 && lengths.dim() == 1 && table.size(0) == lengths.size(0) && (table.size(1) > 0 || table.size(0) == 0),
                    "page_table: [sequences, pages of the longest], lengths: [sequences]");
  TORCH_CHECK_VALUE(v.device() == k.device() && table.device() == k.device() && lengths.device() == k.device(), "all tensors must be on the same device");
  TORCH_CHECK_VALUE(!k.is_cpu(), what, " needs CUDA tensors (there is no CPU implementation)");
}

// Whole numbers as the kernels read them: what 31 bits do not hold stays past every end
Tensor as_int(const Tensor& t) { return t.scalar_type() == at::kInt ? t : t.clamp(-1, INT32_MAX).to(at::kInt); }

// What a call keeps alive of its arguments, and the description of the cache.
struct Cache {
  lact_paged_cache c{};
  Tensor table, lengths;
};
Cache describe(const Tensor& k, const Tensor& v, const OptTensor& ke, const OptTensor& ve, const Tensor& table, const Tensor& lengths) {
  Cache r;
  r.table = as_int(table);
  if (r.table.size(1) > 1 && r.table.stride(1) != 1) r.table = r.table.contiguous();
  r.lengths = as_int(lengths).contiguous();
  r.c.k = ptr(k); r.c.v = ptr(v);
  r.c.k_exponent = ptr(ke); r.c.v_exponent = ptr(ve);
  r.c.pages = k.size(0); r.c.kv_heads = k.size(1); r.c.page_size = k.size(2); r.c.head_dim = k.size(3);
  r.c.k_page_stride = k.stride(0); r.c.v_page_stride = v.stride(0);
  if (given(ke)) {
    r.c.ke_page_stride = ke->stride(0);
    r.c.ve_page_stride = ve->stride(0);
  }
  r.c.page_table = r.table.data_ptr<int32_t>();
  r.c.table_cols = r.table.size(1);
  r.c.table_stride = r.table.size(0) > 1 ? r.table.stride(0) : 0;
  r.c.lengths = r.lengths.data_ptr<int32_t>();
  r.c.sequences = r.lengths.size(0);
  return r;
}

// Bounds of packed sequences as the kernels read them
Tensor bounds(const OptTensor& cu, int64_t sequences, int64_t batch, const Tensor& like) {
  if (!given(cu)) {
    TORCH_CHECK_VALUE(batch == sequences, "a batch entry for each sequence of the page table, or packed sequences (cu_seqlens)");
    return Tensor();
  }
  TORCH_CHECK_VALUE(batch == 1, "packed sequences (cu_seqlens) need a batch of one");
  TORCH_CHECK_TYPE(whole_number(*cu), "cu_seqlens: whole numbers");
  TORCH_CHECK_VALUE(cu->dim() == 1 && cu->size(0) == sequences + 1, "cu_seqlens: [sequences + 1]");
  TORCH_CHECK_VALUE(cu->device() == like.device(), "all tensors must be on the same device");
  return as_int(*cu).contiguous();
}

// The addresses that a tensor's elements lie between
std::pair<uintptr_t, uintptr_t> extent(const Tensor& t) {
  int64_t far = 0;
  for (int64_t i = 0; i < t.dim(); ++i) far += (t.size(i) - 1) * t.stride(i);
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {at, at + static_cast<uintptr_t>((far + 1) * t.element_size())};
}

// [b, l, h, d] with adjacent features and 16-byte aligned rows; anything else is copied
Tensor rows_of(const Tensor& t) {
  bool fine = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) fine = fine && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return fine ? t : plain(t);
}
int64_t stride_of(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }

void write(const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& k_, const Tensor& v_, const Tensor& table,
           const Tensor& lengths, const OptTensor& cu_) {
  TORCH_CHECK_TYPE(k_.scalar_type() == at::kBFloat16 && v_.scalar_type() == at::kBFloat16, "k, v: bf16 activations");
  TORCH_CHECK_VALUE(k_.dim() == 4 && v_.sizes() == k_.sizes(), "k, v: [batch, tokens, kv_heads, head_dim] both");
  TORCH_CHECK_VALUE(kc.dim() == 4 && k_.size(2) == kc.size(1) && k_.size(3) == kc.size(3), "k, v: kv_heads and head_dim of the cache");
  TORCH_CHECK_VALUE(k_.device() == kc.device() && v_.device() == kc.device(), "all tensors must be on the same device");
  const Tensor cu = bounds(cu_, lengths.dim() == 1 ? lengths.size(0) : -1, k_.size(0), kc);
  check_cache("paged_cache_write", kc, vc, ke, ve, table, lengths);
  const c10::cuda::CUDAGuard guard(kc.device());
  if (k_.numel() == 0 || lengths.size(0) == 0) return;
  const auto a = extent(kc), b = extent(vc);
  for (const Tensor* t : {&k_, &v_}) {
    const auto x = extent(*t);
    TORCH_CHECK_VALUE((x.second <= a.first || a.second <= x.first) && (x.second <= b.first || b.second <= x.first), "k, v lie within the cache that they are written to");
  }
  TORCH_CHECK_VALUE(ptr(kc) != ptr(vc) && (!given(ke) || ptr(ke) != ptr(ve)), "the cache's k and v are the same array");
  const Tensor k = rows_of(k_), v = rows_of(v_);
  const Cache r = describe(kc, vc, ke, ve, table, lengths);
  poll_status(kc);
  check(lact_paged_cache_write(&r.c, ptr(k), stride_of(k, 1), stride_of(k, 0), stride_of(k, 2), ptr(v), stride_of(v, 1), stride_of(v, 0), stride_of(v, 2),
                               k.size(0), k.size(1), cu.defined() ? cu.data_ptr<int32_t>() : nullptr, stream_of(kc)),
        "lact_paged_cache_write");
}

Tensor read(const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& table, const Tensor& lengths, int64_t tokens,
            const OptTensor& cu_) {
  TORCH_CHECK_VALUE(tokens >= 0, "num_tokens must not be negative");
  const int64_t batch = given(cu_) ? 1 : lengths.dim() == 1 ? lengths.size(0) : 0;
  const Tensor cu = bounds(cu_, lengths.dim() == 1 ? lengths.size(0) : -1, batch, kc);
  check_cache("paged_cache_read", kc, vc, ke, ve, table, lengths);
  const c10::cuda::CUDAGuard guard(kc.device());
  Tensor out = empty({2 * batch, tokens, kc.size(1), kc.size(3)}, at::kBFloat16, kc);
  if (out.numel() == 0) return out;
  if (lengths.size(0) == 0) return out.zero_();
  const Cache r = describe(kc, vc, ke, ve, table, lengths);
  poll_status(kc);
  check(lact_paged_cache_read(&r.c, ptr(out), batch, tokens, cu.defined() ? cu.data_ptr<int32_t>() : nullptr, stream_of(kc)), "lact_paged_cache_read");
  return out;
}

Tensor step(const Tensor& q_, const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& table, const Tensor& lengths,
            int64_t window, double scale) {
  TORCH_CHECK_VALUE(q_.dim() == 3, "q: [sequences, heads, head_dim]");
  TORCH_CHECK_TYPE(q_.scalar_type() == at::kBFloat16, "q: bf16 activations");
  TORCH_CHECK_VALUE(window >= 0, "window_size must not be negative");
  TORCH_CHECK_VALUE(std::fabs(scale) <= 1e18, "softmax_scale must be finite, of a size of 1e18 at most");
  TORCH_CHECK_VALUE(q_.device() == kc.device(), "all tensors must be on the same device");
  check_cache("paged_attention_step", kc, vc, ke, ve, table, lengths);
  TORCH_CHECK_VALUE(q_.size(0) == lengths.size(0) && q_.size(2) == kc.size(3), "q: [sequences, heads, head_dim] of the page table's sequences and the cache's head_dim");
  TORCH_CHECK_VALUE(q_.size(1) > 0 && q_.size(1) % kc.size(1) == 0, "the heads of the cache must divide those of q");
  const c10::cuda::CUDAGuard guard(kc.device());
  Tensor o = empty(q_.sizes(), at::kBFloat16, q_);
  if (q_.size(0) == 0) return o;
  const bool lies = q_.stride(2) == 1 && (q_.size(1) <= 1 || q_.stride(1) % 8 == 0) && (q_.size(0) <= 1 || q_.stride(0) % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(q_.data_ptr()) % 16 == 0;
  const Tensor q = lies ? q_ : plain(q_);
  const Cache r = describe(kc, vc, ke, ve, table, lengths);
  size_t need = 0;
  check(lact_paged_attention_step_bytes(&r.c, q.size(1), window, &need), "lact_paged_attention_step_bytes");
  Tensor room;
  if (need > 0) room = bytes(need, q);
  check(lact_paged_attention_step(&r.c, ptr(q), stride_of(q, 0), stride_of(q, 1), q.size(1), window, static_cast<float>(scale), ptr(o),
                                  need > 0 ? ptr(room) : nullptr, need, status_word(q), stream_of(q)),
        "lact_paged_attention_step");
  return o;
}

using WriteSig = void(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      const OptTensor&);
using ReadSig = Tensor(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, int64_t, const OptTensor&);
using StepSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&, int64_t, double);
const auto& write_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::paged_cache_write", "").typed<WriteSig>();
  return o;
}
const auto& read_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::paged_cache_read", "").typed<ReadSig>();
  return o;
}
const auto& step_op() {
  static const auto o = c10::Dispatcher::singleton().findSchemaOrThrow("lact_b200::paged_attention_step", "").typed<StepSig>();
  return o;
}

// None of the three has a backward: a call with gradients or tangents raises.
void no_gradients(const char* what, std::initializer_list<const Tensor*> ts) {
  no_tangents(what, ts);
  for (const Tensor* t : ts) TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t->requires_grad()), what, " has no backward");
}
// What is written gets a new version, so that a backward that has saved it raises in place of reading what is there now.
void write_versioned(c10::DispatchKeySet keys, const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& k, const Tensor& v,
                     const Tensor& table, const Tensor& lengths, const OptTensor& cu) {
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    write_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, kc, vc, ke, ve, k, v, table, lengths, cu);
  }
  const Tensor kb = value(ke), vb = value(ve);
  for (const Tensor* t : {&kc, &vc, &kb, &vb})
    if (t->defined() && !t->is_inference()) torch::autograd::impl::bump_version(*t);
}
void write_autograd(c10::DispatchKeySet keys, const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& k, const Tensor& v,
                    const Tensor& table, const Tensor& lengths, const OptTensor& cu) {
  no_gradients("paged_cache_write", {&kc, &vc, &k, &v});
  at::AutoDispatchBelowAutograd guard;
  write_op().redispatch(keys & c10::after_autograd_keyset, kc, vc, ke, ve, k, v, table, lengths, cu);
}
Tensor read_autograd(c10::DispatchKeySet keys, const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve, const Tensor& table,
                     const Tensor& lengths, int64_t tokens, const OptTensor& cu) {
  no_gradients("paged_cache_read", {&kc, &vc});
  at::AutoDispatchBelowADInplaceOrView guard;
  return read_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, kc, vc, ke, ve, table, lengths, tokens, cu);
}
Tensor step_autograd(c10::DispatchKeySet keys, const Tensor& q, const Tensor& kc, const Tensor& vc, const OptTensor& ke, const OptTensor& ve,
                     const Tensor& table, const Tensor& lengths, int64_t window, double scale) {
  no_gradients("paged_attention_step", {&q, &kc, &vc});
  at::AutoDispatchBelowADInplaceOrView guard;
  return step_op().redispatch(keys & c10::after_ADInplaceOrView_keyset, q, kc, vc, ke, ve, table, lengths, window, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lact_b200, m) {
  m.def("paged_cache_write(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_exponent, Tensor(d!)? v_exponent, Tensor k, Tensor v, "
        "Tensor page_table, Tensor lengths, Tensor? cu_seqlens) -> ()");
  m.def("paged_cache_read(Tensor k_cache, Tensor v_cache, Tensor? k_exponent, Tensor? v_exponent, Tensor page_table, Tensor lengths, "
        "int tokens, Tensor? cu_seqlens) -> Tensor");
  m.def("paged_attention_step(Tensor q, Tensor k_cache, Tensor v_cache, Tensor? k_exponent, Tensor? v_exponent, Tensor page_table, "
        "Tensor lengths, int window, float softmax_scale) -> Tensor");
}
TORCH_LIBRARY_IMPL(lact_b200, CUDA, m) {
  m.impl("paged_cache_write", &write);
  m.impl("paged_cache_read", &read);
  m.impl("paged_attention_step", &step);
}
TORCH_LIBRARY_IMPL(lact_b200, CPU, m) {   // (what they refuse, and that they need a GPU)
  m.impl("paged_cache_write", &write);
  m.impl("paged_cache_read", &read);
  m.impl("paged_attention_step", &step);
}
TORCH_LIBRARY_IMPL(lact_b200, ADInplaceOrView, m) { m.impl("paged_cache_write", &write_versioned); }
TORCH_LIBRARY_IMPL(lact_b200, Autograd, m) {
  m.impl("paged_cache_write", &write_autograd);
  m.impl("paged_cache_read", &read_autograd);
  m.impl("paged_attention_step", &step_autograd);
}

}  // namespace lact_torch
