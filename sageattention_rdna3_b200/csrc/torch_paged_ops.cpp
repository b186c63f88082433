// torch.ops.sageattention.* of the operators around a growing cache: a thin wrapper that turns tensors into the pointers,
// sizes and strides of include/sage_paged_b200.h.
#include <Python.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>
#include <torch/types.h>

#include <climits>
#include <cmath>
#include <cstdlib>
#include <numeric>
#include <vector>

#include "../../include/sage_paged_b200.h"
#include "torch_paged.h"

namespace {

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == SAGE_OK, what, " failed: ", sage_last_error()); }

void* current_stream(const at::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

int dtype_code(const at::Tensor& t, bool with_f32) {
  if (with_f32 && t.scalar_type() == at::kFloat) return SAGE_DTYPE_F32;
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "expected an fp16 or bf16 tensor, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf ? SAGE_DTYPE_F16 : SAGE_DTYPE_BF16;
}

int size_of(int64_t n, const char* what) {
  TORCH_CHECK(n >= 0 && n <= INT_MAX, what, " is out of range: ", n);
  return static_cast<int>(n);
}

void check_vectors(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.stride(-1) == 1, name, " must be a CUDA tensor with a contiguous last dim");
  const int64_t unit = 16 / t.element_size();
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % unit == 0);
  TORCH_CHECK(ok, name, " needs a 16-byte aligned base and strides that are multiples of 16 bytes; got strides ", t.strides());
}

void check_int32(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == like.device() && (t.size(-1) <= 1 || t.stride(-1) == 1), name,
              " must be an int32 tensor on the device of the cache with a contiguous last dim");
}

// A dimension of extent 1 is never stepped over and may carry any stride in the caller's tensor.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) <= 1 ? t.size(-1) : t.stride(d); }

sage_strided_t strided_of(const at::Tensor& t, int64_t layout) {
  return {t.data_ptr(), stride_of(t, 0), stride_of(t, layout == 1 ? 1 : 2), stride_of(t, layout == 1 ? 2 : 1)};
}

sage_rotary_t rotary_of(const at::Tensor& freq, const at::Tensor& axis, int64_t n_axes, int64_t interleaved, const at::Tensor& like) {
  TORCH_CHECK(freq.scalar_type() == at::kLong && axis.scalar_type() == at::kInt && freq.is_contiguous() && axis.is_contiguous() &&
                  freq.numel() == axis.numel() && freq.device() == like.device() && axis.device() == like.device(),
              "the rotary table must be contiguous int64 frequencies and int32 axes on the device of the tensors");
  sage_rotary_t r{};
  r.freq = reinterpret_cast<const uint64_t*>(freq.data_ptr<int64_t>());
  r.axis = axis.data_ptr<int32_t>();
  r.pairs = size_of(freq.numel(), "pairs");
  r.n_axes = size_of(n_axes, "n_axes");
  r.interleaved = interleaved != 0;
  return r;
}

// positions: [.., n_axes] of which the last dim is contiguous
void set_positions(sage_rotary_t* r, const at::Tensor& p, const at::Tensor& like) {
  TORCH_CHECK((p.scalar_type() == at::kInt || p.scalar_type() == at::kLong) && p.device() == like.device() && p.size(-1) == r->n_axes &&
                  (p.stride(-1) == 1 || p.size(-1) == 1),
              "positions must be int32 or int64, on the device of the tensors, with one contiguous value per axis");
  r->positions = p.data_ptr();
  r->positions_64 = p.scalar_type() == at::kLong;
  r->stride_s = p.stride(-2);
  r->stride_b = p.dim() == 3 ? p.stride(0) : 0;
}

// rotary(Tensor query, Tensor? key, Tensor positions, Tensor freq, Tensor axis, int interleaved, int tensor_layout, int inverse)
// -> Tensor[]: the turned tensors, new ones.  positions: [S, n_axes] or [B, S, n_axes].
at::Tensor vector_aligned(const at::Tensor& t);
std::vector<at::Tensor> rotary(const at::Tensor& query, const c10::optional<at::Tensor>& key, const at::Tensor& positions,
                               const at::Tensor& freq, const at::Tensor& axis, int64_t interleaved, int64_t layout, int64_t inverse) {
  const at::Tensor q = vector_aligned(query);
  c10::optional<at::Tensor> k;
  if (key.has_value()) k = vector_aligned(*key);
  TORCH_CHECK(layout == 0 || layout == 1, "tensor_layout must be 0 (NHD) or 1 (HND)");
  TORCH_CHECK(q.dim() == 4 && (!k.has_value() || k->dim() == 4), "expected 4-D tensors");
  const int h_dim = layout == 1 ? 1 : 2, s_dim = layout == 1 ? 2 : 1;
  c10::cuda::CUDAGuard guard(q.device());
  check_vectors(q, "query");
  if (k.has_value()) {
    check_vectors(*k, "key");
    TORCH_CHECK(k->scalar_type() == q.scalar_type() && k->device() == q.device() && k->size(0) == q.size(0) &&
                    k->size(s_dim) == q.size(s_dim) && k->size(3) == q.size(3),
                "query and key differ in dtype, device, batch, length or head_dim");
  }
  const int64_t B = q.size(0), S = q.size(s_dim);
  TORCH_CHECK((positions.dim() == 2 && positions.size(0) == S) || (positions.dim() == 3 && positions.size(0) == B && positions.size(1) == S),
              "positions must be [S, n_axes] or [B, S, n_axes]");
  sage_rotary_t r = rotary_of(freq, axis, positions.size(-1), interleaved, q);
  set_positions(&r, positions, q);
  std::vector<at::Tensor> out{at::empty(q.sizes(), q.options())};
  if (k.has_value()) out.push_back(at::empty(k->sizes(), k->options()));
  const sage_strided_t qs = strided_of(q, layout), qo = strided_of(out[0], layout);
  sage_strided_t ks{}, ko{};
  if (k.has_value()) {
    ks = strided_of(*k, layout);
    ko = strided_of(out[1], layout);
  }
  check_rc(sage_apply_rotary(&qs, &qo, k.has_value() ? &ks : nullptr, k.has_value() ? &ko : nullptr, &r, dtype_code(q, true),
                             size_of(B, "batch"), size_of(q.size(h_dim), "heads"), k.has_value() ? size_of(k->size(h_dim), "heads") : 0,
                             size_of(S, "length"), size_of(q.size(3), "head_dim"), inverse != 0, current_stream(q)),
           "rotary");
  return out;
}

// `t`, or a copy of it that 16-byte loads can read.
at::Tensor vector_aligned(const at::Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % unit == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// The operator below autograd: through the dispatcher where a mode wants to see it.
std::vector<at::Tensor> rotary_below(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions, const at::Tensor& freq,
                                     const at::Tensor& axis, int64_t interleaved, int64_t layout, int64_t inverse) {
  if (!c10::impl::TorchDispatchModeTLS::any_modes_set()) return rotary(q, k, positions, freq, axis, interleaved, layout, inverse);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("sageattention::rotary", "").typed<decltype(rotary)>();
  return op.call(q, k, positions, freq, axis, interleaved, layout, inverse);
}

// The gradient of a rotation is the rotation the other way.  (In Python the same node cost 40 us of host time.)
struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const c10::optional<at::Tensor>& k,
                                                const at::Tensor& positions, const at::Tensor& freq, const at::Tensor& axis,
                                                int64_t interleaved, int64_t layout, int64_t inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, freq, axis});
    ctx->saved_data["args"] = std::vector<int64_t>{interleaved, layout, inverse};
    auto out = rotary_below(q, k, positions, freq, axis, interleaved, layout, inverse);
    // (a result of what needs no gradient needs none either)
    if (!q.requires_grad()) ctx->mark_non_differentiable({out[0]});
    else if (k.has_value() && !k->requires_grad()) ctx->mark_non_differentiable({out[1]});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    at::Tensor dq, dk;
    auto turn = [&](const at::Tensor& a, const c10::optional<at::Tensor>& b) {
      return RotaryNode::apply(a, b, saved[0], saved[1], saved[2], args[0], args[1], args[2] == 0 ? 1 : 0);
    };
    const bool want_q = grads[0].defined() && ctx->needs_input_grad(0);
    const bool want_k = grads.size() > 1 && grads[1].defined() && ctx->needs_input_grad(1);
    if (want_q) {
      const auto d = turn(grads[0], want_k ? c10::optional<at::Tensor>(grads[1]) : c10::nullopt);
      dq = d[0];
      if (want_k) dk = d[1];
    } else if (want_k) {
      dk = turn(grads[1], c10::nullopt)[0];
    }
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::vector<at::Tensor> rotary_autograd(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions,
                                        const at::Tensor& freq, const at::Tensor& axis, int64_t interleaved, int64_t layout,
                                        int64_t inverse) {
  return RotaryNode::apply(q, k, positions, freq, axis, interleaved, layout, inverse);
}

sage_paged_kv_t cache_of(const at::Tensor& k, const at::Tensor& v, int64_t layout) {
  TORCH_CHECK(layout == 0 || layout == 1, "tensor_layout must be 0 (NHD) or 1 (HND)");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == v.device(),
              "k_pages and v_pages must be 4-D tensors of one shape, dtype and device");
  check_vectors(k, "k_pages");
  check_vectors(v, "v_pages");
  const int h = layout == 1 ? 1 : 2, s = layout == 1 ? 2 : 1;
  sage_paged_kv_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.num_pages = size_of(k.size(0), "num_pages");
  c.page_size = size_of(k.size(s), "page_size");
  c.Hkv = size_of(k.size(h), "heads");
  c.D = size_of(k.size(3), "head_dim");
  c.dtype = dtype_code(k, false);
  c.k_stride_page = stride_of(k, 0); c.k_stride_slot = stride_of(k, s); c.k_stride_head = stride_of(k, h);
  c.v_stride_page = stride_of(v, 0); c.v_stride_slot = stride_of(v, s); c.v_stride_head = stride_of(v, h);
  return c;
}

sage_paged_batch_t batch_of(const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_q,
                            int64_t tokens, const at::Tensor& like) {
  TORCH_CHECK(page_table.dim() == 2 && kv_lens.dim() == 1 && page_table.size(0) == kv_lens.size(0),
              "page_table must be [B, pages] and kv_lens [B]");
  check_int32(page_table, like, "page_table");
  check_int32(kv_lens, like, "kv_lens");
  sage_paged_batch_t b{};
  b.page_table = page_table.data_ptr<int32_t>();
  b.table_stride = page_table.stride(0);
  b.table_width = size_of(page_table.size(1), "table width");
  b.kv_lens = kv_lens.data_ptr<int32_t>();
  b.B = size_of(kv_lens.size(0), "batch");
  b.T = size_of(tokens, "tokens");
  if (cu_q.has_value()) {
    TORCH_CHECK(cu_q->dim() == 1 && cu_q->size(0) == kv_lens.size(0) + 1, "cu_q must be [B + 1]");
    check_int32(*cu_q, like, "cu_q");
    b.cu_q = cu_q->data_ptr<int32_t>();
  }
  return b;
}

sage_rows_t rows_of(const at::Tensor& t) { return {t.data_ptr(), stride_of(t, 0), stride_of(t, 1)}; }

int* status_of(const at::Tensor& status, const at::Tensor& like) {
  TORCH_CHECK(status.scalar_type() == at::kInt && status.numel() >= 1 && status.device() == like.device(),
              "status must be an int32 tensor on the device of the cache");
  return status.data_ptr<int>();
}

void check_rows(const at::Tensor& t, const at::Tensor& k_pages, int64_t heads, const char* name) {
  TORCH_CHECK(t.dim() == 3 && t.size(2) == k_pages.size(3) && (heads < 0 || t.size(1) == heads) && t.scalar_type() == k_pages.scalar_type() &&
                  t.device() == k_pages.device(),
              name, " must be [T, heads, D] in the dtype and on the device of the cache");
  check_vectors(t, name);
}

// Counts a change of `t` in place: a backward pass that kept it is refused then.  (Tensors made for inference count none.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// paged_append(Tensor(a!) k_pages, Tensor(b!) v_pages, int tensor_layout, Tensor key, Tensor value, Tensor page_table, Tensor kv_lens,
//              Tensor? cu_q, Tensor? query, Tensor? freq, Tensor? axis, int n_axes, int interleaved, Tensor? positions, Tensor(c!) status)
// -> Tensor[]: the turned query, if one is given.  positions: [T, n_axes].
std::vector<at::Tensor> paged_append(at::Tensor& k_pages, at::Tensor& v_pages, int64_t layout, const at::Tensor& k, const at::Tensor& v,
                                     const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_q,
                                     const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& freq,
                                     const c10::optional<at::Tensor>& axis, int64_t n_axes, int64_t interleaved,
                                     const c10::optional<at::Tensor>& positions, const at::Tensor& status) {
  const sage_paged_kv_t cache = cache_of(k_pages, v_pages, layout);
  c10::cuda::CUDAGuard guard(k_pages.device());
  check_rows(k, k_pages, cache.Hkv, "key");
  check_rows(v, k_pages, cache.Hkv, "value");
  const int64_t T = k.size(0);
  TORCH_CHECK(v.size(0) == T, "key and value differ in length");
  const sage_paged_batch_t batch = batch_of(page_table, kv_lens, cu_q, T, k_pages);
  sage_rotary_t r{};
  const bool turn = freq.has_value();
  if (turn) {
    TORCH_CHECK(axis.has_value(), "freq and axis come together");
    r = rotary_of(*freq, *axis, n_axes, interleaved, k_pages);
    if (positions.has_value()) {
      TORCH_CHECK(positions->dim() == 2 && positions->size(0) == T, "positions must be [T, n_axes]");
      set_positions(&r, *positions, k_pages);
    }
  }
  std::vector<at::Tensor> out;
  sage_rows_t qs{}, qo{};
  if (q.has_value()) {
    check_rows(*q, k_pages, -1, "query");
    TORCH_CHECK(q->size(0) == T, "query and key differ in length");
    out.push_back(at::empty(q->sizes(), q->options()));
    qs = rows_of(*q);
    qo = rows_of(out[0]);
  }
  const sage_rows_t ks = rows_of(k), vs = rows_of(v);
  check_rc(sage_paged_append(&cache, &batch, &ks, &vs, q.has_value() ? &qs : nullptr, q.has_value() ? &qo : nullptr,
                             q.has_value() ? size_of(q->size(1), "heads") : 0, turn ? &r : nullptr, status_of(status, k_pages),
                             current_stream(k_pages)),
           "paged_append");
  written(k_pages);
  written(v_pages);
  return out;
}

// First and last byte of a tensor, and whether two of them can share any.
struct Bytes {
  int64_t lo, hi;
  explicit Bytes(const at::Tensor& t) : lo(reinterpret_cast<int64_t>(t.data_ptr())), hi(lo + t.element_size()) {
    for (int64_t i = 0; i < t.dim(); ++i) hi += (t.size(i) - 1) * t.stride(i) * static_cast<int64_t>(t.element_size());
  }
};
bool apart(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return true;
  const Bytes x(a), y(b);
  return x.hi <= y.lo || y.hi <= x.lo;
}

// Rows `a` and `b`, [T, H, D] both, known to lie between one another: true if no row of one meets a row of the other.  It is enough
// that they keep to different parts of a period in memory: that of all their rows (slots of a head), of a token, or of a head.
bool rows_apart(const at::Tensor& a, const at::Tensor& b) {
  const int64_t T = a.size(0), H = a.size(1), D = a.size(2), size = a.element_size();
  const int64_t distance = (reinterpret_cast<int64_t>(b.data_ptr()) - reinterpret_cast<int64_t>(a.data_ptr())) / size;
  const int64_t st = T > 1 ? a.stride(0) : 0, sh = H > 1 ? a.stride(1) : 0;
  if ((T > 1 && b.stride(0) != st) || (H > 1 && b.stride(1) != sh)) return false;
  auto separate = [&](int64_t period, int64_t length) {          // `length` values from a multiple of `period` and from `distance` on
    if (period <= 0) return false;
    const int64_t d = (distance % period + period) % period;
    return d >= length && d + length <= period;
  };
  return separate(std::gcd(st, sh), D) || separate(st, (H - 1) * sh + D) || separate(sh, (T - 1) * st + D);
}

// Each row of q is read by the thread blocks that write the same row of o and no others: o may be q, but not a shifted q.
void check_output(const at::Tensor& o, const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages) {
  at::assert_no_internal_overlap(o);
  bool same = o.data_ptr() == q.data_ptr();
  for (int64_t i = 0; i < 3; ++i) same = same && (o.size(i) <= 1 || o.stride(i) == q.stride(i));
  TORCH_CHECK(same || apart(o, q) || rows_apart(o, q), "the output must be q or share no memory with it: they overlap");
  TORCH_CHECK(apart(o, k_pages) && apart(o, v_pages), "the output must share no memory with the cache: they overlap");
}

// paged_attn(Tensor query, Tensor(a!) output, Tensor k_pages, Tensor v_pages, int tensor_layout, Tensor page_table, Tensor kv_lens,
//            Tensor? cu_q, int max_q, int is_causal, float sm_scale, Tensor(b!)? lse, Tensor? shared_pages, int zero_rest, Tensor(c!) status) -> ()
void paged_attn(const at::Tensor& q, at::Tensor& o, const at::Tensor& k_pages, const at::Tensor& v_pages, int64_t layout,
                const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_q, int64_t max_q,
                int64_t is_causal, double sm_scale, const c10::optional<at::Tensor>& lse, const c10::optional<at::Tensor>& shared_pages,
                int64_t zero_rest, const at::Tensor& status) {
  const sage_paged_kv_t cache = cache_of(k_pages, v_pages, layout);
  c10::cuda::CUDAGuard guard(k_pages.device());
  check_rows(q, k_pages, -1, "query");
  check_rows(o, k_pages, q.size(1), "output");
  TORCH_CHECK(o.size(0) == q.size(0), "query and output differ in length");
  check_output(o, q, k_pages, v_pages);
  const sage_paged_batch_t batch = batch_of(page_table, kv_lens, cu_q, q.size(0), k_pages);
  const int Hq = size_of(q.size(1), "heads"), longest = size_of(max_q, "max_q");
  int n_shared = 0;
  if (shared_pages.has_value()) {
    TORCH_CHECK(shared_pages->dim() == 1, "shared_pages must be 1-D");
    check_int32(*shared_pages, k_pages, "shared_pages");
    n_shared = size_of(shared_pages->size(0), "shared pages");
  }
  float* lse_ptr = nullptr;
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() == q.size(0) * q.size(1) && lse->device() == q.device(),
                "lse must be a contiguous fp32 [T, heads] tensor");
    lse_ptr = lse->data_ptr<float>();
  }
  const int64_t bytes = sage_paged_workspace_bytes(&cache, &batch, Hq, longest, n_shared);
  TORCH_CHECK(bytes >= 0, "paged_attn failed: ", sage_last_error());
  at::Tensor workspace = at::empty({bytes}, k_pages.options().dtype(at::kByte));
  const sage_rows_t qs = rows_of(q), os = rows_of(o);
  check_rc(sage_paged_attn(&cache, &batch, &qs, &os, Hq, longest, is_causal != 0, static_cast<float>(sm_scale), lse_ptr,
                           n_shared > 0 ? shared_pages->data_ptr<int32_t>() : nullptr, n_shared, zero_rest != 0,
                           status_of(status, k_pages), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, current_stream(k_pages)),
           "paged_attn");
  written(o);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sageattention, m) {
  m.def("rotary(Tensor query, Tensor? key, Tensor positions, Tensor freq, Tensor axis, int interleaved, int tensor_layout, "
        "int inverse) -> Tensor[]");
  m.def("paged_append(Tensor(a!) k_pages, Tensor(b!) v_pages, int tensor_layout, Tensor key, Tensor value, Tensor page_table, "
        "Tensor kv_lens, Tensor? cu_q, Tensor? query, Tensor? freq, Tensor? axis, int n_axes, int interleaved, Tensor? positions, "
        "Tensor(c!) status) -> Tensor[]");
  m.def("paged_attn(Tensor query, Tensor(a!) output, Tensor k_pages, Tensor v_pages, int tensor_layout, Tensor page_table, "
        "Tensor kv_lens, Tensor? cu_q, int max_q, int is_causal, float sm_scale, Tensor(b!)? lse, Tensor? shared_pages, int zero_rest, "
        "Tensor(c!) status) -> ()");
}

TORCH_LIBRARY_IMPL(sageattention, AutogradCUDA, m) {
  m.impl("rotary", &rotary_autograd);
}

TORCH_LIBRARY_IMPL(sageattention, CUDA, m) {
  m.impl("rotary", &rotary);
  m.impl("paged_append", &paged_append);
  m.impl("paged_attn", &paged_attn);
}

// ---------------------------------------------------------------- short ways
// A call of a few microseconds on the GPU is bound by the host: of 19 us per call, the checks in Python and the conversion of
// fifteen arguments by torch.ops took 13.  These functions make the same checks on the tensors themselves; whatever is not a plain
// call - a check that fails, an argument of another type, a tensor that needs a gradient or a copy, a subclass, an active mode -
// returns None and takes the way through Python, which raises the errors.
namespace {

// A strided CUDA tensor that is just that; *out is left alone for None where that is allowed.
bool plain(PyObject* o, const at::Tensor** out, bool none = false) {
  if (none && o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (at::isTensorSubclassLike(t) || t.layout() != at::kStrided || !t.is_cuda() || t.unsafeGetTensorImpl()->has_symbolic_sizes_strides() ||
      t.is_neg() || t.is_conj() || torch::autograd::isFwGradDefined(t)) {
    return false;
  }
  *out = &t;
  return true;
}

bool modes_active() { return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set(); }

// Every call is to be looked at when it is done (core.py).
bool checks_status() {
  const char* e = std::getenv("SAGEATTN_B200_CHECK_STATUS");
  return e != nullptr && *e != '\0';
}

bool vectors(const at::Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  if (t.stride(-1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) {
    if (t.stride(i) % unit != 0 || (t.size(i) > 1 && t.stride(i) == 0)) return false;
  }
  return true;
}

at::Tensor new_like(const at::Tensor& t) { return at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), c10::nullopt); }

bool needs_grad(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

int64_t layout_of(PyObject* o) {
  if (!PyUnicode_CheckExact(o)) return -1;
  return PyUnicode_CompareWithASCIIString(o, "HND") == 0 ? 1 : PyUnicode_CompareWithASCIIString(o, "NHD") == 0 ? 0 : -1;
}

bool small_int(PyObject* o, int* out) {
  if (!PyLong_CheckExact(o)) return false;
  const long v = PyLong_AsLong(o);
  if (v < 0 || v > INT_MAX) {
    PyErr_Clear();
    return false;
  }
  *out = static_cast<int>(v);
  return true;
}

bool plain_int32(const at::Tensor& t, const at::Tensor& like, int64_t dim) {
  return t.scalar_type() == at::kInt && t.device() == like.device() && t.dim() == dim && (t.size(-1) <= 1 || t.stride(-1) == 1) && t.numel() > 0;
}

bool plain_cache(const at::Tensor& k, const at::Tensor& v, int64_t layout) {
  if (layout < 0 || k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type() || k.device() != v.device()) return false;
  if (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16) return false;
  return vectors(k) && vectors(v) && k.numel() > 0;
}

bool plain_batch(const at::Tensor& table, const at::Tensor& lens, const at::Tensor* cu, const at::Tensor& rows, const at::Tensor& like) {
  if (!plain_int32(table, like, 2) || !plain_int32(lens, like, 1) || table.size(0) != lens.size(0)) return false;
  if (cu == nullptr) return rows.size(0) == lens.size(0);
  return plain_int32(*cu, like, 1) && cu->size(0) == lens.size(0) + 1;
}

bool plain_rows(const at::Tensor& t, const at::Tensor& pages, int64_t heads) {
  return t.dim() == 3 && t.numel() > 0 && t.size(2) == pages.size(3) && (heads < 0 || t.size(1) == heads) && t.scalar_type() == pages.scalar_type() &&
         t.device() == pages.device() && vectors(t) && !needs_grad(t);
}

bool plain_table(const at::Tensor& freq, const at::Tensor& axis, int n_axes, const at::Tensor& like) {
  return freq.device() == like.device() && axis.device() == like.device() && n_axes >= 1 && n_axes <= SAGE_MAX_ROTARY_AXES &&
         freq.is_contiguous() && axis.is_contiguous() && freq.scalar_type() == at::kLong && axis.scalar_type() == at::kInt;
}

// positions [n] or [n, axes] (`batch` < 0), or with a batch dimension in front; false if they do not fit.  *bare: without a
// dimension for the one axis.
bool plain_positions(sage_rotary_t* r, const at::Tensor& p, const at::Tensor& like, int64_t batch, int64_t n, bool* bare) {
  if ((p.scalar_type() != at::kInt && p.scalar_type() != at::kLong) || p.device() != like.device()) return false;
  int64_t dim = p.dim();
  *bare = r->n_axes == 1 && (dim == 1 ? p.size(0) == n : batch >= 0 && dim == 2 && p.size(0) == batch && p.size(1) == n);
  if (!*bare) {
    if (dim < 2 || p.size(-1) != r->n_axes || (r->n_axes > 1 && p.stride(-1) != 1)) return false;
    --dim;
  }
  if (p.size(dim - 1) != n || dim > (batch >= 0 ? 2 : 1) || (dim == 2 && p.size(0) != batch)) return false;
  r->positions = p.data_ptr();
  r->positions_64 = p.scalar_type() == at::kLong;
  r->stride_s = p.stride(dim - 1);
  r->stride_b = dim == 2 ? p.stride(0) : 0;
  return true;
}

}  // namespace

// rotary_plain(q, k or None, positions, freq, axis, n_axes, interleaved, head_dim, tensor_layout) -> (q, k) or q, or None
PyObject* sage_rotary_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *q = nullptr, *k = nullptr, *positions = nullptr, *freq = nullptr, *axis = nullptr;
  int n_axes = 0, head_dim = 0;
  if (nargs != 9 || !plain(args[0], &q) || !plain(args[1], &k, true) || !plain(args[2], &positions) || !plain(args[3], &freq) ||
      !plain(args[4], &axis) || !small_int(args[5], &n_axes) || !PyBool_Check(args[6]) || !small_int(args[7], &head_dim) || modes_active()) {
    Py_RETURN_NONE;
  }
  const int64_t layout = layout_of(args[8]);
  const at::ScalarType dt = q->scalar_type();
  if (layout < 0 || (dt != at::kHalf && dt != at::kBFloat16 && dt != at::kFloat) || q->dim() != 4 || q->numel() == 0 || q->size(3) != head_dim ||
      !vectors(*q) || !plain_table(*freq, *axis, n_axes, *q)) {
    Py_RETURN_NONE;
  }
  const int h_dim = layout == 1 ? 1 : 2, s_dim = layout == 1 ? 2 : 1;
  const int64_t B = q->size(0), S = q->size(s_dim);
  if (k != nullptr && (k->dim() != 4 || k->numel() == 0 || k->scalar_type() != dt || k->device() != q->device() || k->size(0) != B ||
                       k->size(s_dim) != S || k->size(3) != head_dim || !vectors(*k))) {
    Py_RETURN_NONE;
  }
  sage_rotary_t r = rotary_of(*freq, *axis, n_axes, args[6] == Py_True, *q);
  bool bare = false;
  if (!plain_positions(&r, *positions, *q, B, S, &bare)) Py_RETURN_NONE;
  at::Tensor qo, ko;
  if (needs_grad(*q) || (k != nullptr && needs_grad(*k))) {
    pybind11::gil_scoped_release no_gil;
    const auto d = RotaryNode::apply(*q, k != nullptr ? c10::optional<at::Tensor>(*k) : c10::nullopt, bare ? positions->unsqueeze(-1) : *positions, *freq, *axis,
                                     args[6] == Py_True ? 1 : 0, layout, 0);
    qo = d[0];
    if (k != nullptr) ko = d[1];
  } else {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::CUDAGuard guard(q->device());
    qo = new_like(*q);
    if (k != nullptr) ko = new_like(*k);
    const sage_strided_t qs = strided_of(*q, layout), qos = strided_of(qo, layout);
    sage_strided_t ks{}, kos{};
    if (k != nullptr) {
      ks = strided_of(*k, layout);
      kos = strided_of(ko, layout);
    }
    check_rc(sage_apply_rotary(&qs, &qos, k != nullptr ? &ks : nullptr, k != nullptr ? &kos : nullptr, &r, dtype_code(*q, true),
                               size_of(B, "batch"), size_of(q->size(h_dim), "heads"), k != nullptr ? size_of(k->size(h_dim), "heads") : 0,
                               size_of(S, "length"), head_dim, 0, current_stream(*q)),
             "rotary");
  }
  if (k == nullptr) return THPVariable_Wrap(qo);
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(qo));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(ko));
  return pair;
  END_HANDLE_TH_ERRORS
}

// paged_append_plain(k_pages, v_pages, tensor_layout, k, v, page_table, kv_lens, cu_q or None, q or None, freq or None, axis or None, n_axes,
//                    interleaved, positions or None) -> q, or True without one, or None
PyObject* sage_paged_append_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *kp = nullptr, *vp = nullptr, *k = nullptr, *v = nullptr, *table = nullptr, *lens = nullptr, *cu = nullptr, *q = nullptr,
                   *freq = nullptr, *axis = nullptr, *positions = nullptr;
  int n_axes = 0;
  if (nargs != 14 || !plain(args[0], &kp) || !plain(args[1], &vp) || !plain(args[3], &k) || !plain(args[4], &v) || !plain(args[5], &table) ||
      !plain(args[6], &lens) || !plain(args[7], &cu, true) || !plain(args[8], &q, true) || !plain(args[9], &freq, true) ||
      !plain(args[10], &axis, true) || !small_int(args[11], &n_axes) || !PyBool_Check(args[12]) || !plain(args[13], &positions, true) || modes_active() || checks_status()) {
    Py_RETURN_NONE;
  }
  const int64_t layout = layout_of(args[2]);
  if (!plain_cache(*kp, *vp, layout) || !plain_batch(*table, *lens, cu, *k, *kp)) Py_RETURN_NONE;
  const int64_t Hkv = kp->size(layout == 1 ? 1 : 2), T = k->size(0);
  if (!plain_rows(*k, *kp, Hkv) || !plain_rows(*v, *kp, Hkv) || v->size(0) != T || (q != nullptr && (!plain_rows(*q, *kp, -1) || q->size(0) != T)) ||
      (freq == nullptr) != (axis == nullptr) || (freq == nullptr && (q != nullptr || positions != nullptr)) ||
      (freq != nullptr && !plain_table(*freq, *axis, n_axes, *kp))) {
    Py_RETURN_NONE;
  }
  int* status = nullptr;
  const volatile int32_t* mirror = nullptr;
  if (!sage_device_status(kp->get_device(), &status, &mirror) || (mirror != nullptr && *mirror != 0)) Py_RETURN_NONE;
  sage_rotary_t r{};
  if (freq != nullptr) {
    r = rotary_of(*freq, *axis, n_axes, args[12] == Py_True, *kp);
    bool bare = false;
    if (positions != nullptr && !plain_positions(&r, *positions, *kp, -1, T, &bare)) Py_RETURN_NONE;
  }
  at::Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::CUDAGuard guard(kp->device());
    const sage_paged_kv_t cache = cache_of(*kp, *vp, layout);
    const sage_paged_batch_t batch = batch_of(*table, *lens, cu != nullptr ? c10::optional<at::Tensor>(*cu) : c10::nullopt, T, *kp);
    sage_rows_t qs{}, qo{};
    if (q != nullptr) {
      out = new_like(*q);
      qs = rows_of(*q);
      qo = rows_of(out);
    }
    const sage_rows_t ks = rows_of(*k), vs = rows_of(*v);
    check_rc(sage_paged_append(&cache, &batch, &ks, &vs, q != nullptr ? &qs : nullptr, q != nullptr ? &qo : nullptr,
                               q != nullptr ? size_of(q->size(1), "heads") : 0, freq != nullptr ? &r : nullptr, status, current_stream(*kp)),
             "paged_append");
    written(*kp);
    written(*vp);
  }
  if (q == nullptr) Py_RETURN_TRUE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// paged_attn_plain(q, k_pages, v_pages, tensor_layout, page_table, kv_lens, cu_q or None, max_q or None, is_causal, sm_scale or None,
//                  return_lse, shared_pages or None) -> o or (o, lse), or None
PyObject* sage_paged_attn_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const at::Tensor *q = nullptr, *kp = nullptr, *vp = nullptr, *table = nullptr, *lens = nullptr, *cu = nullptr, *shared = nullptr;
  int max_q = 0;
  if (nargs != 12 || !plain(args[0], &q) || !plain(args[1], &kp) || !plain(args[2], &vp) || !plain(args[4], &table) || !plain(args[5], &lens) ||
      !plain(args[6], &cu, true) || (args[7] != Py_None && !small_int(args[7], &max_q)) || !PyBool_Check(args[8]) ||
      (args[9] != Py_None && !PyFloat_CheckExact(args[9])) || !PyBool_Check(args[10]) || !plain(args[11], &shared, true) || modes_active() || checks_status()) {
    Py_RETURN_NONE;
  }
  const int64_t layout = layout_of(args[3]);
  if (!plain_cache(*kp, *vp, layout) || !plain_rows(*q, *kp, -1) || !plain_batch(*table, *lens, cu, *q, *kp)) Py_RETURN_NONE;
  const int64_t Hkv = kp->size(layout == 1 ? 1 : 2), Hq = q->size(1), T = q->size(0);
  if (Hq % Hkv != 0 || Hq / Hkv > 128 || (shared != nullptr && (!plain_int32(*shared, *kp, 1) || shared->size(0) > table->size(1)))) Py_RETURN_NONE;
  int* status = nullptr;
  const volatile int32_t* mirror = nullptr;
  if (!sage_device_status(kp->get_device(), &status, &mirror) || (mirror != nullptr && *mirror != 0)) Py_RETURN_NONE;
  const double sm_scale = args[9] == Py_None ? std::pow(static_cast<double>(kp->size(3)), -0.5) : PyFloat_AS_DOUBLE(args[9]);
  const bool causal = args[8] == Py_True, want_lse = args[10] == Py_True;
  at::Tensor out, lse;
  {
    pybind11::gil_scoped_release no_gil;
    c10::cuda::CUDAGuard guard(kp->device());
    const sage_paged_kv_t cache = cache_of(*kp, *vp, layout);
    const sage_paged_batch_t batch = batch_of(*table, *lens, cu != nullptr ? c10::optional<at::Tensor>(*cu) : c10::nullopt, T, *kp);
    const int heads = size_of(Hq, "heads"), n_shared = shared != nullptr ? size_of(shared->size(0), "shared pages") : 0;
    out = new_like(*q);
    if (want_lse) lse = at::detail::empty_cuda({T, Hq}, at::kFloat, q->device(), c10::nullopt);
    const int64_t bytes = sage_paged_workspace_bytes(&cache, &batch, heads, max_q, n_shared);
    TORCH_CHECK(bytes >= 0, "paged_attn failed: ", sage_last_error());
    const c10::DataPtr workspace = c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes));
    const sage_rows_t qs = rows_of(*q), os = rows_of(out);
    check_rc(sage_paged_attn(&cache, &batch, &qs, &os, heads, max_q, causal, static_cast<float>(sm_scale), want_lse ? lse.data_ptr<float>() : nullptr,
                             n_shared > 0 ? shared->data_ptr<int32_t>() : nullptr, n_shared, cu != nullptr, status, workspace.get(), bytes,
                             current_stream(*kp)),
             "paged_attn");
  }
  if (!want_lse) return THPVariable_Wrap(out);
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(lse));
  return pair;
  END_HANDLE_TH_ERRORS
}
