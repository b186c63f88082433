// torch.ops.sageattention.* of the operators around a growing cache: a thin wrapper that turns tensors into the pointers,
// sizes and strides of include/sage_paged_b200.h.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/types.h>

#include <climits>
#include <vector>

#include "../../include/sage_paged_b200.h"

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
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == like.device() && t.stride(-1) == 1, name,
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
std::vector<at::Tensor> rotary(const at::Tensor& q, const c10::optional<at::Tensor>& k, const at::Tensor& positions,
                               const at::Tensor& freq, const at::Tensor& axis, int64_t interleaved, int64_t layout, int64_t inverse) {
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

// paged_append(Tensor(a!) k_pages, Tensor(b!) v_pages, int tensor_layout, Tensor key, Tensor value, Tensor page_table, Tensor kv_lens,
//              Tensor? cu_q, Tensor? query, Tensor? freq, Tensor? axis, int n_axes, int interleaved, Tensor? positions, Tensor status)
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
  return out;
}

// paged_attn(Tensor query, Tensor(a!) output, Tensor k_pages, Tensor v_pages, int tensor_layout, Tensor page_table, Tensor kv_lens,
//            Tensor? cu_q, int max_q, int is_causal, float sm_scale, Tensor? lse, Tensor? shared_pages, int zero_rest, Tensor status) -> ()
void paged_attn(const at::Tensor& q, at::Tensor& o, const at::Tensor& k_pages, const at::Tensor& v_pages, int64_t layout,
                const at::Tensor& page_table, const at::Tensor& kv_lens, const c10::optional<at::Tensor>& cu_q, int64_t max_q,
                int64_t is_causal, double sm_scale, const c10::optional<at::Tensor>& lse, const c10::optional<at::Tensor>& shared_pages,
                int64_t zero_rest, const at::Tensor& status) {
  const sage_paged_kv_t cache = cache_of(k_pages, v_pages, layout);
  c10::cuda::CUDAGuard guard(k_pages.device());
  check_rows(q, k_pages, -1, "query");
  check_rows(o, k_pages, q.size(1), "output");
  TORCH_CHECK(o.size(0) == q.size(0), "query and output differ in length");
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
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sageattention, m) {
  m.def("rotary(Tensor query, Tensor? key, Tensor positions, Tensor freq, Tensor axis, int interleaved, int tensor_layout, "
        "int inverse) -> Tensor[]");
  m.def("paged_append(Tensor(a!) k_pages, Tensor(b!) v_pages, int tensor_layout, Tensor key, Tensor value, Tensor page_table, "
        "Tensor kv_lens, Tensor? cu_q, Tensor? query, Tensor? freq, Tensor? axis, int n_axes, int interleaved, Tensor? positions, "
        "Tensor status) -> Tensor[]");
  m.def("paged_attn(Tensor query, Tensor(a!) output, Tensor k_pages, Tensor v_pages, int tensor_layout, Tensor page_table, "
        "Tensor kv_lens, Tensor? cu_q, int max_q, int is_causal, float sm_scale, Tensor? lse, Tensor? shared_pages, int zero_rest, "
        "Tensor status) -> ()");
}

TORCH_LIBRARY_IMPL(sageattention, CUDA, m) {
  m.impl("rotary", &rotary);
  m.impl("paged_append", &paged_append);
  m.impl("paged_attn", &paged_attn);
}
