// Host side of the C ABI declared in include/sage_paged_b200.h: argument checks, choice of the kernel, launches.  No torch
// types, no allocation, no synchronisation.
#include "../../include/sage_paged_b200.h"

#include <algorithm>

#include "host_common.h"
#include "rotary_kernels.cuh"

using namespace sage_host;
using namespace sage::paged;

namespace {

Status status_of(int* word) {
  Status s;
  s.word = word;
  s.host = nullptr;
  int dev = 0;
  if (word != nullptr && cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
    s.host = g_status_host[dev].load(std::memory_order_relaxed);
  }
  return s;
}

// (`unit`: elements of 16 bytes)
bool stride_ok(int64_t stride, int unit) { return stride % unit == 0; }
bool rows_ok(const sage_rows_t* r) { return r->ptr != nullptr && aligned16(r->ptr) && r->stride_t % 8 == 0 && r->stride_h % 8 == 0; }

int check_rotary(const sage_rotary_t* r, int D) {
  SAGE_REQUIRE(r->freq != nullptr && r->axis != nullptr, "rotary: null table");
  SAGE_REQUIRE(r->pairs >= 8 && r->pairs % 8 == 0 && 2 * r->pairs <= D, "rotary: the number of pairs must be a multiple of 8 and at most head_dim / 2, got %d", r->pairs);
  SAGE_REQUIRE(r->n_axes >= 1 && r->n_axes <= SAGE_MAX_ROTARY_AXES, "rotary: 1 to %d axes, got %d", SAGE_MAX_ROTARY_AXES, r->n_axes);
  return SAGE_OK;
}

Rotary rotary_of(const sage_rotary_t* r, int inverse) {
  Rotary x;
  memset(&x, 0, sizeof(x));
  if (r == nullptr) return x;
  x.freq = r->freq;
  x.axis = r->axis;
  x.pairs = r->pairs;
  x.n_axes = r->n_axes;
  x.interleaved = r->interleaved;
  x.positions = r->positions;
  x.positions_64 = r->positions_64;
  x.stride_b = r->stride_b;
  x.stride_s = r->stride_s;
  x.inverse = inverse;
  return x;
}

// Heads per block of the rotary and append kernels: as many as leave four blocks of 256 threads to every SM, at most 8; few
// tokens get a thread per group and head.
struct HeadSplit {
  int per_block, unroll;
};
int split_heads(HeadSplit* out, long long token_blocks, int heads) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  out->unroll = 4;
  for (int n : {8, 4}) {
    out->per_block = n;
    if (token_blocks * ((heads + n - 1) / n) >= 4LL * sms) return SAGE_OK;
  }
  out->per_block = out->unroll = 1;
  return SAGE_OK;
}

template <typename T, int D>
int launch_rotary(const RotaryParams& p, const HeadSplit& split, unsigned token_blocks, cudaStream_t stream) {
  const int heads = p.Hq + p.Hkv;
  const dim3 grid(token_blocks, static_cast<unsigned>((heads + split.per_block - 1) / split.per_block));
  return split.unroll == 1 ? launch(sage_rotary_kernel<T, D, 1>, grid, kRotaryThreads, 0, stream, p)
                           : launch(sage_rotary_kernel<T, D, 4>, grid, kRotaryThreads, 0, stream, p);
}

template <typename T, int D>
int launch_append(const AppendParams& p, const HeadSplit& split, unsigned token_blocks, cudaStream_t stream) {
  const int heads = p.Hq + 2 * p.Hkv;
  const dim3 grid(token_blocks, static_cast<unsigned>((heads + split.per_block - 1) / split.per_block));
  return split.unroll == 1 ? launch(sage_paged_append_kernel<T, D, 1>, grid, kRotaryThreads, 0, stream, p)
                           : launch(sage_paged_append_kernel<T, D, 4>, grid, kRotaryThreads, 0, stream, p);
}

int check_cache(const sage_paged_kv_t* c) {
  SAGE_REQUIRE(c->D == 64 || c->D == 128, "head_dim must be 64 or 128, got %d", c->D);
  SAGE_REQUIRE(c->dtype == SAGE_DTYPE_F16 || c->dtype == SAGE_DTYPE_BF16, "the cache must be fp16 or bf16");
  SAGE_REQUIRE(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
               "page_size must be 16, 32, 64, 128 or 256, got %d", c->page_size);
  SAGE_REQUIRE(c->num_pages >= 1 && c->Hkv >= 1, "the cache needs a page and a head");
  SAGE_REQUIRE(c->k != nullptr && c->v != nullptr && aligned16(c->k) && aligned16(c->v), "the pages need 16-byte aligned bases");
  for (int64_t s : {c->k_stride_page, c->k_stride_slot, c->k_stride_head, c->v_stride_page, c->v_stride_slot, c->v_stride_head}) {
    SAGE_REQUIRE(s > 0 && s % 8 == 0, "the strides of the pages must be positive multiples of 8 elements (16-byte access)");
  }
  return SAGE_OK;
}

int check_batch(const sage_paged_batch_t* b) {
  SAGE_REQUIRE(b->B >= 0 && b->T >= 0, "negative sizes");
  SAGE_REQUIRE(b->cu_q != nullptr || b->T == b->B, "without cu_q every sequence has one token: T must be B");
  SAGE_REQUIRE(b->B == 0 || (b->kv_lens != nullptr && b->page_table != nullptr), "null kv_lens or page_table");
  SAGE_REQUIRE(b->table_width >= 0 && b->table_stride >= 0, "negative extent of the page table");
  return SAGE_OK;
}

Batch batch_of(const sage_paged_batch_t* b, const sage_paged_kv_t* c) {
  Batch x;
  x.table = b->page_table;
  x.table_stride = b->table_stride;
  x.table_width = b->table_width;
  x.kv_lens = b->kv_lens;
  x.cu_q = b->cu_q;
  x.B = b->B;
  x.T = b->T;
  x.page_log2 = 0;
  while ((1 << x.page_log2) < c->page_size) ++x.page_log2;
  x.num_pages = c->num_pages;
  return x;
}

}  // namespace

extern "C" {

int sage_apply_rotary(const sage_strided_t* q, const sage_strided_t* q_out, const sage_strided_t* k, const sage_strided_t* k_out,
                      const sage_rotary_t* rotary, int dtype, int B, int Hq, int Hkv, int S, int D, int inverse, void* stream) {
  SAGE_REQUIRE(q != nullptr && q_out != nullptr && rotary != nullptr, "rotary: null argument");
  SAGE_REQUIRE((k == nullptr) == (k_out == nullptr) && (k != nullptr || Hkv == 0), "rotary: k and k_out come together");
  SAGE_REQUIRE(D == 64 || D == 128, "head_dim must be 64 or 128, got %d", D);
  SAGE_REQUIRE(dtype == SAGE_DTYPE_F16 || dtype == SAGE_DTYPE_BF16 || dtype == SAGE_DTYPE_F32, "rotary: dtype must be fp16, bf16 or fp32");
  SAGE_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && S >= 0, "negative sizes");
  int rc = check_rotary(rotary, D);
  if (rc) return rc;
  if (B == 0 || S == 0 || Hq + Hkv == 0) return SAGE_OK;
  SAGE_REQUIRE(rotary->positions != nullptr, "rotary: null positions");
  const int unit = dtype == SAGE_DTYPE_F32 ? 4 : 8;
  for (const sage_strided_t* t : {q, q_out, k, k_out}) {
    if (t == nullptr || ((t == q || t == q_out) && Hq == 0)) continue;
    SAGE_REQUIRE(t->ptr != nullptr && aligned16(t->ptr) && stride_ok(t->stride_b, unit) && stride_ok(t->stride_h, unit) && stride_ok(t->stride_s, unit),
                 "rotary: tensors need a 16-byte aligned base and strides that are multiples of 16 bytes");
  }
  RotaryParams p;
  memset(&p, 0, sizeof(p));
  auto span = [](const sage_strided_t* in, const sage_strided_t* out) {
    HeadSpan x;
    x.in = in->ptr; x.out = const_cast<void*>(out->ptr);
    x.in_b = in->stride_b; x.in_h = in->stride_h; x.in_s = in->stride_s;
    x.out_b = out->stride_b; x.out_h = out->stride_h; x.out_s = out->stride_s;
    return x;
  };
  p.q = span(q, q_out);
  if (k != nullptr) p.k = span(k, k_out);
  p.rotary = rotary_of(rotary, inverse);
  p.B = B; p.S = S; p.Hq = Hq; p.Hkv = Hkv;
  const int per_block = kRotaryThreads / (D / 16);
  const long long blocks = (static_cast<long long>(B) * S + per_block - 1) / per_block;
  SAGE_REQUIRE(blocks <= 0x7fffffffLL, "rotary: too many tokens");
  HeadSplit split;
  rc = split_heads(&split, blocks, Hq + Hkv);
  if (rc) return rc;
  SAGE_REQUIRE((Hq + Hkv + split.per_block - 1) / split.per_block <= 65535, "rotary: too many heads");
  p.heads_per_block = split.per_block;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned n = static_cast<unsigned>(blocks);
  if (dtype == SAGE_DTYPE_F32) return D == 64 ? launch_rotary<float, 64>(p, split, n, st) : launch_rotary<float, 128>(p, split, n, st);
  if (dtype == SAGE_DTYPE_F16) return D == 64 ? launch_rotary<__half, 64>(p, split, n, st) : launch_rotary<__half, 128>(p, split, n, st);
  return D == 64 ? launch_rotary<__nv_bfloat16, 64>(p, split, n, st) : launch_rotary<__nv_bfloat16, 128>(p, split, n, st);
}

int sage_paged_append(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, const sage_rows_t* k, const sage_rows_t* v,
                      const sage_rows_t* q, const sage_rows_t* q_out, int Hq, const sage_rotary_t* rotary, int* status, void* stream) {
  SAGE_REQUIRE(cache != nullptr && batch != nullptr && k != nullptr && v != nullptr, "append: null argument");
  SAGE_REQUIRE((q == nullptr) == (q_out == nullptr) && (q != nullptr ? Hq >= 0 : Hq == 0), "append: q and q_out come together");
  int rc = check_cache(cache);
  if (rc) return rc;
  rc = check_batch(batch);
  if (rc) return rc;
  if (rotary != nullptr) {
    rc = check_rotary(rotary, cache->D);
    if (rc) return rc;
  }
  SAGE_REQUIRE(q == nullptr || rotary != nullptr, "append: q is only turned, which needs rotary");
  if (batch->T == 0 || batch->B == 0) return SAGE_OK;
  SAGE_REQUIRE(rows_ok(k) && rows_ok(v) && (q == nullptr || Hq == 0 || (rows_ok(q) && rows_ok(q_out))),
               "append: rows need a 16-byte aligned base and strides that are multiples of 8 elements");
  AppendParams p;
  memset(&p, 0, sizeof(p));
  if (q != nullptr) {
    p.q.in = q->ptr; p.q.in_h = q->stride_h; p.q.in_s = q->stride_t;
    p.q.out = const_cast<void*>(q_out->ptr); p.q.out_h = q_out->stride_h; p.q.out_s = q_out->stride_t;
  }
  p.k.in = k->ptr; p.k.in_h = k->stride_h; p.k.in_s = k->stride_t;
  p.k.out = cache->k; p.k.out_b = cache->k_stride_page; p.k.out_h = cache->k_stride_head; p.k.out_s = cache->k_stride_slot;
  p.v.in = v->ptr; p.v.in_h = v->stride_h; p.v.in_s = v->stride_t;
  p.v.out = cache->v; p.v.out_b = cache->v_stride_page; p.v.out_h = cache->v_stride_head; p.v.out_s = cache->v_stride_slot;
  p.rotary = rotary_of(rotary, 0);
  p.batch = batch_of(batch, cache);
  p.status = status_of(status);
  p.Hq = Hq; p.Hkv = cache->Hkv;
  const int per_block = kRotaryThreads / (cache->D / 16);
  const unsigned blocks = static_cast<unsigned>((static_cast<long long>(batch->T) + per_block - 1) / per_block);
  HeadSplit split;
  rc = split_heads(&split, blocks, Hq + 2 * cache->Hkv);
  if (rc) return rc;
  SAGE_REQUIRE((Hq + 2 * cache->Hkv + split.per_block - 1) / split.per_block <= 65535, "append: too many heads");
  p.heads_per_block = split.per_block;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == SAGE_DTYPE_F16) return cache->D == 64 ? launch_append<__half, 64>(p, split, blocks, st) : launch_append<__half, 128>(p, split, blocks, st);
  return cache->D == 64 ? launch_append<__nv_bfloat16, 64>(p, split, blocks, st) : launch_append<__nv_bfloat16, 128>(p, split, blocks, st);
}

}  // extern "C"
