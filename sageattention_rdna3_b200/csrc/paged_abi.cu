// Host side of the C ABI declared in include/sage_paged_b200.h: argument checks, choice of the kernel, launches.  No torch
// types, no allocation, no synchronisation.
#include "../../include/sage_paged_b200.h"

#include <algorithm>

#include "host_common.h"
#include "paged_tile_kernel.cuh"
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
  SAGE_REQUIRE(r->freq != nullptr && r->axis != nullptr && aligned16(r->freq) && aligned16(r->axis), "rotary: the table needs 16-byte aligned bases");
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

// Heads per block of the rotary and append kernels: 8, or as many as leave every SM its blocks; 2 for few tokens, whose
// time is the latency of a call (117 tokens, 60 heads, us with 2 / 4 / 8: 3.8 / 5.0 / 6.6).
int split_heads(int* per_block, long long token_blocks, int heads) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  for (int n : {8, 4, 2}) {
    *per_block = n;
    if (token_blocks * ((heads + n - 1) / n) >= static_cast<long long>(kRotaryBlocks) * sms) break;
  }
  return SAGE_OK;
}

template <typename T, int D>
int launch_rotary(const RotaryParams& p, unsigned token_blocks, cudaStream_t stream) {
  const int heads = p.Hq + p.Hkv;
  const dim3 grid(token_blocks, static_cast<unsigned>((heads + p.heads_per_block - 1) / p.heads_per_block));
  return launch(sage_rotary_kernel<T, D>, grid, kRotaryThreads, 0, stream, p);
}

template <typename T, int D>
int launch_append(const AppendParams& p, unsigned token_blocks, cudaStream_t stream) {
  const int heads = p.Hq + 2 * p.Hkv;
  const dim3 grid(token_blocks, static_cast<unsigned>((heads + p.heads_per_block - 1) / p.heads_per_block));
  return launch(sage_paged_append_kernel<T, D>, grid, kRotaryThreads, 0, stream, p);
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
  SAGE_REQUIRE(b->B == 0 || (b->kv_lens != nullptr && (b->page_table != nullptr || b->table_width == 0)), "null kv_lens or page_table");
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

// One pass of attention over the cache: which kernel, how many CTAs, and what it needs of the workspace.
struct PagedPlan {
  bool tensor = false;          // sage_paged_tile_kernel
  int tile_rows = 0;
  int item_cost = 0, tile_cost = 1, light_cost = 1;
  int grid = 0;
  bool merge = false;           // an item may be cut
  int64_t header_bytes = 0, e_bytes = 0, o_bytes = 0;
  int64_t bytes() const { return header_bytes + e_bytes + o_bytes; }
};
int64_t round16(int64_t n) { return (n + 15) & ~int64_t{15}; }

// seqs: sequences of the pass, max_q: new tokens of one of them, tokens: of all; max_keys: keys of one.
int plan_pass(PagedPlan* plan, const sage_paged_kv_t* c, int64_t seqs, int64_t tokens, int64_t max_q, int64_t max_keys, int group) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  *plan = PagedPlan();
  const int64_t rows = std::min(max_q, tokens) * group;
  plan->tensor = rows > 32;
  plan->tile_rows = plan->tensor ? 2 * (kTileM / group) * group : rows <= 16 ? 16 : 32;
  // Steps.  With few rows a key tile costs the same whatever the rows.  On tensor cores a key tile with one / two row tiles takes, D=128,
  // 1.64 / 2.07 us, D=64 1.37 / 1.80; us of chunks of prompts next to single tokens, the costs taken as 2 to 5 / 3 to 5 / 4 to 5 /
  // 5 to 5 / 3 to 4: 246 / 179 / 165 / 170 / 162.  With few rows the start and end of an item take a key
  // tile for every 8 rows, which the warps join one after the other (the most rows that an item may have: counted for every item by the
  // device the small calls lost 0.1 to 1.7 us).  us for 0 / 1 / 2 key tiles, 4 rows, 64 sequences of 60 to 16000 keys:
  // 137 / 125 / 126; for 1 / 2 / 3 / 4, 12 to 20 rows, 32 sequences of 500 to 6000 keys: 70 / 66 / 64 / 66; for 2 / 3 / 4, 24 rows, 128 sequences
  // of up to 800: 92 / 84 / 86, 32 rows, 64 sequences of 50 to 3000: 115 / 104 / 98.
  if (plan->tensor) {
    plan->item_cost = 10;
    plan->tile_cost = 4;
    plan->light_cost = 3;
  } else {
    plan->item_cost = static_cast<int>((rows + 7) / 8);
  }
  const int64_t tiles = std::max<int64_t>(1, (max_keys + kTileKeys - 1) / kTileKeys);
  const int64_t row_tiles = tokens * group / plan->tile_rows + seqs;
  const int64_t slots = static_cast<int64_t>(sms) * (plan->tensor ? 1 : rows_ctas_per_sm(c->D, plan->tile_rows / 16));
  plan->grid = static_cast<int>(std::min<int64_t>(slots, std::min<int64_t>(row_tiles * c->Hkv, slots) * tiles));
  plan->merge = tiles > 1;
  plan->header_bytes = round16(static_cast<int64_t>(plan->grid) * sizeof(PartHeader));
  plan->e_bytes = round16(static_cast<int64_t>(plan->grid) * 2 * plan->tile_rows * sizeof(float));
  plan->o_bytes = plan->merge ? static_cast<int64_t>(plan->grid) * 2 * plan->tile_rows * c->D * static_cast<int64_t>(sizeof(float)) : 0;
  return SAGE_OK;
}

struct CallPlan {
  PagedPlan own, shared;
  int64_t joined_o_bytes = 0, joined_e_bytes = 0;     // what the sequences' own keys give, before the shared ones join
  int64_t bytes() const { return std::max(own.bytes(), shared.bytes()) + joined_o_bytes + joined_e_bytes; }
};
int plan_call(CallPlan* plan, const sage_paged_kv_t* c, const sage_paged_batch_t* b, int Hq, int max_q, int n_shared) {
  const int group = Hq / c->Hkv;
  int longest = b->cu_q == nullptr ? 1 : b->T;
  if (max_q > 0) longest = std::min(longest, max_q);
  const int64_t own_keys = static_cast<int64_t>(std::max(0, b->table_width - n_shared)) * c->page_size;
  int rc = plan_pass(&plan->own, c, b->B, b->T, longest, own_keys, group);
  if (rc || n_shared == 0) return rc;
  rc = plan_pass(&plan->shared, c, 1, b->T, b->T, static_cast<int64_t>(n_shared) * c->page_size, group);
  plan->joined_o_bytes = static_cast<int64_t>(b->T) * Hq * c->D * static_cast<int64_t>(sizeof(float));
  plan->joined_e_bytes = round16(static_cast<int64_t>(b->T) * Hq * sizeof(float));
  return rc;
}

template <typename T, int D, int MT>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const AttnParams& p, const PagedPlan& plan, cudaStream_t stream) {
  constexpr int kSmem = RowsSmem<D, MT>::kTotal;
  static std::atomic<bool> configured[64];
  const int rc = configure_smem(sage_paged_rows_kernel<T, D, MT>, kSmem, configured);
  if (rc) return rc;
  return launch(sage_paged_rows_kernel<T, D, MT>, static_cast<unsigned>(plan.grid), kRowsThreads, kSmem, stream, tk, tv, p);
}

template <typename T, int D>
int launch_tile(const CUtensorMap& tk, const CUtensorMap& tv, const AttnParams& p, const PagedPlan& plan, CUtensorMapDataType dt, cudaStream_t stream) {
  constexpr int kSmem = TileSmem<D>::kTotal;
  static std::atomic<bool> configured[64];
  int rc = configure_smem(sage_paged_tile_kernel<T, D>, kSmem, configured);
  if (rc) return rc;
  // Q as (D, heads, tokens), a box: 64 values, the heads of a group, as many tokens as fill a tile.  A dimension of extent 1
  // may carry any stride in the caller's tensor; it gets the span of the others.
  const cuuint64_t row = static_cast<cuuint64_t>(D) * 2;
  cuuint64_t sh = static_cast<cuuint64_t>(p.q_stride_h) * 2, st = static_cast<cuuint64_t>(p.q_stride_t) * 2;
  if (p.Hq == 1) sh = p.batch.T > 1 ? st * p.batch.T : row;
  if (p.batch.T == 1) st = p.Hq > 1 ? sh * p.Hq : row;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(p.Hq), static_cast<cuuint64_t>(p.batch.T)};
  const cuuint64_t strides[2] = {sh, st};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(plan.tile_rows / 2 / p.group)};
  CUtensorMap tq;
  rc = encode_map(&tq, dt, 3, p.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "q");
  if (rc) return rc;
  return launch(sage_paged_tile_kernel<T, D>, static_cast<unsigned>(plan.grid), kTileThreads, kSmem, stream, tq, tk, tv, p);
}

// Map of keys or values, a box: `rows` tokens of one head in one page (up to a whole key tile).  For the tensor cores 64 values
// of them, in a 4-D map; else all values, 64 behind 64, in a 5-D map (half as many loads to issue).
int encode_pages(CUtensorMap* map, CUtensorMapDataType dt, const sage_paged_kv_t* c, const void* base, int64_t slot, int64_t head, int64_t page,
                 bool tensor, const char* what) {
  const int rows = std::min(c->page_size, kTileKeys);
  if (tensor) return encode_strided_16bit(map, dt, base, c->D, c->page_size, c->Hkv, c->num_pages, slot, head, page, rows, what);
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(c->page_size), static_cast<cuuint64_t>(c->D / 64), static_cast<cuuint64_t>(c->Hkv),
                              static_cast<cuuint64_t>(c->num_pages)};
  // (a dimension of extent 1 may carry any stride in the caller's tensor; it gets the span of the others)
  if (c->num_pages == 1) page = std::max(slot * c->page_size, c->Hkv > 1 ? head * c->Hkv : 0);
  if (c->Hkv == 1) head = page;
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(slot) * 2, 128, static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(page) * 2};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(rows), static_cast<cuuint32_t>(c->D / 64), 1, 1};
  return encode_map(map, dt, 5, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

template <typename T, int D>
int launch_pass(const sage_paged_kv_t* c, AttnParams p, const PagedPlan& plan, char* workspace, cudaStream_t stream) {
  p.tile_rows = plan.tile_rows;
  p.item_cost = plan.item_cost;
  p.tile_cost = plan.tile_cost;
  p.light_cost = plan.light_cost;
  p.by_group = FastDiv::of(p.group);
  p.by_tile_rows = FastDiv::of(p.tile_rows);
  p.headers = reinterpret_cast<PartHeader*>(workspace);
  p.part_e = reinterpret_cast<float*>(workspace + plan.header_bytes);
  p.part_o = reinterpret_cast<float*>(workspace + plan.header_bytes + plan.e_bytes);
  const CUtensorMapDataType dt = c->dtype == SAGE_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tk, tv;
  int rc = encode_pages(&tk, dt, c, c->k, c->k_stride_slot, c->k_stride_head, c->k_stride_page, plan.tensor, "k_pages");
  if (rc) return rc;
  rc = encode_pages(&tv, dt, c, c->v, c->v_stride_slot, c->v_stride_head, c->v_stride_page, plan.tensor, "v_pages");
  if (rc) return rc;
  if (plan.tensor) {
    rc = launch_tile<T, D>(tk, tv, p, plan, dt, stream);
    if (rc || !plan.merge) return rc;
    return launch(sage_paged_merge_columns_kernel<T, D>, dim3(static_cast<unsigned>(plan.grid), static_cast<unsigned>((plan.tile_rows + 31) / 32), MergeColumns<D>::kBlocks),
                  kMergeThreads, 0, stream, p);
  }
  rc = plan.tile_rows == 16 ? launch_rows<T, D, 1>(tk, tv, p, plan, stream) : launch_rows<T, D, 2>(tk, tv, p, plan, stream);
  if (rc || !plan.merge) return rc;
  return launch(sage_paged_merge_rows_kernel<T, D, 2>, dim3(static_cast<unsigned>(plan.grid), static_cast<unsigned>(plan.tile_rows / 2)), kMergeThreads, 0, stream, p);
}

int dispatch_pass(const sage_paged_kv_t* c, const AttnParams& p, const PagedPlan& plan, char* workspace, cudaStream_t stream) {
  if (c->dtype == SAGE_DTYPE_F16) return c->D == 64 ? launch_pass<__half, 64>(c, p, plan, workspace, stream) : launch_pass<__half, 128>(c, p, plan, workspace, stream);
  return c->D == 64 ? launch_pass<__nv_bfloat16, 64>(c, p, plan, workspace, stream) : launch_pass<__nv_bfloat16, 128>(c, p, plan, workspace, stream);
}

int check_attn(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, int Hq, int max_q, int n_shared) {
  SAGE_REQUIRE(cache != nullptr && batch != nullptr, "paged attention: null argument");
  int rc = check_cache(cache);
  if (rc) return rc;
  rc = check_batch(batch);
  if (rc) return rc;
  SAGE_REQUIRE(Hq >= 1 && Hq % cache->Hkv == 0 && Hq / cache->Hkv <= 128, "num_qo_heads must be a multiple of num_kv_heads, at most 128 times it; got %d and %d", Hq, cache->Hkv);
  SAGE_REQUIRE(max_q >= 0 && n_shared >= 0, "negative sizes");
  SAGE_REQUIRE(static_cast<int64_t>(batch->T) * Hq <= 0x7fff0000, "paged attention: too many rows");
  SAGE_REQUIRE(static_cast<int64_t>(n_shared) * cache->page_size <= 0x3fffffff && static_cast<int64_t>(batch->table_width) * cache->page_size <= 0x3fffffff,
               "a sequence may have at most 2^30 keys");
  SAGE_REQUIRE(n_shared <= batch->table_width || batch->B == 0, "the page table has fewer columns than there are shared pages");
  return SAGE_OK;
}

}  // namespace

extern "C" {

int64_t sage_paged_workspace_bytes(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, int Hq, int max_q, int n_shared) {
  if (check_attn(cache, batch, Hq, max_q, n_shared) != SAGE_OK) return -1;
  if (batch->T == 0 || batch->B == 0) return 0;
  CallPlan plan;
  return plan_call(&plan, cache, batch, Hq, max_q, n_shared) == SAGE_OK ? plan.bytes() : -1;
}

int sage_paged_attn(const sage_paged_kv_t* cache, const sage_paged_batch_t* batch, const sage_rows_t* q, const sage_rows_t* o, int Hq,
                    int max_q, int is_causal, float sm_scale, float* lse, const int32_t* shared_pages, int n_shared, int zero_rest,
                    int* status, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_attn(cache, batch, Hq, max_q, n_shared);
  if (rc) return rc;
  SAGE_REQUIRE(q != nullptr && o != nullptr, "paged attention: null argument");
  if (batch->T == 0 || batch->B == 0) return SAGE_OK;
  SAGE_REQUIRE(rows_ok(q) && rows_ok(o), "paged attention: rows need a 16-byte aligned base and strides that are multiples of 8 elements");
  SAGE_REQUIRE((batch->T <= 1 || q->stride_t > 0) && (Hq == 1 || q->stride_h > 0), "paged attention: the strides of q must be positive");
  SAGE_REQUIRE(n_shared == 0 || shared_pages != nullptr, "paged attention: null shared_pages");
  CallPlan plan;
  rc = plan_call(&plan, cache, batch, Hq, max_q, n_shared);
  if (rc) return rc;
  SAGE_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= plan.bytes(),
               "paged attention: the workspace must be 16-byte aligned and have %lld bytes", static_cast<long long>(plan.bytes()));
  AttnParams p;
  memset(&p, 0, sizeof(p));
  p.q = q->ptr; p.q_stride_t = q->stride_t; p.q_stride_h = q->stride_h;
  p.o = const_cast<void*>(o->ptr); p.o_stride_t = o->stride_t; p.o_stride_h = o->stride_h;
  p.lse = lse;
  p.batch = batch_of(batch, cache);
  p.status = status_of(status);
  p.shared_len = n_shared * cache->page_size;
  p.shared_pages = shared_pages;
  p.Hq = Hq; p.Hkv = cache->Hkv; p.group = Hq / cache->Hkv;
  p.causal = is_causal != 0;
  p.zero_rest = zero_rest != 0;
  p.score_scale = sm_scale * 1.4426950408889634f;
  p.wait_limit_cycles = g_wait_limit_cycles.load(std::memory_order_relaxed);
  p.test_drop_load = g_test_drop_v_load.load(std::memory_order_relaxed) != 0 && p.wait_limit_cycles < sage::kWaitLimitCycles;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (n_shared == 0) return dispatch_pass(cache, p, plan.own, ws, st);
  // The sequences' own keys first, into fp32; the pass over the shared keys joins them on writing the output.
  AttnParams own = p;
  own.o = nullptr;
  own.lse = nullptr;
  own.zero_rest = 0;
  own.o32 = reinterpret_cast<float*>(ws + std::max(plan.own.bytes(), plan.shared.bytes()));
  own.e32 = own.o32 + static_cast<int64_t>(batch->T) * Hq * cache->D;
  rc = dispatch_pass(cache, own, plan.own, ws, st);
  if (rc) return rc;
  p.shared_pass = 1;
  p.prior_o = own.o32;
  p.prior_e = own.e32;
  return dispatch_pass(cache, p, plan.shared, ws, st);
}

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
    if (t == nullptr || (t == q || t == q_out ? Hq : Hkv) == 0) continue;
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
  SAGE_REQUIRE((Hq + Hkv + 1) / 2 <= 65535, "rotary: too many heads");
  rc = split_heads(&p.heads_per_block, blocks, Hq + Hkv);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned n = static_cast<unsigned>(blocks);
  if (dtype == SAGE_DTYPE_F32) return D == 64 ? launch_rotary<float, 64>(p, n, st) : launch_rotary<float, 128>(p, n, st);
  if (dtype == SAGE_DTYPE_F16) return D == 64 ? launch_rotary<__half, 64>(p, n, st) : launch_rotary<__half, 128>(p, n, st);
  return D == 64 ? launch_rotary<__nv_bfloat16, 64>(p, n, st) : launch_rotary<__nv_bfloat16, 128>(p, n, st);
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
  SAGE_REQUIRE((Hq + 2 * cache->Hkv + 1) / 2 <= 65535, "append: too many heads");
  rc = split_heads(&p.heads_per_block, blocks, Hq + 2 * cache->Hkv);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == SAGE_DTYPE_F16) return cache->D == 64 ? launch_append<__half, 64>(p, blocks, st) : launch_append<__half, 128>(p, blocks, st);
  return cache->D == 64 ? launch_append<__nv_bfloat16, 64>(p, blocks, st) : launch_append<__nv_bfloat16, 128>(p, blocks, st);
}

}  // extern "C"
