// How attention over a paged cache is cut into work for a fixed grid, without the host knowing a length.
//
// An item is one row tile of one kv head of one sequence: up to `tile_rows` rows (new token, query head of the group) that
// read the same keys, those up to the last key that its last token sees.  It costs `item_cost` steps for its start and end
// and then some per tile of 128 keys (at least one tile: an item without keys writes zeros).  The steps of all items, sequence
// after sequence, kv head after kv head, row tile after row tile, form one line that is cut into equal spans, one per CTA:
// lengths may differ as they like and all CTAs get the same amount of work.  A key tile belongs to the CTA that has its first
// step.  A span that covers part of an item leaves its result in a slot of the workspace (slot 1 the head of an item, slot 0
// anything else: at most one of each per CTA) and a header that tells the merge kernels which parts follow.  Every CTA works
// this out for itself from kv_lens and cu_q, by a block-wide prefix sum; nothing is communicated and the order of all sums is
// fixed.  Both are read more than once.  A program that changes them before the call is through gets numbers that mean
// nothing, but every walk ends and every access stays in its tensor: what is derived from a sequence comes from one reading of it, and
// walks end with the last sequence and the last CTA.
#pragma once

#include "paged_common.cuh"

namespace sage {
namespace paged {

constexpr int kTileKeys = 128;

// Division of numbers below 2^31 by a constant that the host knows: a multiplication and a shift.
struct FastDiv {
  uint32_t mul;                 // 0: the divisor is 1
  int shift;
  __host__ static FastDiv of(int d) {
    FastDiv f{0, 0};
    int s = 0;
    while ((2 << s) <= d) ++s;                        // 2^s <= d < 2^(s+1)
    if ((1 << s) == d) {
      if (s > 0) f = FastDiv{0x80000000u, s - 1};
    } else {
      f = FastDiv{static_cast<uint32_t>(((1ull << (32 + s)) + d - 1) / d), s};
    }
    return f;
  }
  __device__ __forceinline__ int operator()(int n) const {
    return mul == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), mul) >> shift);
  }
};

// (Small code matters here: a kernel of this file runs for tens of microseconds, and its instructions come from the L2 or
// from memory at first.  What is called once an item stands once, in loops that are not unrolled.)
__device__ __noinline__ long long long_div(long long a, long long b) { return a / b; }
__device__ __forceinline__ long long floor_div(long long a, long long b) {
  if (a <= 0x7fffffffLL && b <= 0x7fffffffLL) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return long_div(a, b);
}

struct AttnParams {
  const void* q;
  long long q_stride_t, q_stride_h;
  void* o;                      // 16-bit output, or null: `o32` is written
  long long o_stride_t, o_stride_h;
  float* o32;                   // [T, Hq, D] fp32 and [T, Hq] base-2 log-sum-exp: the result as one part of a larger one
  float* e32;
  const float* prior_o;         // ... and such a part to be merged with on writing `o`, or null
  const float* prior_e;
  float* lse;                   // optional [T, Hq], natural log
  Batch batch;                  // of the sequences; cu_q and kv_lens also give the visible keys of every row
  Status status;
  const int32_t* shared_pages;  // keys [0, shared_len) of every sequence, or null
  int shared_len;
  int shared_pass;              // 1: one sequence of all T tokens against the shared keys; 0: every sequence against its keys behind them
  int Hq, Hkv, group;           // group = Hq / Hkv
  int tile_rows;                // rows of a row tile
  FastDiv by_group, by_tile_rows;
  int item_cost;                // steps that stand for the start and end of an item
  int tile_cost;                // steps of a key tile; and ...
  int light_cost;               // ... where the item has at most half the rows of a row tile
  int causal;
  int zero_rest;                // write zeros to rows that belong to no sequence
  float score_scale;            // sm_scale * log2(e)
  float* part_o;                // [grid][2][tile rows][D] fp32
  float* part_e;                // [grid][2][tile rows]
  struct PartHeader* headers;   // [grid]
  long long wait_limit_cycles;
  int test_drop_load;           // test hook: one load of the first key tile is left out
};

struct PartHeader {             // of the part in slot 1 of a CTA, if it is the head of an item that others finish
  int n_parts;                  // 0: none
  int token0, tokens;           // new tokens of the sequence: rows [token0, token0 + tokens)
  int head0;                    // first query head of the group
  int row0;                     // first row of the tile, counted (token, head of the group) from the sequence's first token
  int rows;                     // rows in the tile
  int pad[2];
};

// One sequence as the schedule sees it.
struct Seq {
  int q0, n_q;                  // new tokens
  int key0, len;                // keys [key0, len)
  int row_tiles;
  long long head_steps;         // steps of one kv head
};

__device__ __forceinline__ int n_seqs(const AttnParams& p) { return p.shared_pass ? 1 : p.batch.B; }

__device__ __forceinline__ int clipped_len(const AttnParams& p, int b) {
  const long long most = static_cast<long long>(p.batch.table_width) << p.batch.page_log2;
  return static_cast<int>(min(static_cast<long long>(max(p.batch.kv_lens[b], 0)), most));
}

// Key tiles of row tile `rt`, and the steps of one of them.
__device__ __forceinline__ void item_of(const AttnParams& p, const Seq& s, int rt, int* tiles, int* cost) {
  const int last_row = (rt + 1) * p.tile_rows;
  int end = s.len;
  if (p.causal && !p.shared_pass) end -= max(0, s.n_q - (p.by_group(last_row - 1) + 1));
  *tiles = max(1, (end - s.key0 + kTileKeys - 1) / kTileKeys);
  *cost = s.n_q * p.group - rt * p.tile_rows > p.tile_rows / 2 ? p.tile_cost : p.light_cost;
}

__device__ __forceinline__ Seq seq_at(const AttnParams& p, int b) {
  Seq s;
  if (p.shared_pass) {
    s.q0 = 0;
    s.n_q = p.batch.T;
    s.key0 = 0;
    s.len = p.shared_len;
  } else {
    int q1;
    p.batch.tokens(b, &s.q0, &q1);
    s.n_q = q1 - s.q0;
    s.key0 = p.shared_len;
    s.len = clipped_len(p, b);
  }
  s.row_tiles = p.by_tile_rows(s.n_q * p.group + p.tile_rows - 1);
  s.head_steps = 0;
#pragma unroll 1
  for (int rt = 0; rt < s.row_tiles; ++rt) {
    int tiles, cost;
    item_of(p, s, rt, &tiles, &cost);
    s.head_steps += p.item_cost + static_cast<long long>(tiles) * cost;
  }
  return s;
}

__device__ __forceinline__ long long steps_of(const AttnParams& p, const Seq& s) { return s.head_steps * p.Hkv; }

// Keys that a new token sees: [0, limit).
__device__ __forceinline__ int visible_keys(const AttnParams& p, int b, int q1, int token) {
  const int len = clipped_len(p, b);
  return p.causal ? max(0, len - (q1 - 1 - token)) : len;
}
// The sequence of a token, by search (the shared pass, where a row tile spans sequences); B if it belongs to none.
__device__ __forceinline__ int seq_of_token(const AttnParams& p, int token, int* q1) {
  if (p.batch.cu_q == nullptr) {
    *q1 = token + 1;
    return token;
  }
  int lo = 0, hi = p.batch.B;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.batch.cu_q[mid] <= token) lo = mid;
    else hi = mid;
  }
  int q0;
  p.batch.tokens(lo, &q0, q1);
  return token >= q0 && token < *q1 ? lo : p.batch.B;
}

// The span of a CTA and where it starts; found once by all threads together.
struct Span {
  long long t, t_end;           // steps
  long long share;              // CTA c owns share steps, the first `extra` one more
  int extra;
  int ctas;                     // CTAs that have steps at all
  int b;                        // sequence of step t ...
  long long before;             // ... the steps before that sequence, and the sequence
  Seq seq;
};
struct SpanScratch {            // in shared memory
  long long warp_steps[16];
  long long before;
  Seq seq;
  int b;
};

// Ends with a barrier.
template <int kThreads>
__device__ __forceinline__ Span find_span(const AttnParams& p, SpanScratch* scratch) {
  static_assert(kThreads <= 512, "");
  const int n = n_seqs(p);
  const int per = (n + kThreads - 1) / kThreads;
  const int first = threadIdx.x * per, last = min(first + per, n);
  long long mine = 0;
#pragma unroll 1
  for (int b = first; b < last; ++b) {
    mine += steps_of(p, seq_at(p, b));
    if (blockIdx.x == 0 && !p.shared_pass && p.batch.kv_lens[b] > clipped_len(p, b)) p.status.report(kStatusBadLength);
  }
  long long upto = mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long other = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 31) scratch->warp_steps[warp] = upto;
  __syncthreads();
  long long total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) base += scratch->warp_steps[w];
    total += scratch->warp_steps[w];
  }
  upto += base;
  Span s;
  // (a CTA has at least the steps of a key tile: none that stands inside an item is without one)
  const long long most = p.tile_cost == 1 ? total : floor_div(total, p.tile_cost);
  s.ctas = total == 0 ? 0 : static_cast<int>(max(1LL, min(static_cast<long long>(gridDim.x), most)));
  const int c = blockIdx.x;
  const bool idle = c >= s.ctas;
  s.share = floor_div(total, max(s.ctas, 1));
  s.extra = static_cast<int>(total - s.share * s.ctas);
  s.t = idle ? 0 : s.share * c + min(c, s.extra);
  s.t_end = idle ? 0 : s.t + s.share + (c < s.extra ? 1 : 0);
  // The thread whose sequences hold step t walks through them.
  if (!idle && s.t >= upto - mine && s.t < upto) {
    long long before = upto - mine;
    int b = first;
    Seq seq;
#pragma unroll 1
    while (true) {
      seq = seq_at(p, b);
      const long long steps = steps_of(p, seq);
      if (s.t < before + steps || b + 1 == last) break;        // (the latter if lengths change meanwhile)
      before += steps;
      ++b;
    }
    scratch->b = b;
    scratch->before = before;
    scratch->seq = seq;
  }
  __syncthreads();
  s.b = scratch->b;
  s.before = scratch->before;
  s.seq = scratch->seq;
  return s;
}

// A part of a span that belongs to one item, as the producer warp of a CTA tells it to the others.
struct Segment {
  int q0, n_q, len;             // of the sequence
  int key0;                     // first key of the segment's first tile
  int n_tiles;                  // 0: no more segments
  int head0, row0;              // first query head of the group, first row of the tile
  int slot;                     // -1: the whole item; 1: its head, 0: another part
  int n_parts;                  // slot 1: parts of the item
  int b, kv_head;
  int pad;
};

// Walks through a span; by a whole warp, whose lanes look ahead at 32 sequences at a time, so that an item costs no
// round trip to memory.
struct SegmentIter {
  const AttnParams& p;
  Span s;
  int base;                     // lane i holds sequence base + i
  Seq mine;
  Seq seq;                      // of s.b
  long long steps;              // of seq
  int head, rt, tiles, cost;    // the item at hand
  long long item_at;            // its first step
  __device__ __forceinline__ SegmentIter(const AttnParams& pp, const Span& span) : p(pp), s(span), base(-32), seq(span.seq), head(-1) {
    steps = s.t < s.t_end ? steps_of(p, seq) : 0;
  }
  __device__ __forceinline__ void find(int b) {
    const int lane = threadIdx.x & 31;
    if (base < 0 || b >= base + 32) {
      base = b;
      if (b + lane < n_seqs(p)) mine = seq_at(p, b + lane);
    }
    const int from = b - base;
    seq.q0 = __shfl_sync(0xffffffffu, mine.q0, from);
    seq.n_q = __shfl_sync(0xffffffffu, mine.n_q, from);
    seq.key0 = p.shared_pass ? 0 : p.shared_len;
    seq.len = __shfl_sync(0xffffffffu, mine.len, from);
    seq.row_tiles = __shfl_sync(0xffffffffu, mine.row_tiles, from);
    seq.head_steps = __shfl_sync(0xffffffffu, mine.head_steps, from);
    steps = steps_of(p, seq);
    head = -1;
  }
  __device__ __forceinline__ Segment next() {
    Segment g;
    g.n_tiles = 0;
#pragma unroll 1
    while (s.t < s.t_end && g.n_tiles == 0) {
#pragma unroll 1
      while (s.t >= s.before + steps) {               // (sequences without new tokens have no steps)
        s.before += steps;
        if (++s.b >= n_seqs(p)) return g;
        find(s.b);
      }
      if (head < 0) {                                 // the head by division, its row tile step by step
        head = static_cast<int>(floor_div(s.t - s.before, seq.head_steps));
        item_at = s.before + head * seq.head_steps;
        rt = 0;
        item_of(p, seq, rt, &tiles, &cost);
      }
#pragma unroll 1
      while (s.t >= item_at + p.item_cost + static_cast<long long>(tiles) * cost) {
        item_at += p.item_cost + static_cast<long long>(tiles) * cost;
        if (++rt == seq.row_tiles) {
          rt = 0;
          ++head;
        }
        item_of(p, seq, rt, &tiles, &cost);
      }
      const long long item_end = item_at + p.item_cost + static_cast<long long>(tiles) * cost;
      const long long first_tile = item_at + p.item_cost, stop = min(item_end, s.t_end);
      // tiles whose first step is in [t, stop)
      const int lo = s.t <= first_tile ? 0 : static_cast<int>(s.t - first_tile + cost - 1) / cost;
      const int hi = stop <= first_tile ? 0 : static_cast<int>(stop - first_tile + cost - 1) / cost;
      g.n_tiles = hi - lo;
      g.q0 = seq.q0;
      g.n_q = seq.n_q;
      g.len = seq.len;
      g.key0 = seq.key0 + lo * kTileKeys;
      g.kv_head = head;
      g.head0 = head * p.group;
      g.row0 = rt * p.tile_rows;
      g.b = s.b;
      g.n_parts = 1;
      if (lo > 0) {
        g.slot = 0;
      } else if (hi == tiles) {
        g.slot = -1;
      } else {
        g.slot = 1;
        // the CTA that has the first step of the last tile
        const long long e = item_end - cost, longer = s.extra * (s.share + 1);
        const long long c = e < longer ? floor_div(e, s.share + 1) : s.extra + floor_div(e - longer, s.share);
        g.n_parts = min(static_cast<int>(c), s.ctas - 1) - static_cast<int>(blockIdx.x) + 1;
      }
      s.t = stop;
    }
    return g;
  }
};

// Row r of a tile -> new token (counted in the batch) and query head; false if the row is empty.
__device__ __forceinline__ bool row_at(const AttnParams& p, int token0, int tokens, int head0, int row0, int rows, int r, int* token, int* head) {
  if (r >= rows) return false;
  const int flat = row0 + r;
  const int i = p.by_group(flat);
  *token = token0 + i;
  *head = head0 + flat - i * p.group;
  return i < tokens;
}

// Base-2 log-sum-exp of a part with maximum m and sum l.  A part that is not a number gets +inf, which fmaxf keeps where it
// would drop a NaN: the weights of all parts of the row become NaN then.
__device__ __forceinline__ float part_lse(float m, float l) {
  const float e = m + log2f(l);
  return l == 0.0f ? -INFINITY : e != e ? INFINITY : e;
}

// Joins a finished row with what is already known of it: both normalised, with their base-2 log-sum-exp.
__device__ __forceinline__ void join_weights(float e, float prior, float* w, float* w_prior, float* joined) {
  const float top = fmaxf(e, prior);
  if (e == -INFINITY && prior == -INFINITY) {
    *w = *w_prior = 0.0f;
    *joined = -INFINITY;
    return;
  }
  const float a = ex2(e - top), b = ex2(prior - top), inv = __fdividef(1.0f, a + b);
  *w = a * inv;
  *w_prior = b * inv;
  *joined = top + log2f(a + b);
}

template <int N>
__device__ __forceinline__ void store_floats(float* dst, const float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  } else {
    *reinterpret_cast<float2*>(dst) = make_float2(x[0], x[1]);
  }
}
template <int N>
__device__ __forceinline__ void load_floats(const float* src, float (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = reinterpret_cast<const float4*>(src)[i];
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  } else {
    const float2 v = *reinterpret_cast<const float2*>(src);
    x[0] = v.x; x[1] = v.y;
  }
}

// Writes N (2, 4 or a multiple of 8) neighbouring values of a finished row: normalised `x`, log-sum-exp e (base 2).
template <typename T, int N>
__device__ __forceinline__ void write_row(const AttnParams& p, int token, int head, int D, int col, float (&x)[N], float e, bool with_lse) {
  const long long row = static_cast<long long>(token) * p.Hq + head;
  if (p.o == nullptr) {
    store_floats(p.o32 + row * D + col, x);
    if (with_lse) p.e32[row] = e;
    return;
  }
  if (p.prior_o != nullptr) {
    float w, wp, joined;
    join_weights(e, p.prior_e[row], &w, &wp, &joined);
    float y[N];
    load_floats(p.prior_o + row * D + col, y);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = w * x[i] + wp * y[i];
    e = joined;
  }
  T* dst = static_cast<T*>(p.o) + token * p.o_stride_t + head * p.o_stride_h + col;
  uint32_t packed[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) packed[i] = from_float2(x[2 * i], x[2 * i + 1], static_cast<const T*>(nullptr));
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = packed[0];
  }
  if (with_lse && p.lse != nullptr) p.lse[row] = e * 0.6931471805599453f;      // (-inf stays -inf)
}

// Rows that belong to no sequence, as the calling CTA's share of them.  `threads` threads take part, this one is `thread`.
template <typename T>
__device__ __forceinline__ void zero_rest(const AttnParams& p, int D, int thread, int threads) {
  if (!p.zero_rest || p.batch.cu_q == nullptr) return;
  const int first = min(max(p.batch.cu_q[0], 0), p.batch.T), last = min(max(p.batch.cu_q[p.batch.B], 0), p.batch.T);
  const int rest = first + p.batch.T - last;
  const int vecs = p.Hq * (D / 8);
#pragma unroll 1
  for (int i = blockIdx.x; i < rest; i += gridDim.x) {
    const int token = i < first ? i : last + i - first;
#pragma unroll 1
    for (int v = thread; v < vecs; v += threads) {
      const int head = v / (D / 8);
      *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + token * p.o_stride_t + head * p.o_stride_h + (v - head * (D / 8)) * 8) = make_uint4(0, 0, 0, 0);
      if (p.lse != nullptr && v % (D / 8) == 0) p.lse[static_cast<long long>(token) * p.Hq + head] = -INFINITY;
    }
  }
}

// Joins the parts of items.  blockIdx.x: header, blockIdx.y: rows.  Two layouts of a part (tile_rows x D floats), each as its
// writer stores it in whole lines:
//   rows (sage_paged_rows_kernel)  row after row; a warp has one row, kWarps / ROWS warps every so many parts of it
//   columns (sage_paged_tile_kernel, a thread per row)  4 neighbouring values of all rows, then the next 4; here a warp has 32
//   rows and kVecs of their float4 columns (blockIdx.z: which)
// Four parts are in flight together, in the order of the keys: the result does not depend on who came first.
constexpr int kMergeThreads = 256;

template <int N>
struct PartSum {
  float e = -INFINITY, sum = 0.0f, x[N];              // maximum; the row so far is x / sum
  __device__ __forceinline__ PartSum() {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.0f;
  }
  template <int K>
  __device__ __forceinline__ void add(const float (&pe)[K], const float (&px)[K][N]) {
    float top = e;
#pragma unroll
    for (int c = 0; c < K; ++c) top = fmaxf(top, pe[c]);
    if (top == -INFINITY) return;                     // no visible keys so far
    const float back = ex2(e - top);
    sum *= back;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= back;
    e = top;
#pragma unroll
    for (int c = 0; c < K; ++c) {
      const float f = ex2(pe[c] - top);
      sum += f;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += f * px[c][i];
    }
  }
  __device__ __forceinline__ void normalise() {
    const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= inv;
  }
  __device__ __forceinline__ float lse() const { return sum == 0.0f ? -INFINITY : e + log2f(sum); }
};

// The row of a merge thread, if it has one that belongs to a sequence.
__device__ __forceinline__ bool merge_row(const AttnParams& p, const PartHeader& h, int r, int* token, int* head) {
  if (!row_at(p, h.token0, h.tokens, h.head0, h.row0, h.rows, r, token, head)) return false;
  int q1;
  return !p.shared_pass || seq_of_token(p, *token, &q1) < p.batch.B;
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kMergeThreads) sage_paged_merge_rows_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kWarps = kMergeThreads / 32, kRowWarps = kWarps / ROWS, kPer = D / 32;   // values per lane: 4 or 2
  __shared__ float s_o[kWarps][D];
  __shared__ float s_e[kWarps];
  grid_dependency_wait();
  grid_launch_dependents();
  const PartHeader h = p.headers[blockIdx.x];
  if (h.n_parts < 2 || static_cast<long long>(h.tokens) * p.group <= h.row0 + static_cast<int>(blockIdx.y) * ROWS) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.y * ROWS + warp / kRowWarps, w = warp % kRowWarps;
  int token = 0, head = 0;
  const bool live = merge_row(p, h, r, &token, &head);
  PartSum<kPer> acc;
  if (live) {
#pragma unroll 1
    for (int k0 = w; k0 < h.n_parts; k0 += 4 * kRowWarps) {
      float pe[4], px[4][kPer];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int k = k0 + c * kRowWarps;
        pe[c] = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; ++i) px[c][i] = 0.0f;
        if (k < h.n_parts) {
          const long long at = ((static_cast<long long>(blockIdx.x) + k) * 2 + (k == 0 ? 1 : 0)) * p.tile_rows + r;
          pe[c] = p.part_e[at];
          load_floats(p.part_o + at * D + lane * kPer, px[c]);
        }
      }
      acc.add(pe, px);
    }
  }
  acc.normalise();
  if constexpr (kRowWarps > 1) {
    const float e = part_lse(acc.e, acc.sum);
    store_floats(&s_o[warp][lane * kPer], acc.x);
    if (lane == 0) s_e[warp] = e;
    __syncthreads();
    if (w != 0 || !live) return;
    acc = PartSum<kPer>();
#pragma unroll
    for (int c0 = 0; c0 < kRowWarps; c0 += 4) {
      float pe[4], px[4][kPer];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        pe[c] = s_e[warp + c0 + c];
        load_floats(&s_o[warp + c0 + c][lane * kPer], px[c]);
      }
      acc.add(pe, px);
    }
    acc.normalise();
  }
  if (live) write_row<T, kPer>(p, token, head, D, lane * kPer, acc.x, acc.lse(), lane == 0);
}

template <int D>
struct MergeColumns {
  static constexpr int kVecs = 2;                      // float4 columns of a thread; with 4 / 1 the join of 9 parts of 256 rows each takes
  static constexpr int kFlight = 4;                    // 9.8 / 10 us instead of 8.5; parts in flight: with 2 / 8 9.5 / 10.5
  static constexpr int kBlocks = D / 4 / (kMergeThreads / 32 * kVecs);   // of 32 rows
};
template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) sage_paged_merge_columns_kernel(const __grid_constant__ AttnParams p) {
  using M = MergeColumns<D>;
  constexpr int kVecs = M::kVecs, kFlight = M::kFlight;
  grid_dependency_wait();
  grid_launch_dependents();
  const PartHeader h = p.headers[blockIdx.x];
  if (h.n_parts < 2 || static_cast<long long>(h.tokens) * p.group <= h.row0 + static_cast<int>(blockIdx.y) * 32) return;
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), c0 = (blockIdx.z * (kMergeThreads / 32) + (threadIdx.x >> 5)) * kVecs;
  int token = 0, head = 0;
  if (!merge_row(p, h, r, &token, &head)) return;
  PartSum<4 * kVecs> acc;
#pragma unroll 1
  for (int k0 = 0; k0 < h.n_parts; k0 += kFlight) {
    float pe[kFlight], px[kFlight][4 * kVecs];
#pragma unroll
    for (int c = 0; c < kFlight; ++c) {
      const int k = k0 + c;
      pe[c] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4 * kVecs; ++i) px[c][i] = 0.0f;
      if (k < h.n_parts) {
        const long long slot = (static_cast<long long>(blockIdx.x) + k) * 2 + (k == 0 ? 1 : 0);
        pe[c] = p.part_e[slot * p.tile_rows + r];
        const float4* src = reinterpret_cast<const float4*>(p.part_o) + (slot * (D / 4) + c0) * p.tile_rows + r;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
          const float4 v = src[i * p.tile_rows];
          px[c][4 * i] = v.x; px[c][4 * i + 1] = v.y; px[c][4 * i + 2] = v.z; px[c][4 * i + 3] = v.w;
        }
      }
    }
    acc.add(pe, px);
  }
  acc.normalise();
  write_row<T, 4 * kVecs>(p, token, head, D, 4 * c0, acc.x, acc.lse(), c0 == 0);
}

}  // namespace paged
}  // namespace sage
