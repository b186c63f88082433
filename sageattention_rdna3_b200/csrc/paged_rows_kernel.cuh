// Attention of a few rows over a paged cache: single tokens, drafted tokens.
//
// o_r = sum_j 2^(s_rj - m) v_j / sum_j 2^(s_rj - m), s = q.k sm_scale log2 e, one pass over the keys with the running
// maximum m.  With a handful of rows per key the cache is read once and everything else is small: the bound is HBM
// (D=128: 512 bytes per key and kv head against 4 D flops per row).  So the split follows the loads: a CTA per SM takes an
// equal span of key tiles (paged_schedule.cuh); of every 128-key tile each of its four warps takes 32 keys, with a ring
// of TMA loads of its own (kStages x 16 KB at D=128, 192 KB in flight per SM) and its own running maximum and sum.  Warps meet
// only at the end of an item, so none waits for another in between, and the loads of the next item are under way
// while this one is finished.
//
// The products are mma.sync (m16n8k16, fp32 accumulators): the 16 rows of one instruction hold the query heads of a GQA group
// (and the drafted tokens).  tcgen05 has no shape below 64 rows, and its accumulator would go through TMEM to the
// one warp that owns the few rows.
// P is rounded to the type of V as a matrix operand (half a step of 2^-8 or 2^-11 of each weight); fp16 weights are
// taken times 2^15, or those far below the maximum would lose bits to fp16's smallest numbers: a long context behind one
// large score is made of such weights.  Scores, maximum, sum and O are fp32; l is summed before P is rounded.
#pragma once

#include <type_traits>

#include "paged_schedule.cuh"

namespace sage {
namespace paged {

constexpr int kRowsThreads = 128;
constexpr int kUnitKeys = 32;                         // keys of one warp's load

template <int D, int MT>
struct RowsSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kSlab = kUnitKeys * 128;       // 32 keys x 64 values, 128-byte swizzle
  static constexpr int kUnit = 2 * (D / 64) * kSlab;  // K and V
  static constexpr int kMergeCols = 64 / MT;          // columns joined at a time
  static constexpr int kMergeStride = kMergeCols + 8;
  static constexpr int kOffMerge = 4 * kStages * kUnit;
  static constexpr int kOffStats = kOffMerge + 4 * kRows * kMergeStride * 4;     // m, l of every warp and row
  static constexpr int kOffBar = kOffStats + 2 * 4 * kRows * 4;
  static constexpr int kOffScratch = kOffBar + 4 * kStages * 8;
  static constexpr int kOffMisc = kOffScratch + (kRowsThreads / 32 + 4) * 8;
  static constexpr int kTotal = kOffMisc + 16;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __half*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const __nv_bfloat16*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The page that holds key `key` of a segment's sequence, as the table has it, and as it may be loaded: an index outside the cache
// is reported and replaced, the load stays inside the cache whatever the table holds.
__device__ __forceinline__ int page_of_key(const AttnParams& p, int b, int key) {
  const int col = key >> p.batch.page_log2;
  return p.shared_pass ? p.shared_pages[col] : p.batch.table[b * p.batch.table_stride + col];
}
__device__ __forceinline__ int checked_page(const AttnParams& p, int page) {
  if (page >= 0 && page < p.batch.num_pages) return page;
  p.status.report(kStatusBadPage);
  return 0;
}

// The units (32 keys) of one warp in the order in which they are used, across segments.
struct UnitIter {
  SegmentIter it;
  Segment g;
  int tile, left;
  __device__ __forceinline__ UnitIter(const AttnParams& p, const Span& s) : it(p, s), left(0) {}
  // The next unit that has keys: first key and their number (at most 32); false at the end of the span.
  __device__ __forceinline__ bool next(int warp, int* first, int* keys) {
    while (true) {
      if (left == 0) {
        if (!it.next(&g)) return false;
        tile = g.tile;
        left = g.n_tiles;
      }
      *first = g.seq.key0 + tile * kTileKeys + warp * kUnitKeys;
      *keys = min(kUnitKeys, g.seq.len - *first);
      ++tile;
      --left;
      if (*keys > 0) return true;
    }
  }
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kRowsThreads, 1)
sage_paged_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
  using L = RowsSmem<D, MT>;
  constexpr int kRows = L::kRows, kStages = L::kStages, kSlabs = D / 64;
  constexpr float kBias = std::is_same<T, __half>::value ? 15.0f : 0.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + warp * kStages;
  uint8_t* ring = smem + warp * kStages * L::kUnit;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc);
  const bool misaligned = (smem_u32(smem) & 1023u) != 0u;    // (the swizzled slabs need it)
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bars + s, 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    if (warp == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  grid_dependency_wait();
  if (threadIdx.x == 0) {
    // a wait of an earlier launch that ran out and was not looked at yet: this launch does nothing (as attn_kernel.cuh)
    const int before = p.status.word != nullptr ? *reinterpret_cast<volatile int*>(p.status.word) : 0;
    *abort_flag = misaligned || (before & 15) == 2;
    if (misaligned) p.status.report(kStatusMisaligned);
    p.headers[blockIdx.x].n_parts = 0;
  }
  const Span span = find_span<kRowsThreads>(p, reinterpret_cast<long long*>(smem + L::kOffScratch));
  grid_launch_dependents();
  if (*abort_flag) return;

  // ---- loads
  const int box_rows = min(1 << p.batch.page_log2, kUnitKeys);
  UnitIter producer(p, span);
  int issued = 0;
  int next_first = 0, next_keys = 0, next_pages[2] = {0, 0}, next_head = 0;
  bool more = true;
  // Finds the next unit and asks for its pages, which are looked at when it is issued, a unit later.
  auto fetch = [&]() {
    more = producer.next(warp, &next_first, &next_keys);
    if (more) {
      next_head = producer.g.head;
      next_pages[0] = page_of_key(p, producer.g.b, next_first);
      next_pages[1] = 0;
      if (box_rows < kUnitKeys && next_keys > box_rows) next_pages[1] = page_of_key(p, producer.g.b, next_first + box_rows);
    }
  };
  auto issue = [&]() {
    if (lane == 0) {
      uint64_t* bar = bars + issued % kStages;
      uint8_t* dst = ring + (issued % kStages) * L::kUnit;
      const int boxes = box_rows < kUnitKeys && next_keys > box_rows ? 2 : 1;
      const int slot = next_first & ((1 << p.batch.page_log2) - 1);
#pragma unroll
      for (int x = 0; x < 2; ++x) next_pages[x] = checked_page(p, next_pages[x]);
      mbar_arrive_expect_tx(bar, boxes * box_rows * D * 2 * 2);
      for (int x = 0; x < boxes; ++x) {
#pragma unroll
        for (int c = 0; c < kSlabs; ++c) tma_load_4d(dst + c * L::kSlab + x * box_rows * 128, &tm_k, bar, c * 64, slot, next_head, next_pages[x]);
      }
      for (int x = 0; x < boxes; ++x) {
#pragma unroll
        for (int c = 0; c < kSlabs; ++c) tma_load_4d(dst + (kSlabs + c) * L::kSlab + x * box_rows * 128, &tm_v, bar, c * 64, slot, next_head, next_pages[x]);
      }
    }
    ++issued;
  };
  fetch();
#pragma unroll 1
  for (int s = 0; s < kStages && more; ++s) {
    issue();
    fetch();
  }

  // ---- work
  float* s_merge = reinterpret_cast<float*>(smem + L::kOffMerge);
  float* s_m = reinterpret_cast<float*>(smem + L::kOffStats);
  float* s_l = s_m + 4 * kRows;
  int used = 0;
  bool ok = true;
  SegmentIter it(p, span);
  Segment g;
#pragma unroll 1
  while (it.next(&g)) {
    const int row0 = g.row_tile * kRows, head0 = g.head * p.group;
    // this thread's rows of the accumulators: lane / 4 and 8 below, of every 16
    uint32_t qf[MT][D / 16][4];
    int limit[MT][2];
    int least = g.seq.len;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        int token, head;
        bool live = row_at(g.seq.q0, g.seq.n_q, head0, p.group, row0, kRows, mt * 16 + half * 8 + lane / 4, &token, &head);
        int lim = 0;
        if (live) {
          if (p.shared_pass) {
            int q1;
            const int b = seq_of_token(p, token, &q1);
            live = b < p.batch.B;
            if (live) lim = min(g.seq.len, visible_keys(p, b, q1, token));
          } else {
            lim = visible_keys(p, g.b, g.seq.q0 + g.seq.n_q, token);
          }
        }
        limit[mt][half] = lim;
        if (live) least = min(least, lim);
        const T* src = live ? static_cast<const T*>(p.q) + token * p.q_stride_t + head * p.q_stride_h + (lane % 4) * 2 : nullptr;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[mt][k][half] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
          qf[mt][k][2 + half] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) least = min(least, __shfl_xor_sync(0xffffffffu, least, d));

    float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.0f;
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.0f;
    }

#pragma unroll 1
    for (int tile = g.tile; tile < g.tile + g.n_tiles; ++tile) {
      const int first = g.seq.key0 + tile * kTileKeys + warp * kUnitKeys;
      const int keys = min(kUnitKeys, g.seq.len - first);
      if (keys <= 0) continue;
      const int stage = used % kStages;
      if (ok && !warp_wait<false>(bars + stage, (used / kStages) & 1, abort_flag, p.wait_limit_cycles)) {
        ok = false;
        if (lane == 0) p.status.report(kStatusWait);
      }
      if (!ok) continue;
      ++used;
      const uint32_t s_k = smem_u32(ring + stage * L::kUnit), s_v = s_k + kSlabs * L::kSlab;

      // S = Q.K^T: 4 groups of 8 keys
      float s[MT][4][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][n][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2) {
          // matrices: (keys 0-7, values 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) of a 16 x 16 block
          const int key = n2 * 16 + (lane >> 4) * 8 + (lane & 7);
          const int chunk = (k % 4) * 2 + ((lane >> 3) & 1);
          uint32_t b[4];
          ldmatrix_x4(s_k + (k / 4) * L::kSlab + key * 128 + ((chunk ^ (key & 7)) << 4), b);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma_16816(s[mt][2 * n2], qf[mt][k], b[0], b[1], static_cast<const T*>(nullptr));
            mma_16816(s[mt][2 * n2 + 1], qf[mt][k], b[2], b[3], static_cast<const T*>(nullptr));
          }
        }
      }

      uint32_t pf[MT][2][4];                          // P as the A operand, 16 keys each
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][n][i] *= p.score_scale;
        if (first + kUnitKeys > least) {              // (some row does not see all keys)
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = first + n * 8 + (lane % 4) * 2 + (i & 1);
              if (key >= limit[mt][i >> 1]) s[mt][n][i] = -INFINITY;
            }
        }
        float top[2] = {m[mt][0], m[mt][1]};
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], s[mt][n][i]);
        float neg[2], back[2];
        bool moved = false;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
          top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
          moved |= top[half] > m[mt][half];
          const float base = top[half] == -INFINITY ? 0.0f : top[half];      // (a row that has seen nothing yet)
          back[half] = ex2(m[mt][half] - base);
          neg[half] = kBias - base;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            l[mt][half] *= back[half];
            m[mt][half] = top[half];
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              o[mt][n][2 * half] *= back[half];
              o[mt][n][2 * half + 1] *= back[half];
            }
          }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[mt][n][i] = ex2(s[mt][n][i] + neg[i >> 1]);
            l[mt][i >> 1] += s[mt][n][i];
          }
          pf[mt][n / 2][(n & 1) * 2] = from_float2(s[mt][n][0], s[mt][n][1], static_cast<const T*>(nullptr));
          pf[mt][n / 2][(n & 1) * 2 + 1] = from_float2(s[mt][n][2], s[mt][n][3], static_cast<const T*>(nullptr));
        }
      }

      // O += P.V.  Behind the last key a page holds whatever it held: those values of V are taken as zero (0 * NaN is NaN).
      const bool partial = keys < kUnitKeys;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t mask0 = 0xffffffffu, mask1 = 0xffffffffu;
        if (partial) {
          const int key = k * 16 + (lane % 4) * 2;
          mask0 = (key < keys ? 0xffffu : 0u) | (key + 1 < keys ? 0xffff0000u : 0u);
          mask1 = (key + 8 < keys ? 0xffffu : 0u) | (key + 9 < keys ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int n2 = 0; n2 < D / 16; ++n2) {
          // matrices: (keys 0-7, values 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15) of a 16 x 16 block, transposed
          const int key = k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
          const int chunk = (n2 % 4) * 2 + (lane >> 4);
          uint32_t b[4];
          ldmatrix_x4_trans(s_v + (n2 / 4) * L::kSlab + key * 128 + ((chunk ^ (key & 7)) << 4), b);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma_16816(o[mt][2 * n2], pf[mt][k], b[0] & mask0, b[1] & mask1, static_cast<const T*>(nullptr));
            mma_16816(o[mt][2 * n2 + 1], pf[mt][k], b[2] & mask0, b[3] & mask1, static_cast<const T*>(nullptr));
          }
        }
      }
      __syncwarp();                                   // all lanes have read the stage
      if (more) {
        issue();
        fetch();
      }
    }

    // ---- the four warps' parts become one
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 1);
        l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 2);
        if (lane % 4 == 0) {
          s_m[warp * kRows + mt * 16 + half * 8 + lane / 4] = m[mt][half];
          s_l[warp * kRows + mt * 16 + half * 8 + lane / 4] = l[mt][half];
        }
      }
    __syncthreads();
    if (g.slot == 1 && threadIdx.x == 0) {
      p.headers[blockIdx.x] = PartHeader{g.n_parts, g.seq.q0, g.seq.n_q, head0, row0, kRows, {0, 0}};
    }
    const bool dead = *abort_flag != 0;               // (uniform: set before the barrier, or by a later wait that ends all the same)
    float mine[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = mt * 16 + half * 8 + lane / 4;
        const float top = fmaxf(fmaxf(s_m[r], s_m[kRows + r]), fmaxf(s_m[2 * kRows + r], s_m[3 * kRows + r]));
        mine[mt][half] = top == -INFINITY ? 1.0f : ex2(m[mt][half] - top);
      }
#pragma unroll
    for (int pass = 0; pass < D / L::kMergeCols; ++pass) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < L::kMergeCols / 8; ++n)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float* x = &o[mt][pass * (L::kMergeCols / 8) + n][2 * half];
            float* dst = s_merge + (warp * kRows + mt * 16 + half * 8 + lane / 4) * L::kMergeStride + n * 8 + (lane % 4) * 2;
            *reinterpret_cast<float2*>(dst) = make_float2(x[0] * mine[mt][half], x[1] * mine[mt][half]);
          }
      __syncthreads();
      constexpr int kGroups = kRows * L::kMergeCols / 4;
#pragma unroll
      for (int i = threadIdx.x; i < kGroups; i += kRowsThreads) {
        const int r = i / (L::kMergeCols / 4), c = (i - r * (L::kMergeCols / 4)) * 4;
        int token, head;
        bool live = !dead && row_at(g.seq.q0, g.seq.n_q, head0, p.group, row0, kRows, r, &token, &head);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, s_m[w * kRows + r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_merge + (w * kRows + r) * L::kMergeStride + c);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          sum += s_l[w * kRows + r] * (top == -INFINITY ? 1.0f : ex2(s_m[w * kRows + r] - top));
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        float out[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
        const int col = pass * L::kMergeCols + c;
        if (g.slot >= 0) {
          const long long at = (static_cast<long long>(blockIdx.x) * 2 + g.slot) * kRows + r;
          *reinterpret_cast<float4*>(p.part_o + at * D + col) = make_float4(out[0], out[1], out[2], out[3]);
          if (col == 0) p.part_e[at] = part_lse(top - kBias, sum);
        } else if (live) {
          if (p.shared_pass) {
            int q1;
            live = seq_of_token(p, token, &q1) < p.batch.B;
          }
          if (live) write_row<T, 4>(p, token, head, D, col, out, sum == 0.0f ? -INFINITY : top - kBias + log2f(sum), col == 0);
        }
      }
      __syncthreads();
    }
  }
  zero_rest<T>(p, D, threadIdx.x, kRowsThreads);
  // a launch that gave up waits (for a bounded time again) for its own copies in flight
  if (!ok) {
    volatile int* again = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
    *again = 0;
    for (int u = used; u < issued; ++u) mbar_wait<false>(bars + u % kStages, (u / kStages) & 1, again, p.wait_limit_cycles);
  }
}

}  // namespace paged
}  // namespace sage
