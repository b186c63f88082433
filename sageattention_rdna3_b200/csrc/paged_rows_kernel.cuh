// Attention of a few rows over a paged cache: single tokens, drafted tokens.
//
// o_r = sum_j 2^(s_rj - m) v_j / sum_j 2^(s_rj - m), s = q.k sm_scale log2 e, one pass over the keys with the running
// maximum m.  With a handful of rows per key the cache is read once and everything else is small: the bound is HBM
// (D=128: 512 bytes per key and kv head against 4 D flops per row).  So the split follows the loads: a CTA per SM takes an
// equal span of 128-key tiles (paged_schedule.cuh).  A producer warp walks through it and keeps a ring of TMA loads full (192 KB in
// flight per SM), across items, with the rows of Q of the next item: what it has to look up - lengths, pages -
// it asks for ahead of its use.  Of every tile each of four warps takes 32 keys with a running maximum and sum of
// its own; they meet only at the end of an item.
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

constexpr int kRowsThreads = 160;
constexpr int kRowsWarps = 4;                         // that compute
constexpr int kUnitKeys = 32;                         // keys of a tile that one of them takes

// CTAs of an SM.  A key tile of D=64 is half the bytes and two thirds of the instructions of one of D=128: two CTAs share the SM.
// (With 32 rows their shared memory does not fit.)
constexpr int rows_ctas_per_sm(int D, int MT) { return D == 64 && MT == 1 ? 2 : 1; }

template <int D, int MT>
struct RowsSmem {
  static constexpr int kRows = 16 * MT;
  static constexpr int kStages = D == 128 || MT == 1 ? 3 : 6;
  static constexpr int kTile = kTileKeys * D * 2;     // K or V: box after box, each [D / 64][keys][64 values], 128-byte swizzle
  static constexpr int kStage = 2 * kTile;
  static constexpr int kItems = 2;                    // items ahead: segment and rows of Q
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kJoinRows = 8;                 // rows that the warps join at a time
  static constexpr int kJoinStride = D + 8;
  static constexpr int kOffQ = kStages * kStage;
  static constexpr int kOffJoin = kOffQ + kItems * kQBytes;
  static constexpr int kOffStats = kOffJoin + kRowsWarps * kJoinRows * kJoinStride * 4;     // m, l of every warp and row
  static constexpr int kOffSegments = kOffStats + 2 * kRowsWarps * kRows * 4;
  static constexpr int kOffBar = kOffSegments + kItems * static_cast<int>(sizeof(Segment));
  static constexpr int kNumBars = 2 * kStages + 2 * kItems + 1;
  static constexpr int kOffScratch = kOffBar + kNumBars * 8;
  static constexpr int kOffMisc = kOffScratch + static_cast<int>(sizeof(SpanScratch));
  static constexpr int kTotal = kOffMisc + 16;
  static_assert((kTotal + 1024) * rows_ctas_per_sm(D, MT) <= 233472, "shared memory of an SM");
};

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

// 16 bytes from global to shared memory; counted on an mbarrier by cp_async_arrive.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kRowsThreads, rows_ctas_per_sm(D, MT))
sage_paged_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
  using L = RowsSmem<D, MT>;
  constexpr int kRows = L::kRows, kStages = L::kStages, kItems = L::kItems;
  constexpr float kBias = std::is_same<T, __half>::value ? 15.0f : 0.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* empty = full + kStages;
  uint64_t* item_full = empty + kStages;
  uint64_t* item_empty = item_full + kItems;
  uint64_t* joined = item_empty + kItems;
  Segment* segments = reinterpret_cast<Segment*>(smem + L::kOffSegments);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc);
  const bool misaligned = (smem_u32(smem) & 1023u) != 0u;    // (the swizzled slabs need it)
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kRowsWarps);
    }
    for (int s = 0; s < kItems; ++s) {
      mbar_init(item_full + s, 33);                   // every lane's part of Q, and the segment
      mbar_init(item_empty + s, kRowsWarps);
    }
    mbar_init(joined, kRowsWarps);
    fence_mbar_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  grid_dependency_wait();
  if (threadIdx.x == kRowsThreads - 1) {               // (a thread that has no sequence to look up, as a rule)
    // a wait of an earlier launch that ran out and was not looked at yet: this launch does nothing (as attn_kernel.cuh)
    const int before = p.status.word != nullptr ? *reinterpret_cast<volatile int*>(p.status.word) : 0;
    *abort_flag = misaligned || status_stops(before);
    if (misaligned) p.status.report(kStatusMisaligned);
    p.headers[blockIdx.x].n_parts = 0;
  }
  const Span span = find_span<kRowsThreads>(p, reinterpret_cast<SpanScratch*>(smem + L::kOffScratch));
  grid_launch_dependents();
  if (*abort_flag) return;

  if (warp == kRowsWarps) {
    // ------------------------------------------------------------------ producer
    const bool leader = elect_one();
    const int box_rows = min(1 << p.batch.page_log2, kTileKeys);
    const int slot_mask = (1 << p.batch.page_log2) - 1;
    SegmentIter it(p, span);
    bool ok = true;
    int tiles = 0;                                    // so far
    int checked = 0;                                  // pages of the 32 boxes at hand
    // Pages are looked up 32 at a time, a lane each, the next 32 while these are loaded.  (64 sequences of 60 to 16000 keys in pages
    // of 16, us per call, a lookup per tile / per 32 pages: 138 / 130.)
    const int block_tiles = 32 * box_rows / kTileKeys;
    int pages = 0;
    auto find_pages = [&](const Segment& g, int j) {  // from tile j on
      const int key = g.key0 + j * kTileKeys + lane * box_rows;
      if (key < g.len) pages = page_of_key(p, g.b, key);
    };
#pragma unroll 1
    for (int item = 0; ok; ++item) {
      const int slot = item % kItems;
      const Segment g = it.next();
      if (g.n_tiles > 0) find_pages(g, 0);
      ok = warp_wait<true>(item_empty + slot, ((item / kItems) & 1) ^ 1u, abort_flag, p.wait_limit_cycles);
      if (!ok) break;
      if (g.n_tiles > 0) {
        // Rows without a token stay what they are: no row's result depends on another's.
        constexpr int kPerRow = 32 / kRows, kChunks = D / 8 / kPerRow;         // lanes of a row, 16-byte pieces of each
        const int r = lane / kPerRow, c0 = lane % kPerRow * kChunks;
        int token = 0, head = 0;
        if (row_at(p, g.q0, g.n_q, g.head0, g.row0, kRows, r, &token, &head)) {
          const T* src = static_cast<const T*>(p.q) + token * p.q_stride_t + head * p.q_stride_h;
          const uint32_t s_q = smem_u32(smem + L::kOffQ + slot * L::kQBytes) + r * (D * 2);
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int c = c0 + i;
            cp_async16(s_q + ((c & ~7) << 4) + (((c ^ r) & 7) << 4), src + c * 8);
          }
        }
      }
      if (lane == 0) segments[slot] = g;
      cp_async_arrive(item_full + slot);
      if (lane == 0) mbar_arrive(item_full + slot);
      if (g.n_tiles == 0) break;
#pragma unroll 1
      for (int j = 0; j < g.n_tiles; ++j, ++tiles) {
        const int stage = tiles % kStages;
        ok = warp_wait<true>(empty + stage, ((tiles / kStages) & 1) ^ 1u, abort_flag, p.wait_limit_cycles);
        if (!ok) break;
        uint8_t* dst = smem + stage * L::kStage;
        const int first = g.key0 + j * kTileKeys, in_block = j & (block_tiles - 1);
        if (in_block == 0) {
          checked = checked_page(p, pages);
          if (j + block_tiles < g.n_tiles) find_pages(g, j + block_tiles);
        }
        int boxes = (min(max(g.len - first, 0), kTileKeys) + box_rows - 1) / box_rows;
        if (p.test_drop_load && tiles == 0) boxes = 0;                       // failure-detection test: this stage never fills
        else if (leader) mbar_arrive_expect_tx(full + stage, boxes * box_rows * D * 2 * 2);
#pragma unroll 1
        for (int x = 0; x < boxes; ++x) {
          const int page = __shfl_sync(0xffffffffu, checked, in_block * kTileKeys / box_rows + x);
          if (leader) {
            tma_load_5d(dst + x * box_rows * (D * 2), &tm_k, full + stage, 0, first & slot_mask, 0, g.kv_head, page);
            tma_load_5d(dst + L::kTile + x * box_rows * (D * 2), &tm_v, full + stage, 0, first & slot_mask, 0, g.kv_head, page);
          }
        }
      }
    }
    if (!ok) {
      if (lane == 0) p.status.report(kStatusWait);
      // A launch that gave up waits (for a bounded time again) for its own copies in flight.
      volatile int* again = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
      *again = 0;
      for (int n = max(tiles - kStages, 0); n < tiles; ++n) warp_wait<true>(full + n % kStages, (n / kStages) & 1, again, p.wait_limit_cycles);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  // -------------------------------------------------------------------- work
  // Where this warp's 32 keys of a tile are: `at`, keys 16-31 `upper` behind 0-15, the next 64 values `slab` behind.
  const int box_rows = min(1 << p.batch.page_log2, kTileKeys);
  const uint32_t slab = box_rows * 128, upper = box_rows == 16 ? 16 * D * 2 : 16 * 128;
  const uint32_t at = (warp * kUnitKeys & ~(box_rows - 1)) * (D * 2) + (warp * kUnitKeys & (box_rows - 1)) * 128;
  float* s_join = reinterpret_cast<float*>(smem + L::kOffJoin);
  float* s_m = reinterpret_cast<float*>(smem + L::kOffStats);
  float* s_l = s_m + kRowsWarps * kRows;
  bool ok = true;
  int tiles = 0;
  // A barrier of the four warps whose wait is bounded: one of them may have given up.
  uint32_t joins = 0;
  auto warps_sync = [&]() -> bool {
    __syncwarp();
    if (lane == 0) mbar_arrive(joined);
    ok = ok && warp_wait<false>(joined, joins++ & 1, abort_flag, p.wait_limit_cycles);
    return ok;
  };
#pragma unroll 1
  for (int item = 0;; ++item) {
    const int q_slot = item % kItems;
    ok = ok && warp_wait<false>(item_full + q_slot, (item / kItems) & 1, abort_flag, p.wait_limit_cycles);
    if (!ok) break;
    const Segment g = segments[q_slot];
    if (g.n_tiles == 0) break;
    const uint32_t s_q = smem_u32(smem + L::kOffQ + q_slot * L::kQBytes);
    const int live_rows = min(kRows, g.n_q * p.group - g.row0);
    // this thread's rows of the accumulators: lane / 4 and 8 below, of every 16
    int limit[MT][2];
    int least = g.len;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        int token, head, lim = 0;
        bool live = row_at(p, g.q0, g.n_q, g.head0, g.row0, kRows, mt * 16 + half * 8 + lane / 4, &token, &head);
        if (live) {
          if (p.shared_pass) {
            int q1;
            const int b = seq_of_token(p, token, &q1);
            live = b < p.batch.B;
            if (live) lim = min(g.len, visible_keys(p, b, q1, token));
          } else {
            lim = p.causal ? max(0, g.len - (g.q0 + g.n_q - 1 - token)) : g.len;
          }
        }
        limit[mt][half] = lim;
        if (live) least = min(least, lim);
      }
    least = __reduce_min_sync(0xffffffffu, least);

    // (rows 0-7 and 8-15, values 0-7 and 8-15 of every 16: the A operand).  With 32 rows there are no registers to keep it in.
    auto load_q = [&](int mt, int k, uint32_t (&a)[4]) {
      const int r = mt * 16 + (lane & 15), c = 2 * k + (lane >> 4);
      ldmatrix_x4(s_q + r * (D * 2) + ((c & ~7) << 4) + (((c ^ r) & 7) << 4), a);
    };
    uint32_t qf[MT == 1 ? D / 16 : 1][4];
    if constexpr (MT == 1) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) load_q(0, k, qf[k]);
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty + q_slot);
    }

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
    for (int j = 0; j < g.n_tiles; ++j, ++tiles) {
      const int stage = tiles % kStages;
      ok = ok && warp_wait<false>(full + stage, (tiles / kStages) & 1, abort_flag, p.wait_limit_cycles);
      if (!ok) break;
      const int first = g.key0 + j * kTileKeys + warp * kUnitKeys;
      const int keys = min(kUnitKeys, g.len - first);
      if (keys > 0) {
        const uint32_t s_k = smem_u32(smem + stage * L::kStage) + at, s_v = s_k + L::kTile;

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
          uint32_t a[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if constexpr (MT == 1) {
#pragma unroll
              for (int i = 0; i < 4; ++i) a[mt][i] = qf[k][i];
            } else {
              load_q(mt, k, a[mt]);
            }
          }
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {
            // matrices: (keys 0-7, values 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) of a 16 x 16 block
            const int key = (lane >> 4) * 8 + (lane & 7);
            const int chunk = (k % 4) * 2 + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix_x4(s_k + (k / 4) * slab + n2 * upper + key * 128 + ((chunk ^ (key & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_16816(s[mt][2 * n2], a[mt], b[0], b[1], static_cast<const T*>(nullptr));
              mma_16816(s[mt][2 * n2 + 1], a[mt], b[2], b[3], static_cast<const T*>(nullptr));
            }
          }
        }

        uint32_t pf[MT][2][4];                        // P as the A operand, 16 keys each
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[mt][n][i] *= p.score_scale;
          if (first + kUnitKeys > least) {            // (some row does not see all keys)
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
            const float base = top[half] == -INFINITY ? 0.0f : top[half];    // (a row that has seen nothing yet)
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
            const int key = ((lane >> 3) & 1) * 8 + (lane & 7);
            const int chunk = (n2 % 4) * 2 + (lane >> 4);
            uint32_t b[4];
            ldmatrix_x4_trans(s_v + (n2 / 4) * slab + k * upper + key * 128 + ((chunk ^ (key & 7)) << 4), b);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_16816(o[mt][2 * n2], pf[mt][k], b[0] & mask0, b[1] & mask1, static_cast<const T*>(nullptr));
              mma_16816(o[mt][2 * n2 + 1], pf[mt][k], b[2] & mask0, b[3] & mask1, static_cast<const T*>(nullptr));
            }
          }
        }
        __syncwarp();                                 // all lanes have read the stage
      }
      if (lane == 0) mbar_arrive(empty + stage);
    }
    if (!ok) break;
    if (MT > 1 && lane == 0) mbar_arrive(item_empty + q_slot);

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
    if (g.slot == 1 && threadIdx.x == 0) {
      p.headers[blockIdx.x] = PartHeader{g.n_parts, g.q0, g.n_q, g.head0, g.row0, kRows, {0, 0}};
    }
#pragma unroll 1
    for (int pass = 0; pass * 8 < live_rows; ++pass) {          // rows 8 * pass to 8 * pass + 7
      if (pass > 0 && !warps_sync()) break;           // the buffer has been read
      float* dst = s_join + (warp * 8 + lane / 4) * L::kJoinStride + (lane % 4) * 2;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        float2 x = make_float2(o[0][n][0], o[0][n][1]);
#pragma unroll
        for (int i = 1; i < 2 * MT; ++i) {
          if (pass == i) x = make_float2(o[i / 2][n][2 * (i % 2)], o[i / 2][n][2 * (i % 2) + 1]);
        }
        *reinterpret_cast<float2*>(dst + n * 8) = x;
      }
      if (!warps_sync()) break;
#pragma unroll 1
      for (int i = threadIdx.x; i < 8 * D / 4; i += 128) {
        const int r8 = i / (D / 4), r = pass * 8 + r8, col = (i - r8 * (D / 4)) * 4;
        if (r >= live_rows) break;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, s_m[w * kRows + r]);
        float out[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(s_join + (w * 8 + r8) * L::kJoinStride + col);
          const float f = top == -INFINITY ? 1.0f : ex2(s_m[w * kRows + r] - top);
          out[0] += f * y.x; out[1] += f * y.y; out[2] += f * y.z; out[3] += f * y.w;
          sum += f * s_l[w * kRows + r];
        }
        const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
#pragma unroll
        for (int c = 0; c < 4; ++c) out[c] = sum == 0.0f ? 0.0f : out[c] * inv;    // (of a row without keys: 0 * V)
        if (g.slot >= 0) {
          const long long at = (static_cast<long long>(blockIdx.x) * 2 + g.slot) * kRows + r;
          store_floats(p.part_o + at * D + col, out);
          if (col == 0) p.part_e[at] = part_lse(top - kBias, sum);
        } else {
          int token, head;
          bool live = row_at(p, g.q0, g.n_q, g.head0, g.row0, kRows, r, &token, &head);
          if (live && p.shared_pass) {
            int q1;
            live = seq_of_token(p, token, &q1) < p.batch.B;
          }
          if (live) write_row<T, 4>(p, token, head, D, col, out, sum == 0.0f ? -INFINITY : top - kBias + log2f(sum), col == 0);
        }
      }
    }
    if (!warps_sync()) break;                         // statistics and buffer are free again
  }
  if (ok) zero_rest<T>(p, D, threadIdx.x, 128);
  else if (lane == 0) p.status.report(kStatusWait);
}

}  // namespace paged
}  // namespace sage
