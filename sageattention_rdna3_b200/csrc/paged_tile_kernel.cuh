// Attention of many rows over a paged cache: chunks of prompts, and a whole batch against the prefix that it shares.
//
// The mathematics is that of paged_rows_kernel.cuh; with many rows per key tile the products are the work (4 D flops per
// row and key against 4 D bytes per key), so they go to the tensor cores through tcgen05.  A CTA owns two tiles of up to 128 rows, the
// query heads of a GQA group for 128 / group new tokens each (one TMA box), and streams 128-key tiles past both:
//   warp 8     TMA producer  Q; K and V tiles page by page (a box per page, or per 128 keys of a larger page), two stages
//   warp 9+q   MMA issuer    S_q = Q_q.K^T, O_q += P_q.V, fp32 accumulators in TMEM
//   warps 4q.. softmax of tile q: thread t owns row t, running maximum and sum in fp32, P back into TMEM over S
// Q.K^T of one half of a key tile runs while the softmax is at the other half, and each row tile has an issuer of its own, or one would
// wait for the other's rows: with Q.K^T of whole key tiles the scores of the next tile came only when P.V was through,
// and the same work as below took 159 us instead of 133 (though 64 columns are read from shared memory at 3/4 of
// the tensor cores' rate).  Two row tiles to a key tile also halve what is fetched through the L2.  A second tile without rows (fewer
// than 128 rows in all) is left out.
// The grid is a persistent CTA per SM over equal spans of key tiles (paged_schedule.cuh); loads and the first Q.K^T of the next item
// run under the end of this one.  TMEM columns: [128 q, 128 q + 128) S_q, in place P_q (16-bit pairs); [256 + D q, ..) O_q.
//
// Masks: a row sees the keys below its limit.  Behind the last key of a sequence pages hold anything; the softmax warps
// write zeros over those rows of V before the product reads them (0 * NaN is NaN), and pages behind it are not
// loaded at all.  Weights are 2^(s - m + 7): an optimistic pass takes them against the maximum so far, which moves only when
// 64 of them add up to more than 2^15, and for fp16 the smallest numbers (2^-24) are 2^-31 of the largest weight.
// P is rounded to the type of V; the sum is taken before that.
#pragma once

#include "paged_rows_kernel.cuh"

namespace sage {
namespace paged {

constexpr int kTileThreads = 384;
constexpr int kSoftmaxWarps = 8;
constexpr int kTileM = 128;
constexpr int kHalfKeys = 64;
constexpr int kTileTmemCols = 512;
constexpr int kColO = 256;
constexpr float kTileBias = 7.0f;                     // log2 of the largest weight while the maximum stands still
constexpr float kTileLazy = 8.0f;                     // growth of the maximum that is let pass: weights up to 2^15
constexpr float kTileSumMax = 32768.0f;
constexpr float kTileRefusedLazy = 2.0f;              // 64 weights add up to more than 2^15: one is above 2^9

// Every fourth pair of weights is computed without the exponential unit (exp2_by_polynomial).  us, 128 rows of 32 heads on 8
// against 65536 shared keys, D=128 / D=64: none 136 / 120, every eighth 131 / 117, fourth 133 / 113, third 133 / 115.
constexpr int kHandEvery = 4;

template <int D>
struct TileSmem {
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kQBytes = kTileM * D * 2;      // of one row tile
  static constexpr int kKVBytes = kTileKeys * D * 2;
  static constexpr int kSlab = 128 * 128;             // 128 rows x 64 values, 128-byte swizzle
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kQBytes;
  static constexpr int kOffV = kOffK + kStages * kKVBytes;
  static constexpr int kOffBar = kOffV + kStages * kKVBytes;
  static constexpr int kItems = 2;                    // items ahead
  static constexpr int kNumBars = 18 + 4 * kStages + 2 * kItems;
  static constexpr int kOffSegments = kOffBar + 8 * kNumBars;
  static constexpr int kOffScratch = kOffSegments + kItems * static_cast<int>(sizeof(Segment));
  static constexpr int kOffMisc = kOffScratch + static_cast<int>(sizeof(SpanScratch));
  static constexpr int kTotal = kOffMisc + 16;
};

// 2^x for two numbers on the multipliers instead of the exponential unit: x = n + f with f in [-1/2, 1/2] by adding and
// taking away 1.5 2^23, 2^f by a polynomial of degree 5 (fitted for the smallest largest relative error, 2^-23.7 in exact arithmetic), n
// into the exponent.  Below 2^-126 it stays there.  `high` collects the largest x: above 16 the result is not to be
// used.  Not a number comes out as 3.4e38.
__device__ __forceinline__ float2 exp2_by_polynomial(float x0, float x1, float* high) {
  *high = fmaxf(*high, fmaxf(x0, x1));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x0) : "f"(-126.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x1) : "f"(-126.0f));
  auto both = [](float c) { return pack2(c, c); };
  const f32x2_t x = pack2(x0, x1);
  const f32x2_t t = fadd2(x, both(12582912.0f));
  const f32x2_t f = ffma2(fadd2(t, both(-12582912.0f)), both(-1.0f), x);
  f32x2_t y = ffma2(f, both(0.001327647191654736f), both(0.009675541333844113f));
  y = ffma2(f, y, both(0.05550713273732967f));
  y = ffma2(f, y, both(0.24022119723855265f));
  y = ffma2(f, y, both(0.6931469670646163f));
  y = ffma2(f, y, both(1.0000000716546804f));
  const float2 n = unpack2(t), r = unpack2(y);
  return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

// Row tiles of a segment that have rows.
__device__ __forceinline__ int n_row_tiles(const AttnParams& p, const Segment& g) {
  return static_cast<long long>(g.n_q) * p.group - g.row0 > p.tile_rows / 2 ? 2 : 1;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
sage_paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const AttnParams p) {
  using L = TileSmem<D>;
  constexpr int kStages = L::kStages, kSlabs = D / 64;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* s_q = smem + L::kOffQ;
  uint8_t* s_k = smem + L::kOffK;
  uint8_t* s_v = smem + L::kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;     // every Q.K^T of the item is complete
  uint64_t* o_final = bars + 2;     // [2] every P.V of the item's row tile is complete
  uint64_t* o_free = bars + 4;      // [2] all four warps of the tile hold its O in registers
  uint64_t* s_full = bars + 6;      // [2][2] half h of S_q holds Q_q.K_h^T
  uint64_t* p_full = bars + 10;     // [2][2] half h of P_q is written (and O_q scaled) by all four warps of the tile
  uint64_t* pv_done = bars + 14;    // [2][2] O_q += P_q.V over half h is complete
  uint64_t* k_full = bars + 18;
  uint64_t* v_full = bars + 18 + kStages;
  uint64_t* k_empty = bars + 18 + 2 * kStages;      // (by both issuers)
  uint64_t* v_empty = bars + 18 + 3 * kStages;
  uint64_t* item_full = bars + 18 + 4 * kStages;               // [kItems] the segment is written
  uint64_t* item_empty = bars + 18 + 4 * kStages + L::kItems;  // ... and read by the issuers and the eight softmax warps
  Segment* segments = reinterpret_cast<Segment*>(smem + L::kOffSegments);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  int* fail_code = reinterpret_cast<int*>(smem + L::kOffMisc + 8);
  const bool misaligned = (smem_u32(smem) & 1023u) != 0u;

  if (warp == 8 && elect_one()) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int q = 0; q < 2; ++q) {
      mbar_init(o_final + q, 1);
      mbar_init(o_free + q, 4);
      for (int h = 0; h < 2; ++h) {
        mbar_init(s_full + 2 * q + h, 1);
        mbar_init(p_full + 2 * q + h, 4);
        mbar_init(pv_done + 2 * q + h, 1);
      }
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(v_full + s, 1);
      mbar_init(k_empty + s, 2);
      mbar_init(v_empty + s, 2);
    }
    for (int s = 0; s < L::kItems; ++s) {
      mbar_init(item_full + s, 1);
      mbar_init(item_empty + s, 10);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  grid_dependency_wait();
  if (warp == 9) {                                    // (after the wait: attn_kernel.cuh)
    tmem_alloc(tmem_slot, kTileTmemCols);
    tmem_relinquish();
  }
  if (threadIdx.x == kTileThreads - 1) {               // (a thread that has no sequence to look up, as a rule)
    const int before = p.status.word != nullptr ? *reinterpret_cast<volatile int*>(p.status.word) : 0;
    *abort_flag = misaligned || status_stops(before);
    *fail_code = 0;
    if (misaligned) p.status.report(kStatusMisaligned);
    p.headers[blockIdx.x].n_parts = 0;
  }
  tc_fence_before();
  const Span span = find_span<kTileThreads>(p, reinterpret_cast<SpanScratch*>(smem + L::kOffScratch));
  tc_fence_after();
  grid_launch_dependents();
  const uint32_t tmem_base = *tmem_slot;
  const bool dead_on_arrival = *abort_flag != 0;

// SAGE_PAGED_WAIT_OR: by one thread.  SAGE_PAGED_WARP_WAIT_OR: by a whole warp, whose lanes go on or give up together.
#define SAGE_PAGED_WAIT_OR(hinted, bar_ptr, parity, bar_id, action)                 \
  if (!mbar_wait<hinted>((bar_ptr), (parity), abort_flag, p.wait_limit_cycles)) {   \
    atomicCAS(fail_code, 0, 2 + 16 * (bar_id));                                     \
    action;                                                                         \
  }
#define SAGE_PAGED_WARP_WAIT_OR(hinted, bar_ptr, parity, bar_id, action)            \
  if (!warp_wait<hinted>((bar_ptr), (parity), abort_flag, p.wait_limit_cycles)) {   \
    atomicCAS(fail_code, 0, 2 + 16 * (bar_id));                                     \
    action;                                                                         \
  }

  // ------------------------------------------------------------------ MMA issuers
  // Each for its row tile, in halves of 64 keys: QK(0,0) QK(0,1) | PV(0,0) QK(1,0) | PV(0,1) QK(1,1) | ...  The tile is a constant of the code: the operands of tensor
  // instructions are uniform registers, and addresses that depend on the thread's warp number would be moved there one by one.
  auto issue_products = [&](auto tile_tag) {
    constexpr int q = decltype(tile_tag)::value;
    constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t kIdescQK = umma_idesc(1, kFmt, kFmt, 0, 0, kTileM, kHalfKeys);
    constexpr uint32_t kIdescPV = umma_idesc(1, kFmt, kFmt, 0, 1, kTileM, D);              // V MN-major
    const uint32_t t_s = tmem_base + q * kTileKeys, t_o = tmem_base + kColO + q * D;
    int kt = 0, qt = 0, live_items = 0;             // key tiles so far, those of this row tile, items in which it had rows
    bool ok = true;
    auto issue_qk = [&](int stage, int h) {
      // slabs of [128 rows][64 values], 8 rows = 1024 bytes; an instruction takes 16 values = 32 bytes, half h of K starts
      // 64 rows into each slab
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t slab = (k / 4) * L::kSlab;
        const uint64_t dq = umma_smem_desc(smem_u32(s_q + q * L::kQBytes + slab), 16, 1024, kSwizzle128B) + 2 * (k % 4);
        const uint64_t dk = umma_smem_desc(smem_u32(s_k + stage * L::kKVBytes + slab + h * (kHalfKeys * 128)), 16, 1024, kSwizzle128B) + 2 * (k % 4);
        mma_f16_ss(t_s + h * kHalfKeys, dq, dk, kIdescQK, k > 0 ? 1u : 0u);
      }
      tc_commit(s_full + 2 * q + h);
      if (h == 1) tc_commit(k_empty + stage);
    };
#pragma unroll 1
    for (int items = 0; ok; ++items) {
      SAGE_PAGED_WAIT_OR(false, item_full + items % L::kItems, (items / L::kItems) & 1, 34, { ok = false; break; });
      const int n_tiles = segments[items % L::kItems].n_tiles;
      const bool idle = q >= n_row_tiles(p, segments[items % L::kItems]);
      mbar_arrive(item_empty + items % L::kItems);
      if (n_tiles == 0) break;
      SAGE_PAGED_WAIT_OR(false, q_full, items & 1, 24, { ok = false; break; });
      if (idle) {                                   // lets every stage go as it comes: phases are counted by all
        for (int j = 0; ok && j < n_tiles; ++j, ++kt) {
          const int s = kt % kStages;
          SAGE_PAGED_WAIT_OR(false, k_full + s, (kt / kStages) & 1, 25, { ok = false; break; });
          mbar_arrive(k_empty + s);
          SAGE_PAGED_WAIT_OR(false, v_full + s, (kt / kStages) & 1, 27, { ok = false; break; });
          mbar_arrive(v_empty + s);
        }
        mbar_arrive(q_empty);
        continue;
      }
      SAGE_PAGED_WAIT_OR(false, k_full + kt % kStages, (kt / kStages) & 1, 25, { ok = false; break; });
      tc_fence_after();
      issue_qk(kt % kStages, 0);
      issue_qk(kt % kStages, 1);
      if (n_tiles == 1) tc_commit(q_empty);
      // the first P.V of an item overwrites O: the O of the item before must have been read
      if (live_items > 0) SAGE_PAGED_WAIT_OR(false, o_free + q, (live_items - 1) & 1, 28, { ok = false; break; });
#pragma unroll 1
      for (int j = 0; j < n_tiles; ++j, ++qt) {
        const int t = kt + j, s = t % kStages, s1 = (t + 1) % kStages;
        // (the loads first: what follows P is the chain that the softmax waits for)
        SAGE_PAGED_WAIT_OR(false, v_full + s, (t / kStages) & 1, 27, { ok = false; break; });
        if (j + 1 < n_tiles) SAGE_PAGED_WAIT_OR(false, k_full + s1, ((t + 1) / kStages) & 1, 29, { ok = false; break; });
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          SAGE_PAGED_WAIT_OR(false, p_full + 2 * q + h, qt & 1, 26, { ok = false; break; });
          tc_fence_after();
          // V: [128 keys][64 values] slabs; half h starts 64 rows = 8192 bytes in, an instruction takes 16 rows = 2048 bytes
          const uint64_t dv = umma_smem_desc(smem_u32(s_v + s * L::kKVBytes + h * (kHalfKeys * 128)), L::kSlab, 1024, kSwizzle128B);
#pragma unroll
          for (int k = 0; k < kHalfKeys / 16; ++k) {
            mma_f16_ts(t_o, t_s + h * kHalfKeys + 8 * k, dv + 128 * k, kIdescPV, (j > 0 || h > 0 || k > 0) ? 1u : 0u);
          }
          tc_commit(pv_done + 2 * q + h);
          if (j + 1 < n_tiles) issue_qk(s1, h);
        }
        if (!ok) break;
        if (j + 1 == n_tiles) tc_commit(o_final + q);
        tc_commit(v_empty + s);
        if (j + 2 == n_tiles) tc_commit(q_empty);
      }
      ++live_items;
      kt += n_tiles;
    }
  };

  if (dead_on_arrival) {
    // nothing to do
  } else if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    const bool leader = elect_one();
    const int box_rows = min(1 << p.batch.page_log2, kTileKeys);
    const int slot_mask = (1 << p.batch.page_log2) - 1;
    SegmentIter it(p, span);
    int kt = 0;
    bool ok = true;
    // Pages are looked up 32 at a time, as by the few rows' producer.
    const int block_tiles = 32 * box_rows / kTileKeys;
    int first = 0, boxes = 0, at_box = 0;             // of the tile at hand: first key, boxes, the first one's place among the pages at hand
    int pages = 0, checked = 0;
    auto find_pages = [&](const Segment& g, int j) {  // from tile j on
      const int key = g.key0 + j * kTileKeys + lane * box_rows;
      if (key < g.len) pages = page_of_key(p, g.b, key);
    };
    auto load = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int head) {
      if (leader) mbar_arrive_expect_tx(bar, boxes * box_rows * D * 2);
#pragma unroll 1
      for (int i = 0; i < boxes; ++i) {
        const int id = __shfl_sync(0xffffffffu, checked, at_box + i);
        if (leader) {
#pragma unroll
          for (int c = 0; c < kSlabs; ++c) tma_load_4d(dst + c * L::kSlab + i * box_rows * 128, map, bar, c * 64, first & slot_mask, head, id);
        }
      }
    };
#pragma unroll 1
    for (int items = 0; ok; ++items) {
      const int slot = items % L::kItems;
      const Segment g = it.next();
      if (g.n_tiles > 0) find_pages(g, 0);
      SAGE_PAGED_WARP_WAIT_OR(true, item_empty + slot, ((items / L::kItems) & 1) ^ 1u, 20, { ok = false; break; });
      if (lane == 0) {
        segments[slot] = g;
        mbar_arrive(item_full + slot);
      }
      __syncwarp();
      if (g.n_tiles == 0) break;
      if (items > 0) SAGE_PAGED_WARP_WAIT_OR(true, q_empty, (items - 1) & 1, 22, { ok = false; break; });
      if (leader) {
        const int tiles = n_row_tiles(p, g), half_rows = p.tile_rows / 2;
        mbar_arrive_expect_tx(q_full, tiles * half_rows * D * 2);
#pragma unroll 1
        for (int q = 0; q < tiles; ++q) {
#pragma unroll
          for (int c = 0; c < kSlabs; ++c)
            tma_load_3d(s_q + q * L::kQBytes + c * L::kSlab, &tm_q, q_full, c * 64, g.head0, g.q0 + p.by_group(g.row0 + q * half_rows));
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int j = 0; j < g.n_tiles; ++j, ++kt) {
        const int s = kt % kStages;
        SAGE_PAGED_WARP_WAIT_OR(true, k_empty + s, ((kt / kStages) & 1) ^ 1u, 23, { ok = false; break; });
        const int in_block = j & (block_tiles - 1);
        if (in_block == 0) {
          checked = checked_page(p, pages);
          if (j + block_tiles < g.n_tiles) find_pages(g, j + block_tiles);
        }
        first = g.key0 + j * kTileKeys;
        boxes = (min(max(g.len - first, 0), kTileKeys) + box_rows - 1) / box_rows;
        at_box = in_block * kTileKeys / box_rows;
        load(&tm_k, s_k + s * L::kKVBytes, k_full + s, g.kv_head);
        SAGE_PAGED_WARP_WAIT_OR(true, v_empty + s, ((kt / kStages) & 1) ^ 1u, 21, { ok = false; break; });
        if (!(p.test_drop_load && kt == 0)) load(&tm_v, s_v + s * L::kKVBytes, v_full + s, g.kv_head);   // (failure-detection test)
      }
    }
    __syncwarp();
  } else if (warp == kSoftmaxWarps + 1) {
    if (elect_one()) issue_products(std::integral_constant<int, 0>{});
    __syncwarp();
  } else if (warp == kSoftmaxWarps + 2) {
    if (elect_one()) issue_products(std::integral_constant<int, 1>{});
    __syncwarp();
  } else if (warp == kSoftmaxWarps + 3) {
    // (a warpgroup has four)
  } else {
    // ------------------------------------------------------------------ softmax and output
    const int q = warp >> 2;                          // row tile of this warp
    const int row = (warp & 3) * 32 + lane;           // ... and row of this thread in it
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem_base + lane_base + q * kTileKeys, t_o = tmem_base + lane_base + kColO + q * D;
    int kt = 0, qt = 0, live_items = 0;               // key tiles so far, those of this row tile, items in which it had rows
    bool ok = true;
#pragma unroll 1
    for (int items = 0; ok; ++items) {
      SAGE_PAGED_WARP_WAIT_OR(false, item_full + items % L::kItems, (items / L::kItems) & 1, 34, { ok = false; break; });
      const Segment g = segments[items % L::kItems];
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty + items % L::kItems);
      if (g.n_tiles == 0) break;
      if (q >= n_row_tiles(p, g)) {
        kt += g.n_tiles;
        continue;
      }
      const int half_rows = p.tile_rows / 2;
      int token = 0, head = 0, limit = 0;
      bool live = row_at(p, g.q0, g.n_q, g.head0, g.row0 + q * half_rows, half_rows, row, &token, &head);
      if (live) {
        if (p.shared_pass) {
          int q1;
          const int b = seq_of_token(p, token, &q1);
          live = b < p.batch.B;
          if (live) limit = min(g.len, visible_keys(p, b, q1, token));
        } else {
          limit = p.causal ? max(0, g.len - (g.q0 + g.n_q - 1 - token)) : g.len;
        }
      }
      // Rows without a token hold whatever an earlier kernel left in shared memory, or tokens of another sequence: they have no
      // vote below, or the bits of the others would depend on it.
      const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
      const bool warp_live = live_rows != 0;
      const int warp_limit = __reduce_min_sync(0xffffffffu, live ? limit : 0x7fffffff);
      float m = -INFINITY, l = 0.0f;
      int distrust = 0;                               // > 1: the optimistic pass is skipped
      bool settled = false;                           // every row of the warp that has a token has a maximum
      const f32x2_t scale2 = pack2(p.score_scale, p.score_scale);
#pragma unroll 1
      for (int hh = 0; hh < 2 * g.n_tiles; ++hh) {
        const int h = hh & 1, t = kt + (hh >> 1), tq = qt + (hh >> 1), first = g.key0 + hh * kHalfKeys;
        const uint32_t t_sh = t_s + h * kHalfKeys;
        SAGE_PAGED_WARP_WAIT_OR(false, s_full + 2 * q + h, tq & 1, 31, { ok = false; break; });
        tc_fence_after();
        if (h == 0 && first + kTileKeys > g.len) {
          // The last tile: zeros over what is no value of the sequence, by both row tiles, either of which may be first.  (Behind
          // the wait for S, which says that the stage's load before this one has long been used: a parity cannot tell
          // phases apart that are two turns away.)
          const int stage = t % kStages;
          SAGE_PAGED_WARP_WAIT_OR(false, v_full + stage, (t / kStages) & 1, 30, { ok = false; break; });
          const int keys = max(g.len - first, 0);
#pragma unroll 1
          for (int i = threadIdx.x & 127; i < (kTileKeys - keys) * kSlabs * 8; i += 128) {
            const int r = keys + i / (kSlabs * 8), x = i % (kSlabs * 8);
            *reinterpret_cast<uint4*>(s_v + stage * L::kKVBytes + (x >> 3) * L::kSlab + r * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();                   // the tensor cores read it through the async proxy
        }
        if (warp_live) {
          // Weights of some columns against `base`, packed; returns their sum.
          float high = -INFINITY;
          auto weigh = [&](auto& sr, float base, auto keep, auto by_hand, uint32_t* pk) -> f32x2_t {
            const f32x2_t neg = pack2(kTileBias - base, kTileBias - base);
            f32x2_t acc = pack2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(sr) / 8); ++i) {
              const float2 x = unpack2(ffma2(pack2(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), scale2, neg));
              float2 w;
              if (by_hand(i)) w = exp2_by_polynomial(x.x, x.y, &high);
              else w = make_float2(ex2(x.x), ex2(x.y));
              keep(2 * i, &w.x);
              keep(2 * i + 1, &w.y);
              acc = fadd2(acc, pack2(w.x, w.y));
              pk[i] = from_float2(w.x, w.y, static_cast<const T*>(nullptr));
            }
            return acc;
          };
          const bool masked = first + kHalfKeys > warp_limit;
          const bool attempt = settled && !masked && distrust < 2;
          bool done = false;
          if (attempt) {
            // (P stays in registers until the sum has been looked at: S would be needed again)
            uint32_t sr[2][32], pk[32];
            tmem_ld32(t_sh, sr[0]);
            tmem_ld32(t_sh + 32, sr[1]);
            tc_wait_ld();
            auto by_hand = [](int i) { return i % kHandEvery == kHandEvery - 1; };
            const f32x2_t acc = weigh(sr[0], m, [](int, float*) {}, by_hand, pk);
            const float2 a = unpack2(fadd2(acc, weigh(sr[1], m, [](int, float*) {}, by_hand, pk + 16)));
            const float sum = a.x + a.y;
            done = (__ballot_sync(0xffffffffu, !(sum <= kTileSumMax) || high > 16.0f) & live_rows) == 0;
            if (done) {
              l += sum;
              tmem_st32(t_sh, pk);
            }
            distrust = done ? max(distrust - 1, 0) : min(distrust + 2, 4);
          }
          if (!done) {
            const int col_end = live ? limit - first : kHalfKeys;    // columns below it are visible
            // (16 columns at a time: this path is taken once or twice an item, and its instructions have to be fetched)
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < kHalfKeys; c += 16) {
              uint32_t sr[16];
              tmem_ld16(t_sh + c, sr);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float x = __uint_as_float(sr[i]) * p.score_scale;
                if (c + i < col_end) top = fmaxf(top, x);
              }
            }
            const bool need = top > m + (attempt ? kTileRefusedLazy : kTileLazy) || (m == -INFINITY && top > m);
            const bool moved = (__ballot_sync(0xffffffffu, need) & live_rows) != 0;
            if (!attempt && hh > 0) distrust = moved ? min(distrust + 1, 4) : max(distrust - 1, 0);
            if (moved) {
              if (hh > 0) {
                SAGE_PAGED_WARP_WAIT_OR(false, pv_done + 2 * q + (h ^ 1), (h ? tq : tq - 1) & 1, 32, { ok = false; break; });
                tc_fence_after();
                const float back = need ? ex2(m - top) : 1.0f;
                l *= back;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                  uint32_t orr[16];
                  tmem_ld16(t_o + c, orr);
                  tc_wait_ld();
#pragma unroll
                  for (int i = 0; i < 16; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * back);
                  tmem_st16(t_o + c, orr);
                }
              }
              if (need) m = top;
            }
            settled = (__ballot_sync(0xffffffffu, m == -INFINITY) & live_rows) == 0;
            const float base = m == -INFINITY ? 0.0f : m;            // (a row that has seen nothing yet)
#pragma unroll 1
            for (int c = 0; c < kHalfKeys; c += 16) {                // (P of these columns goes where columns before them were)
              uint32_t sr[16], pk[8];
              tmem_ld16(t_sh + c, sr);
              tc_wait_ld();
              const float2 a = unpack2(weigh(sr, base, [&](int i, float* w) {
                if (c + i >= col_end) *w = 0.0f;
              }, [](int) { return false; }, pk));
              l += a.x + a.y;
              tmem_st8(t_sh + c / 2, pk);
            }
          }
          tc_wait_st();
        }
        tc_fence_before();
        __syncwarp();                                 // (an arrival per warp: 128 of them on one word take turns)
        if (lane == 0) mbar_arrive(p_full + 2 * q + h);
      }
      if (!ok) break;
      SAGE_PAGED_WARP_WAIT_OR(false, o_final + q, live_items & 1, 33, { ok = false; break; });
      tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
      if (__any_sync(0xffffffffu, live && l == 0.0f)) {
        // The sum of 0 * V of a row without keys is no zero where V is infinite.  (Here and not on writing: a choice per value there
        // made chunks of prompts 1.5 % slower.)
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          uint32_t orr[16];
          tmem_ld16(t_o + c, orr);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) orr[i] = l == 0.0f ? 0u : orr[i];
          tmem_st16(t_o + c, orr);
        }
        tc_wait_st();
      }
      if (g.slot == 1 && threadIdx.x == 0) {
        p.headers[blockIdx.x] = PartHeader{g.n_parts, g.q0, g.n_q, g.head0, g.row0, p.tile_rows, {0, 0}};
      }
      const int slot = blockIdx.x * 2 + g.slot, part_row = q * half_rows + row;
      float4* part = reinterpret_cast<float4*>(p.part_o) + static_cast<long long>(slot) * p.tile_rows * (D / 4) + part_row;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t orr[32];
        if (warp_live) {
          tmem_ld32(t_o + 32 * c, orr);
          tc_wait_ld();
        }
        if (c == D / 32 - 1) {                        // O is in registers: the next item may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(o_free + q);
        }
        if (!live) continue;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(orr[i]) * inv;
        if (g.slot >= 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) part[(8 * c + i) * p.tile_rows] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          if (c == 0) p.part_e[slot * p.tile_rows + part_row] = part_lse(m - kTileBias, l);
        } else {
          write_row<T, 32>(p, token, head, D, 32 * c, x, l == 0.0f ? -INFINITY : m - kTileBias + log2f(l), c == 0);
        }
      }
      kt += g.n_tiles;
      qt += g.n_tiles;
      ++live_items;
    }
    if (ok) zero_rest<T>(p, D, threadIdx.x, 256);
  }
#undef SAGE_PAGED_WAIT_OR
#undef SAGE_PAGED_WARP_WAIT_OR

  // ---------------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (*abort_flag && !dead_on_arrival) {
    // A wait gave up: copies and products that are still in flight land before shared memory and TMEM are handed back.
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    if (threadIdx.x == 0) p.status.report(*fail_code ? *fail_code : kStatusWait);
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTileTmemCols);
  }
}

}  // namespace paged
}  // namespace sage
