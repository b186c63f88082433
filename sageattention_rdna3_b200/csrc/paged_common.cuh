// What the kernels over a paged cache share: the batch as the caller describes it, page look-up with its checks, and
// conversions between 16-bit types and fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cfloat>
#include <cstdint>

#include "../../include/sage_paged_b200.h"
#include "ptx_sm100.cuh"

namespace sage {
namespace paged {

constexpr int kStatusBadPage = SAGE_STATUS_BAD_PAGE;
constexpr int kStatusBadLength = SAGE_STATUS_BAD_LENGTH;
constexpr int kStatusMisaligned = 1;                  // as attn_kernel.cuh
constexpr int kStatusWait = 2 + 16 * 20;              // ... and its numbering of waits: 20, a load of keys and values

// A bounded wait by a whole warp: its lanes go on or give up together.
template <bool kHinted>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, long long limit_cycles) {
  return __all_sync(0xffffffffu, mbar_wait<kHinted>(bar, parity, abort_flag, limit_cycles));
}

// As tma_load_4d (ptx_sm100.cuh), five coordinates.
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* tmap, uint64_t* bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

struct Status {
  int* word;                    // optional device word, stays 0 on success
  int* host;                    // optional word in mapped pinned host memory that receives what the device word holds
  __device__ __forceinline__ void report(int code) const { report_status(word, host, code); }
};

struct Batch {
  const int32_t* table;
  long long table_stride;
  int table_width;
  const int32_t* kv_lens;
  const int32_t* cu_q;          // null: one token per sequence
  int B, T;
  int page_log2, num_pages;

  // New tokens [q0, q1) of sequence b; whatever cu_q holds, 0 <= q0 <= q1 <= T.
  __device__ __forceinline__ void tokens(int b, int* q0, int* q1) const {
    if (cu_q == nullptr) {
      *q0 = b;
      *q1 = b + 1;
    } else {
      const int lo = min(max(cu_q[b], 0), T);
      *q0 = lo;
      *q1 = min(max(cu_q[b + 1], lo), T);
    }
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-bit types <-> fp32
__device__ __forceinline__ float2 to_float2(uint32_t w, const __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 to_float2(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t from_float2(float a, float b, const __half*) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));   // first source -> upper half
  return r;
}
__device__ __forceinline__ uint32_t from_float2(float a, float b, const __nv_bfloat16*) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

}  // namespace paged
}  // namespace sage
