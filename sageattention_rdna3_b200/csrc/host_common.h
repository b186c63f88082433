// Host code that the translation units of libsage_b200.so share: the error text, argument checks, TMA tensor maps and
// launches.  Not part of the public C ABI.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "../../include/sage_b200.h"
#include "ptx_sm100.cuh"

namespace sage_host {

inline thread_local char g_err[512] = "";
inline std::atomic<long long> g_wait_limit_cycles{sage::kWaitLimitCycles};
inline std::atomic<int> g_test_drop_v_load{0};
inline std::atomic<int*> g_status_host[64];      // per device: mapped pinned host word for failure codes (sage_set_status_mirror)

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

#define SAGE_REQUIRE(cond, ...) \
  do {                          \
    if (!(cond)) return fail(SAGE_ERR_INVALID, __VA_ARGS__); \
  } while (0)

// (The runtime keeps the error for the thread's next cudaGetLastError as well; it is taken from there, or the
// caller's next launch of something else would report it a second time.)
#define SAGE_CUDA(expr)                                                           \
  do {                                                                            \
    cudaError_t e_ = (expr);                                                      \
    if (e_ != cudaSuccess) {                                                      \
      cudaGetLastError();                                                         \
      return fail(SAGE_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_));        \
    }                                                                             \
  } while (0)

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool strides_ok(const sage_strided_t* t) {
  return t->stride_b % 8 == 0 && t->stride_h % 8 == 0 && t->stride_s % 8 == 0;
}
// cuTensorMapEncodeTiled is taken from the driver at run time, so the library links against the
// CUDA runtime only.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<EncodeTiledFn>(sym);
    }
  });
  return fn;
}

inline int encode_map(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* base, const cuuint64_t* dims,
               const cuuint64_t* strides_bytes, const cuuint32_t* box, CUtensorMapSwizzle swz, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(SAGE_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(map, dt, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides_bytes, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SAGE_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, (int)r);
  return SAGE_OK;
}

// Tiled map of a 16-bit [B,H,S,D] tensor in the caller's layout: dimensions (D, S, H, B) with the
// caller's element strides, boxes of `box_rows` rows x 64 columns, 128-byte swizzle.  A dimension of
// extent 1 may carry any stride in the caller's tensor; it gets the span of the others so that the
// map stays well formed.
inline int encode_strided_16bit(CUtensorMap* map, CUtensorMapDataType dt, const void* base, int D, long long S, long long H,
                         long long B, long long stride_s, long long stride_h, long long stride_b, int box_rows,
                         const char* what) {
  cuuint64_t ss = (cuuint64_t)stride_s * 2, sh = (cuuint64_t)stride_h * 2, sb = (cuuint64_t)stride_b * 2;
  cuuint64_t span = (cuuint64_t)D * 2;
  if (S > 1 && ss * S > span) span = ss * S;
  if (H > 1 && sh * H > span) span = sh * H;
  if (B > 1 && sb * B > span) span = sb * B;
  span = (span + 15) & ~(cuuint64_t)15;
  if (S == 1) ss = span;
  if (H == 1) sh = span;
  if (B == 1) sb = span;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[3] = {ss, sh, sb};
  cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  return encode_map(map, dt, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

// Launch with programmatic serialisation: the set-up of the kernel and its launch latency run under the end
// of the kernel ahead of it in the stream.  Every kernel launched through here calls grid_dependency_wait() before
// it touches global memory or takes TMEM (sage_fold_partial_kernel is an ordinary launch).  A call is one to
// five kernels (K mean, preparation, attention, merge, log-sum-exp), most of them short, and conversions around
// them for fp32 tensors.  Calls back to back, before and after: 20 heads of 1024 tokens, D=64 19.4 -> 17.2 us,
// 10 heads of 4096 tokens 85.4 -> 82, 32 heads of 4096 tokens causal, D=128 159 -> 154; B=2 H=32 S=8192 causal is
// level.
template <typename... Params, typename... Args>
int launch(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  SAGE_CUDA(cudaLaunchKernelEx(&cfg, kern, Params(args)...));
  return SAGE_OK;
}

inline int sm_count(int* out) {
  static std::atomic<int> cached[64];
  int dev = 0;
  SAGE_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64) {
    const int have = cached[dev].load(std::memory_order_relaxed);
    if (have > 0) {
      *out = have;
      return SAGE_OK;
    }
  }
  int sms = 0;
  SAGE_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  if (dev >= 0 && dev < 64) cached[dev].store(sms, std::memory_order_relaxed);
  *out = sms;
  return SAGE_OK;
}

// (Setting the attribute twice from two host threads that race on the first call is harmless.)
template <typename Kernel>
int configure_smem(Kernel kern, int smem_bytes, std::atomic<bool>* configured) {
  int dev = 0;
  SAGE_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    SAGE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  return SAGE_OK;
}

}  // namespace sage_host
