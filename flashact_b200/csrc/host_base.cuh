// Host-side pieces that every part behind the C ABI uses: error reporting without a handle, types, the TMA encoder.
#pragma once
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstddef>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>

#include "../../include/flashact.h"

using bf16 = __nv_bfloat16;

extern thread_local std::string g_create_err;

static inline fa_status fail(std::nullptr_t, fa_status st, const char* fmt, ...) {  // read with fa_last_error(NULL)
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_create_err = buf;
  return st;
}
#define FA_CUDA(h, call)                                                                        \
  do {                                                                                          \
    cudaError_t e_ = (call);                                                                    \
    if (e_ != cudaSuccess) return fail(h, FA_ERR_CUDA, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), \
                                       __FILE__, __LINE__);                                     \
  } while (0)

static inline size_t dtype_size(fa_dtype t) { return t == FA_DT_F32 ? 4 : 2; }

__device__ __forceinline__ float e4m3_value(unsigned char c) {
  __nv_fp8_e4m3 f;
  f.__x = c;
  return (float)f;
}

static inline PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};  // calls may come from several threads
  PFN_cuTensorMapEncodeTiled_v12000 fn = known.load(std::memory_order_relaxed);
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      known.store(fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr), std::memory_order_relaxed);
  }
  return fn;
}
