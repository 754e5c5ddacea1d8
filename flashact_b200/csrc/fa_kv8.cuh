// The 8-bit KV cache's pieces that its kernels share: E4M3 and f16 conversions, the m16n8k16 matrix
// instruction, and the host-side checks of an fa_kv8 descriptor.
#pragma once
#include <cuda_fp16.h>

#include <initializer_list>
#include <utility>

#include "fa_ptx.cuh"
#include "host_base.cuh"

namespace fa {
namespace kv8 {

constexpr float kE4M3Max = 448.0f;
constexpr int kMinExp = -96;  // smallest block scale 2^-96: its reciprocal and 448 / 2^-96 stay finite

// Codes 0, 1 (lo) and 2, 3 (hi) of a word -> two f16 values each, exact (every E4M3 value is an f16 value).
__device__ __forceinline__ uint32_t e4m3_lo_f16x2(uint32_t four) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(four));
  return r;
}

// D(16x8, f32) += A(16x16, f16) B(16x8, f16).
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cp.async with zero fill: copies `bytes` (0 or the full size) and zeroes the rest.
__device__ __forceinline__ void cp_async16_zfill(void* smem_dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem_dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// Keys of a query: j < limit, limit = min(len, max(position + 1, prefix)); full masks see all len keys.
struct Mask {
  const int* lens;
  const int* q_lens;
  const int* prefix;
  int causal, tokens, capacity;
  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), capacity); }
  __device__ __forceinline__ int q_len(int b) const { return q_lens ? min(max(q_lens[b], 0), tokens) : tokens; }
  // -1 where the token is padding (its output is not written)
  __device__ __forceinline__ int limit(int n, int nq, int pre, int t) const {
    if (t >= nq) return -1;
    if (!causal) return n;
    return min(n, max(max(n - nq + t + 1, 0), pre));
  }
};

}  // namespace kv8
}  // namespace fa

// A device pointer of the current device (or managed memory).
static inline bool on_current_device(const void* p, int dev) {
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev);
}
static inline fa_status check_pointers(std::initializer_list<std::pair<const char*, const void*>> ps) {
  int dev = 0;
  FA_CUDA(nullptr, cudaGetDevice(&dev));
  for (const auto& p : ps)
    if (!p.second || !on_current_device(p.second, dev))
      return fail(nullptr, FA_ERR_INVALID, "'%s' must be memory of the current device", p.first);
  return FA_OK;
}


static inline fa_status kv8_check(const fa_kv8* c) {
  if (!c) return fail(nullptr, FA_ERR_INVALID, "null cache");
  if (c->batch < 1 || c->batch > 65535 || c->layers < 1 || c->heads < 1 || c->heads > 65535)
    return fail(nullptr, FA_ERR_INVALID, "cache of batch=%d layers=%d heads=%d", c->batch, c->layers, c->heads);
  if ((long long)c->batch * c->layers > 0x7fffffffLL / c->heads)
    return fail(nullptr, FA_ERR_INVALID, "batch x layers x heads is over 2^31 - 1");
  if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 256)
    return fail(nullptr, FA_ERR_UNSUPPORTED, "head_dim=%d is not 64, 96, 128 or 256", c->head_dim);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(nullptr, FA_ERR_UNSUPPORTED, "block=%d is not 16, 32, 64 or 128", c->block);
  if (c->capacity < c->block || c->capacity % c->block || c->capacity > (1 << 30))
    return fail(nullptr, FA_ERR_INVALID, "capacity=%d is not a multiple of block=%d up to 2^30", c->capacity, c->block);
  if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16 ||
      reinterpret_cast<uintptr_t>(c->k_scale) % 4 || reinterpret_cast<uintptr_t>(c->v_scale) % 4)
    return fail(nullptr, FA_ERR_INVALID, "the codes must be 16-byte aligned, the scales 4-byte aligned");
  return FA_OK;
}
static inline fa_status kv8_check_pointers(const fa_kv8* c) {
  return check_pointers({{"cache k", c->k}, {"cache v", c->v}, {"cache k_scale", c->k_scale}, {"cache v_scale", c->v_scale}});
}
