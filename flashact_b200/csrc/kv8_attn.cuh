// Arguments that the two attention kernels over the 8-bit cache and their merge share.
#pragma once
#include "fa_kv8.cuh"

namespace fa {
namespace kv8 {

struct AttnArgs {
  const unsigned char *k, *v;
  const float *ks, *vs;
  const void* q;
  void* out;
  long long qb, qt, qh, ob, ot, oh;  // element strides: batch, token, head
  Mask mask;
  int layers, layer, heads, group, cap, block, half;  // half: fp16 queries (else bf16)
  float scale_log2;  // score scale * log2(e)
  int nsplit, split_chunks;  // splits of the key axis; chunks of one split
  int tiles;                 // row tiles of a (observation, key head)
  float* part;               // [slot][rows of a tile][D] unnormalised sums, slot = ((b, h), tile, split)
  float2* ml;                // [slot][rows of a tile]: max (log2 units) and sum
};

// A power of two near |x|'s largest value, its exponent cleared of extremes: x * 2^-e is in [1, 2).
__device__ __forceinline__ float row_pow2(float amax) {
  const int x = (__float_as_int(amax) >> 23) - 127;
  return (amax > 0.f && x < 127 && x > -100) ? __int_as_float((x + 127) << 23) : 1.0f;
}
__device__ __forceinline__ float load16(const void* p, long long i, int half) {
  return half ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const bf16*>(p)[i]);
}
// Two consecutive 16-bit outputs: one store where the row is 4-byte aligned.
__device__ __forceinline__ void store16x2(void* p, long long i, float x, float y, int half) {
  const uint32_t hv = pack_f16x2(x, y);
  const __nv_bfloat162 bv = __floats2bfloat162_rn(x, y);
  const uint32_t v = half ? hv : *reinterpret_cast<const uint32_t*>(&bv);
  uint16_t* q = reinterpret_cast<uint16_t*>(p) + i;
  if ((reinterpret_cast<uintptr_t>(q) & 3) == 0) {
    *reinterpret_cast<uint32_t*>(q) = v;
  } else {
    q[0] = (uint16_t)v;
    q[1] = (uint16_t)(v >> 16);
  }
}

}  // namespace kv8
}  // namespace fa

// Launchers (kv8_attn_few.cu). `dim` is the head dimension.
fa_status kv8_launch_few(const fa::kv8::AttnArgs& a, int dim, int batch, cudaStream_t s);
