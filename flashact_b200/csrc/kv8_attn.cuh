// Arguments that the two attention kernels over the 8-bit cache and their merge share.
#pragma once
#include "fa_kv8.cuh"

namespace fa {
namespace kv8 {

struct AttnArgs {
  const float *ks, *vs;
  const void* q;
  void* out;
  long long qb, qt, qh, ob, ot, oh;  // element strides: batch, token, head
  Mask mask;
  int layers, layer, heads, group, dim, blocks, block_log2, half;  // half: fp16 queries (else bf16)
  int q_wide, o_wide;  // rows of queries are 16-byte, of the output 8-byte aligned
  float scale_log2;  // score scale * log2(e)
  uint32_t group_mul;  // ceil(2^32 / group): token of a row without a division
  // Splits of the key axis, joined by the cluster that they are (at most 8), or by the merge kernel. With a cluster
  // each takes an equal share of the observation's own tiles, else tiles [split * split_chunks, + split_chunks).
  int nsplit, cluster, split_chunks;
  int device;
  int fault_split, spin_limit;  // test hook: the split whose first scores are never announced (-1: none); polls of a wait
  int rows;                  // rows of a tile
  int tiles;                 // row tiles of a (observation, key head)
  float* part;               // [slot][rows of a tile][D] unnormalised sums, slot = ((b, h), tile, split)
  float2* ml;                // [slot][rows of a tile]: max (log2 units) and sum
};

// row / group; rows are below 2^24 + 128, so the product is at most one too high.
__device__ __forceinline__ int token_of(const AttnArgs& a, int row) {
  if (a.group == 1) return row;
  const int t = (int)__umulhi((uint32_t)row, a.group_mul);
  return t - (t * a.group > row);
}
// First element of a row (token, head) of the queries or of the output.
__device__ __forceinline__ long long row_at(const AttnArgs& a, int b, int h, int row, long long sb, long long st, long long sh) {
  const int t = token_of(a, row);
  return b * sb + t * st + (h * a.group + row - t * a.group) * sh;
}

// A row of queries is multiplied by 2^(7 - x), x the exponent of its largest magnitude, which brings that to [128, 256); x = 0
// for a row of zeros or of numbers below 2^-100. `back` undoes it; it is NaN for a row with an infinity, whose scores and
// outputs then are NaN.
__device__ __forceinline__ float row_factor(float amax, float& back) {
  int x = (__float_as_int(amax) >> 23) - 127;
  const bool inf = x > 127;
  x = x > -100 && !inf ? x : 0;
  back = inf ? __int_as_float(0x7fffffff) : __int_as_float((x - 7 + 127) << 23);
  return __int_as_float((7 - x + 127) << 23);
}
__device__ __forceinline__ void store16(void* p, long long i, float x, int half) {
  if (half) reinterpret_cast<__half*>(p)[i] = __float2half(x);
  else reinterpret_cast<bf16*>(p)[i] = __float2bfloat16(x);
}

}  // namespace kv8
}  // namespace fa

// The kernels: up to 16 query rows of a key head (kv8_attn_few.cu), and 128 at a time (kv8_attn_rows.cu).
fa_status kv8_launch_few(const fa::kv8::AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s);
fa_status kv8_launch_rows(const fa::kv8::AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s);
// Clusters of n blocks of the kernel for such a call (n = 1: blocks) that the current device has room for at once; 0 if that is not known.
int kv8_resident_few(int rows, bool half, int dim, int device, int n);
int kv8_resident_rows(bool half, int dim, int device, int n);
