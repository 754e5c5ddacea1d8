// What the two tensor-core attention kernels over the 8-bit cache share: tile loads, the 8-bit matrix instruction, the
// splitting of queries and probabilities into 8-bit parts.
#pragma once
#include <atomic>

#include "kv8_attn.cuh"

namespace fa {
namespace kv8 {

constexpr int TILE = 128;         // keys of a tile
constexpr int align_up(int x, int a) { return (x + a - 1) / a * a; }

__device__ __forceinline__ uint32_t swz(int row, int byte) {
  return (uint32_t)(row * 128 + ((((byte >> 4) ^ row) & 7) << 4) + (byte & 15));
}
__device__ __forceinline__ void tma_load_3d_plain(void* dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Low word of sdesc_sw128's descriptor; the upper one is the same for all. Steps inside an operand are added to the low word
// (in units of 16 bytes): the issuing warp has 64 cycles for a product at most, and building each descriptor from its
// address took about 130.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(const void* p) { return ((smem_u32(p) >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// The same with A from tensor memory: row r of A in lane r, four of its elements to a column, eight columns from tmem_a.
__device__ __forceinline__ void mma_f8_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], db, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi)
      : "memory");
}
// kind::f8f6f4, fp32 sums, M = 128, A and B E4M3 or E5M2, both K-major.
__host__ __device__ constexpr uint32_t idesc_f8(int N, bool a_e5m2, bool b_e5m2) {
  return (1u << 4) | ((a_e5m2 ? 1u : 0u) << 7) | ((b_e5m2 ? 1u : 0u) << 10) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t f32x2_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// E5M2 is f16's upper byte: rounding an f16 there (half up in magnitude; |p| is below 57344, so that no carry makes an infinity) leaves
// three significant bits, and what it leaves over, of either sign, is again an f16 and at most 2^-3 of the leading power of two. Three such parts
// are 3 + 4 + 4 bits: all eleven of an f16 (cut instead of rounded they would hold nine).
__device__ __forceinline__ uint32_t round_part(uint32_t p) { return p + 0x00800080u; }
__device__ __forceinline__ uint32_t rest1(uint32_t p, uint32_t rounded) {
  const uint32_t v = rounded & 0xff00ff00u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&p), *reinterpret_cast<const __half2*>(&v));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t rest8(uint32_t p, uint32_t rounded) {  // eight times that: at most 2^15.25 where p was
  const uint32_t d = rest1(p, rounded);
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&d), __float2half2_rn(8.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// What the rounding of x, y to the f16 pair p left over, times `up`, in E5M2 (the lower byte is x's).
__device__ __forceinline__ uint32_t f16_lost(float x, float y, uint32_t p, float up) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&p));
  uint16_t r;
  asm("{\n\t.reg .b64 v, n, m;\n\t.reg .f32 a, b;\n\tmov.b64 v, {%1, %2};\n\tmov.b64 n, {%3, %4};\n\t"
      "mov.b64 m, {%5, %5};\n\tfma.rn.f32x2 v, n, m, v;\n\tmov.b64 {a, b}, v;\n\t"
      "cvt.rn.satfinite.e5m2x2.f32 %0, b, a;\n\t}" : "=h"(r) : "f"(x * up), "f"(y * up), "f"(h.x), "f"(h.y), "f"(-up));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_e4m3x2(uint32_t v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(v));
  return r;
}
// A query's four scaled elements in E4M3 parts, each what the ones before left over, times `up`.
template <int PARTS, class Store>
__device__ __forceinline__ void split_query(float (&y)[4], float up, Store store) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    const uint32_t e0 = f32x2_e4m3x2(y[0], y[1]), e1 = f32x2_e4m3x2(y[2], y[3]);
    store(p, e0 | (e1 << 16));
    const uint32_t f0 = e4m3_lo_f16x2(e0), f1 = e4m3_lo_f16x2(e1);
    const float2 g0 = __half22float2(*reinterpret_cast<const __half2*>(&f0));
    const float2 g1 = __half22float2(*reinterpret_cast<const __half2*>(&f1));
    y[0] = (y[0] - g0.x) * up, y[1] = (y[1] - g0.y) * up;
    y[2] = (y[2] - g1.x) * up, y[3] = (y[3] - g1.y) * up;
  }
}
// Clears a V tile's codes (rows of d, 128-byte swizzle) from key `left` of the tile on: their P is 0, but 0 times a NaN
// code would not be.
__device__ __forceinline__ void clear_behind(unsigned char* tile, int rows, int left, int thread, int threads) {
  for (int d = thread; d < rows; d += threads)
    for (int c = left >> 4; c < 8; ++c) {
      uint4* q = reinterpret_cast<uint4*>(tile + swz(d, c * 16));
      uint4 v = make_uint4(0, 0, 0, 0);
      const int keep = left - c * 16;  // bytes of this piece
      if (keep > 0) {
        v = *q;
        uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = keep - 4 * j;
          x[j] = k >= 4 ? x[j] : k <= 0 ? 0u : x[j] & ((1u << (8 * k)) - 1u);
        }
      }
      *q = v;
    }
}
// ---- the splits of a tile as one cluster
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 peer_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 peer_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
// Four consecutive 16-bit outputs of a row; `wide`: 8-byte aligned.
template <bool HALF>
__device__ __forceinline__ void store16x4(uint16_t* p, const float (&v)[4], bool wide) {
  uint2 u;
  if constexpr (HALF) {
    u = make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    u = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  if (wide) {
    *reinterpret_cast<uint2*>(p) = u;
  } else {
    p[0] = (uint16_t)u.x, p[1] = (uint16_t)(u.x >> 16);
    p[2] = (uint16_t)u.y, p[3] = (uint16_t)(u.y >> 16);
  }
}
// The end of a tile of rows: sums `o` [rows][pitch] relative to their maxima, and (maximum, sum) `ml`, in shared memory.
// More than eight splits leave both for the merge kernel. Otherwise the splits, a cluster (or the only CTA), are joined in
// split order, its CTAs sharing the output; a warp takes 128 dims of GROUP rows at a time. All threads of all the CTAs come here.
// With up to 16 rows each row has a warp of its own, and what counts is the chain (0.3 us less than the other form takes for one
// row of 8 us); with 128, four rows at a time keep enough loads on their way (13 us of a lone CTA's 36 with one, 5 with four).
template <bool HALF, int MT, int GROUP>
__device__ __forceinline__ void finish_rows(const AttnArgs& a, const float* o, int pitch, const float* ml, int ml_pitch, int rank,
                                            int b, int h, int row0, int nrows, int n, int nq, int pre, size_t first_part) {
  if (a.nsplit > 1 && !a.cluster) {
    __syncthreads();
    for (int u = threadIdx.x >> 5; u < nrows * MT; u += blockDim.x >> 5) {
      const int r = u / MT, d = (u % MT) * 128 + (threadIdx.x & 31) * 4;
      if (d < a.dim)
        *reinterpret_cast<float4*>(a.part + (first_part + r) * a.dim + d) = *reinterpret_cast<const float4*>(o + r * pitch + d);
      if (d == 0) a.ml[first_part + r] = *reinterpret_cast<const float2*>(ml + r * ml_pitch);
    }
    return;
  }
  cluster_sync();
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, k8 = lane & 7;
  const int groups = (nrows + GROUP - 1) / GROUP;
  for (int u = rank * warps + (threadIdx.x >> 5); u < groups * MT; u += a.nsplit * warps) {
    const int r0 = u / MT * GROUP, d = (u % MT) * 128 + lane * 4;
    if constexpr (GROUP == 1) {  // lane k weighs split k
      float2 x = make_float2(-INFINITY, 0.f);
      if (lane < a.nsplit) x = peer_f32x2(peer(ml + r0 * ml_pitch, lane));
      const bool none = x.x == -INFINITY && x.y == 0.f;
      const float top = warp_max(x.x), f = none ? 0.f : exp2_approx(x.x - (top == -INFINITY ? 0.f : top));
      const uint32_t live = __ballot_sync(0xffffffffu, !none);
      float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k), lk = __shfl_sync(0xffffffffu, x.y, k);
        if (live >> k & 1) {
          sum += fk * lk;
          const float4 p = peer_f32x4(peer(o + r0 * pitch + d, k));
          v[0] += fk * p.x, v[1] += fk * p.y, v[2] += fk * p.z, v[3] += fk * p.w;
        }
      }
      const float norm = a.mask.limit(n, nq, pre, token_of(a, row0 + r0)) > 0 ? 1.0f / sum : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = norm == 0.f && sum == sum ? 0.f : v[i] * norm;
      if (d < a.dim)
        store16x4<HALF>(reinterpret_cast<uint16_t*>(a.out) + row_at(a, b, h, row0 + r0, a.ob, a.ot, a.oh) + d, v, a.o_wide);
      continue;
    }
    // lane 8 j + k weighs split k in row r0 + j: none of it where the split has left no key to the row; a NaN in its sum stays
    const int r = min(r0 + (lane >> 3), nrows - 1), row = row0 + r;
    float2 x = make_float2(-INFINITY, 0.f);
    if (k8 < a.nsplit) x = peer_f32x2(peer(ml + r * ml_pitch, k8));
    constexpr int STEP = 8 / GROUP;
    float4 p[STEP][GROUP];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int k = 0; k < STEP; ++k)
#pragma unroll
        for (int j = 0; j < GROUP; ++j)
          if (k0 + k < a.nsplit) p[k][j] = peer_f32x4(peer(o + min(r0 + j, nrows - 1) * pitch + d, k0 + k));
    };
    fetch(0);
    const bool none = x.x == -INFINITY && x.y == 0.f;
    float top = x.x;
#pragma unroll
    for (int i = 4; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    float f = none ? 0.f : exp2_approx(x.x - (top == -INFINITY ? 0.f : top)), sum = f * x.y;
#pragma unroll
    for (int i = 4; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    f = none ? 0.f : f * (a.mask.limit(n, nq, pre, token_of(a, row)) > 0 ? 1.0f / sum : 0.f);
    const long long at = row_at(a, b, h, row, a.ob, a.ot, a.oh);
    float v[GROUP][4] = {};
#pragma unroll 1
    for (int k0 = 0; k0 < a.nsplit; k0 += STEP) {
      if (k0 > 0) fetch(k0);
#pragma unroll
      for (int k = 0; k < STEP; ++k)
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
          const float fk = __shfl_sync(0xffffffffu, f, 8 * j + k0 + k);
          if (k0 + k < a.nsplit) {  // a split without a key for the row may hold anything (fk may be a NaN)
            const float4 y = fk != 0.f ? p[k][j] : make_float4(0.f, 0.f, 0.f, 0.f);
            v[j][0] += fk * y.x, v[j][1] += fk * y.y, v[j][2] += fk * y.z, v[j][3] += fk * y.w;
          }
        }
    }
#pragma unroll
    for (int j = 0; j < GROUP; ++j) {
      const long long to = __shfl_sync(0xffffffffu, at, 8 * j);
      if (d < a.dim && r0 + j < nrows) store16x4<HALF>(reinterpret_cast<uint16_t*>(a.out) + to + d, v[j], a.o_wide);
    }
  }
  cluster_sync();  // no CTA leaves while another may read its memory
}

// The merge may be set up from here on; it waits for this grid's end before it reads anything.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Loads that are issued where they stand: the first ones of a block go out together, before lengths are known.
__device__ __forceinline__ uint2 ldg_now8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ldg_now2(const void* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float ldg_now(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
// Four consecutive 16-bit elements of a row that may be 2-byte aligned only.
__device__ __forceinline__ uint2 ldg_row4(const uint16_t* p) {
  if ((reinterpret_cast<uintptr_t>(p) & 7) == 0) return ldg_now8(p);
  return make_uint2(ldg_now2(p) | (ldg_now2(p + 1) << 16), ldg_now2(p + 2) | (ldg_now2(p + 3) << 16));
}
template <bool HALF>
__device__ __forceinline__ float2 pair_f32(uint32_t v) {
  if constexpr (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Order of n tiles of keys in the ring, the scores' products LEAD tiles ahead of P V: LEAD 1: K0, K1, V0, K2, V1, .. V(n-1);
// LEAD 2: K0, K1, K2, V0, K3, V1, .. V(n-2), V(n-1).
template <int LEAD>
__device__ __forceinline__ int pos_k(int i) {
  return i <= LEAD ? i : 2 * i - LEAD;
}
template <int LEAD>
__device__ __forceinline__ int pos_v(int i, int n) {
  return i + LEAD >= n ? n + i : 2 * i + LEAD + 1;
}

enum { ERR_FULL = 1, ERR_EMPTY, ERR_S, ERR_SFREE, ERR_P, ERR_PV, ERR_SEEN };

// A bounded wait, as mbar_wait, whose limit stands behind the block's error word (err[1]).
static __device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t phase, volatile int* err, int code) {
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if ((i & 255u) == 0) {
      if (*err) return false;
      if (i >= (uint32_t)err[1]) break;
      __nanosleep(64);
    }
  }
  atomicCAS((int*)err, 0, code);
  return false;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t phase, volatile int* err, int code) {
  return mbar_test_wait(bar, phase) || wait_slow(bar, phase, err, code);
}

// The end of a block in which a wait ran out, after all its warps have met: what is in flight ends first (again with a limit), the copies
// issued and the products, which the issuing warps put on `drained`; then all its rows are NaN, sums and (maximum, sum). A sum that is NaN
// goes through each join and the merge, where a sum of 0 would be a split without a key. All threads come here.
template <int SLOTS>
static __device__ __noinline__ void give_up(uint64_t* full, int issued, uint64_t* drained, bool issuer, float* o, int pitch, int width,
                                        float* ml, int ml_pitch, int rows) {
  if (issuer) tc_commit_elect(drained);
  if (threadIdx.x == 0) {
    for (int pos = max(0, issued - SLOTS); pos < issued; ++pos)
      for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(full + pos % SLOTS, (pos / SLOTS) & 1); ++i) {}
    for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait(drained, 0); ++i) {}
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * width; i += blockDim.x) o[i / width * pitch + i % width] = __int_as_float(0x7fffffff);
  for (int i = threadIdx.x; i < rows; i += blockDim.x) ml[i * ml_pitch] = -INFINITY, ml[i * ml_pitch + 1] = __int_as_float(0x7fffffff);
  __syncthreads();
}

// The producer warp's lane: K and V tiles of one head into the ring, in the order of pos_k and pos_v, places from .. to. Returns where it ended.
template <int LEAD, int SLOTS, int MT>
__device__ __forceinline__ int produce(unsigned char* ring, uint64_t* full, uint64_t* empty, const CUtensorMap* kmap,
                                        const CUtensorMap* vmap, int t0, int nt, int head, volatile int* err, int from,
                                        int to) {
  constexpr int SLOT = MT * 16384;
  for (int pos = from; pos < to; ++pos) {
    const int slot = pos % SLOTS, use = pos / SLOTS;
    if (use > 0 && !wait_for(empty + slot, (use - 1) & 1, err, ERR_EMPTY)) return pos;
    const bool behind = pos >= 2 * nt - min(LEAD, nt), is_v = behind || (pos > LEAD && (pos - LEAD) % 2 != 0);
    const int i = behind ? pos - nt : is_v ? (pos - LEAD - 1) / 2 : pos <= LEAD ? pos : (pos + LEAD) / 2;
    unsigned char* dst = ring + slot * SLOT;
    mbar_expect_tx(full + slot, SLOT);
    if (is_v) {
      tma_load_3d_plain(dst, vmap, full + slot, (t0 + i) * TILE, 0, head);
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m) tma_load_3d_plain(dst + m * 16384, kmap, full + slot, m * 128, (t0 + i) * TILE, head);
    }
  }
  return to;
}

}  // namespace kv8
}  // namespace fa

// Clusters of n blocks (n = 1: blocks) of `threads` threads and `smem` bytes that `device`, the current one, has room for at once; asked
// once a kernel, size and device. The parts of the chip that a cluster may not span leave some of it idle, differently for each size. Asked for a
// kernel without tensor memory: the runtime counts one that allocates it as one block to an SM, while as many run as shared memory has room for
// (Cfg sees to it that registers and tensor memory do too). 0: not known.
static __global__ void room_kernel() {}
template <auto kernel>
static int kv8_resident(int device, int n, int threads, int smem) {
  static std::atomic<int> known[64][9];
  std::atomic<int>& at = known[device & 63][n];
  int got = at.load(std::memory_order_relaxed), sms = 0;
  if (got > 0) return got;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaFuncSetAttribute(room_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess)
    e = n > 1 ? cudaOccupancyMaxActiveClusters(&got, room_kernel, &cfg) : cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, room_kernel, threads, smem);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (n == 1) got *= sms;
  at.store(got, std::memory_order_relaxed);
  return got;
}

template <auto kernel>
static fa_status kv8_launch(const fa::kv8::AttnArgs& a, int batch, int threads, int smem, const CUtensorMap& km,
                            const CUtensorMap& vm, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.nsplit * a.tiles, a.heads, batch);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.nsplit;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cluster ? 1 : 0;
  // The shared memory limit is set on a device's first launch of a kernel, and again where a launch fails (a device that was reset).
  static std::atomic<unsigned long long> set{0};
  const unsigned long long bit = 1ull << (a.device & 63);
  if (set.load(std::memory_order_relaxed) & bit) {
    if (cudaLaunchKernelEx(&cfg, kernel, a, km, vm) == cudaSuccess) return FA_OK;
    cudaGetLastError();
  }
  FA_CUDA(nullptr, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  FA_CUDA(nullptr, cudaLaunchKernelEx(&cfg, kernel, a, km, vm));
  set.fetch_or(bit, std::memory_order_relaxed);
  return FA_OK;
}
