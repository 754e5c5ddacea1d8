// fa_nvfp4_linear: y = x W^T * tensor_scale (+ bias) for up to 16 rows of x, W read as NVFP4 (E2M1 codes
// and one E4M3 scale for 16 of them), as fa_quantize_nvfp4 lays it out. Bound by the weight's bytes (9/16
// of one each).
//
// A weight's code times its block scale has at most six significant bits, so it is exact in bf16 and
// in f16 alike and the product runs on the 16-bit matrix instruction with x as it is, fp32 sums. A code's
// three magnitude bits are put where the 16-bit type has its lowest exponent bits and first mantissa
// bit: that is the code's value times a power of two, the subnormal code included, and the power is
// made good in the block scale and at the end.
//
// A warp takes 16 * RT rows of W, and every eighth chunk of the CTA's whole K; the eight warps' sums meet in
// shared memory in warp order. The order of k inside the matrix instruction is free as long as both
// operands share it: a lane owns PB bytes of codes (one or two scale blocks) of each of its rows, read
// with one load a turn ahead, and x's pairs follow the order in which the codes come out of a word.
//
// Measured in a graph, inputs beyond L2: 16 rows by 28672 x 8192 in fp16 55 us (2.4 TB/s), 8 by 32768 x 2048 in bf16 17.0 us (2.3 TB/s),
// one by 2560 x 1024 2.3 us. The memory's time for the first two is 20 and 6 us. Two CTAs share an SM at 128 registers (13 to 14 warps at
// work) and use 35% of the issue slots in the first case, 50% in the second. Between two instructions a warp waits 4.4 and 2.5 cycles for loads (a CTA reads
// all of x, in the first case as many bytes as of weights, from L2) and 1.6 and 0.8 for results; taking bf16 codes apart (8 cycles of a
// scheduler for a pair, 2.2 for fp16) keeps the integer pipe 45% busy. The last wave is half empty (448 CTAs at 296 places). The
// instances of 64 rows of W and wide loads, which large matrices take, hold 56 to 120 bytes a thread in local memory.
// Weights through a ring in shared memory, and CTAs that stay for several rows of W, took longer than registers loaded a turn ahead.
#include "fa_kv8.cuh"

namespace {

using namespace fa::kv8;

constexpr int LW = 8;  // warps

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// bf16: a code's bits in place are its value times 2^-126, the scale goes in times 2^100, the rest at the end. fp16: values as they
// are; code times scale lies between 2^-10 and 2688.
constexpr float kScaleUp = 1.2676506002282294e30f;  // 2^100
constexpr float kRest = 67108864.0f;                // 2^26

// Two codes of a word as the two halves: bf16 codes I and I + 4 (bits put in place), fp16 codes 2 I and 2 I + 1 (one conversion,
// measured 2.2 cycles against 8 for the bits; there is none to bf16).
template <bool HALF, int I>
__device__ __forceinline__ uint32_t pair(uint32_t u) {
  if constexpr (HALF) {
    uint32_t r;
    if constexpr (I == 0) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(u));
    if constexpr (I == 1) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(u));
    if constexpr (I == 2) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(r) : "r"(u));
    if constexpr (I == 3) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(r) : "r"(u));
    return r;
  } else {
    constexpr int M = 6 - 4 * I, S = 12 - 4 * I;
    const uint32_t m = M >= 0 ? u << (M >= 0 ? M : 0) : u >> (M < 0 ? -M : 0);
    return (m & 0x01C001C0u) | ((u << S) & 0x80008000u);
  }
}
template <bool HALF>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (HALF) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// One or two E4M3 block scales (the low bytes of `two`), each as a pair of equal 16-bit factors.
template <bool HALF, int N>
__device__ __forceinline__ void factors(uint32_t two, uint32_t (&f)[N]) {
  uint32_t v = e4m3_lo_f16x2(two);
  if constexpr (!HALF) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v));
    const __nv_bfloat162 y = __floats2bfloat162_rn(x.x * kScaleUp, x.y * kScaleUp);
    v = *reinterpret_cast<const uint32_t*>(&y);
  }
  f[0] = __byte_perm(v, 0, 0x1010);
  if constexpr (N == 2) f[1] = __byte_perm(v, 0, 0x3232);
}
// A weight is read once: past L1.
__device__ __forceinline__ uint4 ldg_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

struct LinArgs {
  const void* x;
  const unsigned char *w, *bs;
  const float *ts, *bias;
  void* y;
  long long ldx, ldy;
  int M, N, K;
};

template <bool HALF, int PB, int MT, int RT>
__global__ void __launch_bounds__(LW * 32, 2) linear_kernel(const LinArgs a) {
  constexpr int WORDS = PB / 4, PK = PB * 2, GROUPS = PK / 16;  // 32-bit words, k and scale blocks of a lane's piece
  __shared__ float part[LW][16 * RT][8 * MT + 1];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * 16 * RT;
  const int pieces = (a.K + PK - 1) / PK;
  float acc[RT][MT][4] = {};
  const unsigned char *wp[RT][2], *sp[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const size_t row = min(row0 + r * 16 + i * 8 + g, a.N - 1);
      wp[r][i] = a.w + row * (a.K / 2);
      sp[r][i] = a.bs + row * (a.K / 16);
    }
  const uint16_t* xp[MT];
  bool xon[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    xon[m] = m * 8 + g < a.M;
    xp[m] = reinterpret_cast<const uint16_t*>(a.x) + (xon[m] ? (m * 8 + g) * a.ldx : 0);
  }
  // codes and scales of a piece, fetched one turn ahead of their use
  uint32_t nu[RT][2][WORDS];
  uint32_t ns[RT][2];
  auto fetch = [&](int p) {
    const bool on = p < pieces;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (PB == 16) {
          const uint4 v = on ? ldg_stream(reinterpret_cast<const uint4*>(wp[r][i]) + p) : make_uint4(0, 0, 0, 0);
          nu[r][i][0] = v.x, nu[r][i][1] = v.y, nu[r][i][2] = v.z, nu[r][i][3] = v.w;
          ns[r][i] = on ? __ldg(reinterpret_cast<const uint16_t*>(sp[r][i]) + p) : 0u;
        } else {
          const uint2 v = on ? __ldg(reinterpret_cast<const uint2*>(wp[r][i]) + p) : make_uint2(0, 0);
          nu[r][i][0] = v.x, nu[r][i][1] = v.y;
          ns[r][i] = on ? __ldg(sp[r][i] + p) : 0u;
        }
      }
  };
  fetch(w * 4 + t);
  for (int p = w * 4 + t; p - t < pieces; p += LW * 4) {
    const bool on = p < pieces;
    uint32_t u[RT][2][WORDS], f[RT][2][GROUPS];
    uint4 xv[MT][WORDS];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < WORDS; ++j)
        xv[m][j] = on && xon[m] ? __ldg(reinterpret_cast<const uint4*>(xp[m] + (size_t)p * PK) + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) u[r][i][j] = nu[r][i][j];
        factors<HALF>(ns[r][i], f[r][i]);
      }
    fetch(p + LW * 4);
#pragma unroll
    for (int j = 0; j < WORDS; ++j) {  // eight codes: two steps of the matrix instruction
      uint32_t b[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (HALF) {
          b[m][0] = xv[m][j].x, b[m][1] = xv[m][j].y, b[m][2] = xv[m][j].z, b[m][3] = xv[m][j].w;
          continue;
        }
        b[m][0] = __byte_perm(xv[m][j].x, xv[m][j].z, 0x5410);  // (x0, x4)
        b[m][1] = __byte_perm(xv[m][j].x, xv[m][j].z, 0x7632);  // (x1, x5)
        b[m][2] = __byte_perm(xv[m][j].y, xv[m][j].w, 0x5410);  // (x2, x6)
        b[m][3] = __byte_perm(xv[m][j].y, xv[m][j].w, 0x7632);  // (x3, x7)
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const uint32_t u0 = u[r][0][j], u1 = u[r][1][j], f0 = f[r][0][j / 2], f1 = f[r][1][j / 2];
        const uint32_t a0[4] = {mul2<HALF>(pair<HALF, 0>(u0), f0), mul2<HALF>(pair<HALF, 0>(u1), f1),
                                mul2<HALF>(pair<HALF, 1>(u0), f0), mul2<HALF>(pair<HALF, 1>(u1), f1)};
        const uint32_t a1[4] = {mul2<HALF>(pair<HALF, 2>(u0), f0), mul2<HALF>(pair<HALF, 2>(u1), f1),
                                mul2<HALF>(pair<HALF, 3>(u0), f0), mul2<HALF>(pair<HALF, 3>(u1), f1)};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if constexpr (HALF) {
            mma_f16(acc[r][m], a0, b[m][0], b[m][1]);
            mma_f16(acc[r][m], a1, b[m][2], b[m][3]);
          } else {
            mma_bf16(acc[r][m], a0, b[m][0], b[m][1]);
            mma_bf16(acc[r][m], a1, b[m][2], b[m][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      part[w][r * 16 + g][m * 8 + 2 * t] = acc[r][m][0];
      part[w][r * 16 + g][m * 8 + 2 * t + 1] = acc[r][m][1];
      part[w][r * 16 + g + 8][m * 8 + 2 * t] = acc[r][m][2];
      part[w][r * 16 + g + 8][m * 8 + 2 * t + 1] = acc[r][m][3];
    }
  __syncthreads();
  const float unit = __ldg(a.ts) * (HALF ? 1.0f : kRest);
  for (int i = threadIdx.x; i < 16 * RT * a.M; i += LW * 32) {
    const int r = i % (16 * RT), m = i / (16 * RT), n = row0 + r;
    if (n >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < LW; ++j) s += part[j][r][m];
    s *= unit;
    if (a.bias) s += __ldg(a.bias + n);
    if constexpr (HALF) reinterpret_cast<__half*>(a.y)[m * a.ldy + n] = __float2half(s);
    else reinterpret_cast<bf16*>(a.y)[m * a.ldy + n] = __float2bfloat16(s);
  }
}

template <bool HALF, int PB, int MT>
void launch_rows(const LinArgs& a, int sms, cudaStream_t s) {
  // Rows of W per CTA: the more, the less often x is read; as many as still give each SM two CTAs.
  if (a.N >= 64 * 2 * sms) linear_kernel<HALF, PB, MT, 4><<<(a.N + 63) / 64, LW * 32, 0, s>>>(a);
  else if (a.N >= 32 * 2 * sms) linear_kernel<HALF, PB, MT, 2><<<(a.N + 31) / 32, LW * 32, 0, s>>>(a);
  else linear_kernel<HALF, PB, MT, 1><<<(a.N + 15) / 16, LW * 32, 0, s>>>(a);
}
template <bool HALF, int PB>
void launch_tiles(const LinArgs& a, int sms, cudaStream_t s) {
  if (a.M <= 8) launch_rows<HALF, PB, 1>(a, sms, s);
  else launch_rows<HALF, PB, 2>(a, sms, s);
}

}  // namespace

extern "C" fa_status fa_nvfp4_linear(const void* x, fa_dtype dtype, int M, int K, long long ldx, const unsigned char* packed,
                                     const unsigned char* block_scale, const float* tensor_scale, const float* bias, int N,
                                     void* y, long long ldy, fa_stream stream) {
  if (dtype != FA_DT_BF16 && dtype != FA_DT_F16)
    return fail(nullptr, FA_ERR_UNSUPPORTED, "x is bf16 or fp16 (dtype %d)", (int)dtype);
  if (M < 0 || N < 1 || K < 1 || N > (1 << 30) || K > (1 << 30)) return fail(nullptr, FA_ERR_INVALID, "shape M=%d N=%d K=%d", M, N, K);
  if (M > 16) return fail(nullptr, FA_ERR_UNSUPPORTED, "M=%d rows: up to 16 are a matrix-vector product", M);
  if (K % 16) return fail(nullptr, FA_ERR_INVALID, "K=%d is not a multiple of 16", K);
  if ((M > 1 && ldx < K) || ldx % 8) return fail(nullptr, FA_ERR_INVALID, "ldx=%lld for K=%d (a multiple of 8)", ldx, K);
  if (M > 1 && ldy < N) return fail(nullptr, FA_ERR_INVALID, "ldy=%lld for N=%d", ldy, N);
  if (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(packed) % 8 || reinterpret_cast<uintptr_t>(y) % 2 ||
      reinterpret_cast<uintptr_t>(tensor_scale) % 4 || reinterpret_cast<uintptr_t>(bias) % 4)
    return fail(nullptr, FA_ERR_INVALID, "x must be 16-byte aligned, the codes 8-byte, the others to their type");
  if (M == 0) return FA_OK;
  fa_status st = check_pointers({{"x", x}, {"packed", packed}, {"block_scale", block_scale}, {"tensor_scale", tensor_scale}, {"y", y}});
  if (st != FA_OK) return st;
  if (bias && (st = check_pointers({{"bias", bias}})) != FA_OK) return st;
  // blocks write rows of y while others still read x
  const auto at = [](const void* p, long long elements) { return (long long)reinterpret_cast<uintptr_t>(p) + 2 * elements; };
  for (int i = 0; i < M; ++i)
    for (int j = 0; j < M; ++j)
      if (at(x, i * ldx) < at(y, j * ldy + N) && at(y, j * ldy) < at(x, i * ldx + K))
        return fail(nullptr, FA_ERR_INVALID, "y overlaps x");
  int dev = 0, sms = 148;
  FA_CUDA(nullptr, cudaGetDevice(&dev));
  FA_CUDA(nullptr, cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const LinArgs a{x, packed, block_scale, tensor_scale, bias, y, ldx, ldy, M, N, K};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // 16-byte pieces (two scale blocks, whose scales are one 2-byte load) where the rows allow it
  const bool wide = K % 32 == 0 && reinterpret_cast<uintptr_t>(packed) % 16 == 0 && reinterpret_cast<uintptr_t>(block_scale) % 2 == 0;
  if (dtype == FA_DT_F16) wide ? launch_tiles<true, 16>(a, sms, s) : launch_tiles<true, 8>(a, sms, s);
  else wide ? launch_tiles<false, 16>(a, sms, s) : launch_tiles<false, 8>(a, sms, s);
  FA_CUDA(nullptr, cudaGetLastError());
  return FA_OK;
}
