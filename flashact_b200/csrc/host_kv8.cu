// The 8-bit KV cache behind fa_kv8_append and fa_kv8_read: tokens quantised into blocks with a
// power-of-two scale for each block and head, and the values read back as the prefix that
// fa_bind_prefix_kv takes. Measured in a graph, inputs beyond L2: 16 prompts of up to 1736 tokens, 8 key heads of 128, are written in 35 us
// (3.7 TB/s of what has to be read and written), bound by instructions: 76% of the issue slots are used, the integer pipe 49%, DRAM a third. One token
// of 64 observations takes 4 us, nearly all of it the launch and reads that depend on one another. 32 observations x 6 layers x 493
// tokens are read back in 78 us, 5.1 TB/s, with 68% of the issue slots used; a warp waits mostly for loads and for its block between
// the two halves of V's turn.
#include <type_traits>

#include "fa_kv8.cuh"

namespace {

using namespace fa::kv8;

// Exponent of the smallest power of two s with amax <= 448 s (448 = 1.75 * 2^8), at least 2^-96.
__device__ __forceinline__ int scale_exp(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
  return max(e, kMinExp);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// E4M3 code of x (already divided by the scale): nearest even, saturating; NaN has no code and becomes 0.
__device__ __forceinline__ uint32_t code_of(float x) {
  return x == x ? (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0u;
}
__device__ __forceinline__ uint32_t codes2(float x, float y) {  // of numbers that are not NaN
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
  return r;
}

// Eight consecutive elements of a row as they are, and what is asked of them.
template <class T>
struct Eight {
  static constexpr int WORDS = sizeof(T) * 2;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T* p, bool wide) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(q + 2 * i) | ((uint32_t)__ldg(q + 2 * i + 1) << 16);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  // Largest magnitude's bits (16-bit types: two running maxima in a word); magnitudes order like their bits.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7fffffffu);
      else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    return m;
  }
  __device__ __forceinline__ float2 pair(int i) const {  // elements 2 i, 2 i + 1
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <class T>
__device__ __forceinline__ float magnitude(uint32_t top) {  // of top()'s two halves
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  const uint32_t m = max(top & 0xffffu, top >> 16);
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)m));
  return __uint_as_float(m << 16);
}

struct AppendArgs {
  unsigned char *k, *v;
  float *ks, *vs;
  const void *nk, *nv;
  long long kb, kt, kh, vb, vt, vh;  // element strides of the new rows: batch, token, head
  const int *start, *count;
  int rows, layers, layer, heads, D, cap, block;
  int wide_k, wide_v;
};

// One CTA per (touched block, K or V; head; observation). A thread keeps U units of four tokens by eight dims in registers between
// the maximum over the block's new rows and their conversion: the rows are read once, nothing goes through shared memory. A warp's
// units lie along the dims for K (rows are written 8 bytes a lane) and along the tokens for V (4 tokens a lane of
// the transposed row, 64 bytes together). Rows that are already in the block keep their values: where the new scale is larger
// their codes are rounded again, which is exact but for codes that become subnormal, because the
// scales are powers of two.
template <class T, int THREADS, int U>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
  __shared__ uint32_t red[THREADS / 32];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.x & 1;
  const int start = min(max(a.start[b], 0), a.cap);
  const int n = min(a.count ? min(max(a.count[b], 0), a.rows) : a.rows, a.cap - start);
  const int base = (start / a.block + (blockIdx.x >> 1)) * a.block;
  const int lo = max(start, base), hi = min(start + n, base + a.block);
  if (lo >= hi) return;
  const long long st = is_v ? a.vt : a.kt;
  const T* src = is_v ? reinterpret_cast<const T*>(a.nv) + b * a.vb + h * a.vh : reinterpret_cast<const T*>(a.nk) + b * a.kb + h * a.kh;
  src += (long long)(base - start) * st;  // row of the block's first token
  const bool wide = is_v ? a.wide_v : a.wide_k;
  const size_t hd = ((size_t)b * a.layers + a.layer) * a.heads + h;
  float* scale = (is_v ? a.vs : a.ks) + hd * (a.cap / a.block) + base / a.block;
  const int D8 = a.D / 8, groups = a.block / 4, units = groups * D8, low = min(groups, 16);
  const float had = lo > base ? *scale : 0.f;

  Eight<T> x[U][4];
  int d[U], t[U];  // a unit's first dim and token
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = tid + i * THREADS;
    if (is_v) {
      const int r = u / low;
      d[i] = r % D8 * 8, t[i] = (r / D8 * low + u % low) * 4;
    } else {
      d[i] = u % D8 * 8, t[i] = u / D8 * 4;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = base + t[i] + j;
      if (u < units && row >= lo && row < hi) x[i][j].load(src + (t[i] + j) * st + d[i], wide);
      else x[i][j].zero();
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = x[i][j].top(top);
  auto all = [&](uint32_t v) {  // block maximum of halves (16-bit types) or words
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint32_t y = __shfl_xor_sync(0xffffffffu, v, o);
      v = sizeof(T) == 4 ? max(v, y) : __vmaxu2(v, y);
    }
    if ((tid & 31) == 0) red[tid >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < THREADS / 32; ++i) v = sizeof(T) == 4 ? max(v, red[i]) : __vmaxu2(v, red[i]);
    return magnitude<T>(v);
  };
  float amax = all(top);
  const bool odd = !(amax <= 3.402823466e38f);  // infinities or NaN among them, the same in all threads
  if (odd) {  // which do not set the scale
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 p = x[i][j].pair(k);
          if (fabsf(p.x) <= 3.402823466e38f) m = fmaxf(m, fabsf(p.x));
          if (fabsf(p.y) <= 3.402823466e38f) m = fmaxf(m, fabsf(p.y));
        }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = __float_as_uint(m);
    __syncthreads();
    amax = 0.f;
    for (int i = 0; i < THREADS / 32; ++i) amax = fmaxf(amax, __uint_as_float(red[i]));
  }
  const float now = fmaxf(pow2(scale_exp(amax)), had), inv = 1.0f / now;
  unsigned char* dst = is_v ? a.v + hd * a.D * a.cap + base : a.k + (hd * a.cap + base) * a.D;
  if (lo > base && now != had) {  // the rows that are there go to the larger scale
    const float ratio = had / now;
    const int olds = lo - base;
    for (int i = tid; i < olds * a.D; i += THREADS) {
      unsigned char* p = is_v ? dst + (size_t)(i / olds) * a.cap + i % olds : dst + i;
      *p = (unsigned char)code_of(e4m3_value(*p) * ratio);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (tid + i * THREADS >= units) break;
    uint32_t c[4][2];  // codes: token j, dims 0..3 and 4..7
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 p = x[i][j].pair(2 * k), q = x[i][j].pair(2 * k + 1);
        c[j][k] = odd ? code_of(p.x * inv) | code_of(p.y * inv) << 8 | code_of(q.x * inv) << 16 | code_of(q.y * inv) << 24
                      : codes2(p.x * inv, p.y * inv) | codes2(q.x * inv, q.y * inv) << 16;
      }
    const int row = base + t[i];
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row + j >= lo && row + j < hi) *reinterpret_cast<uint2*>(dst + (t[i] + j) * a.D + d[i]) = make_uint2(c[j][0], c[j][1]);
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // four tokens by four dims of bytes, turned around
        const uint32_t p = __byte_perm(c[0][k], c[1][k], 0x5140), q = __byte_perm(c[2][k], c[3][k], 0x5140);
        const uint32_t r = __byte_perm(c[0][k], c[1][k], 0x7362), s = __byte_perm(c[2][k], c[3][k], 0x7362);
        const uint32_t w[4] = {__byte_perm(p, q, 0x5410), __byte_perm(p, q, 0x7632), __byte_perm(r, s, 0x5410), __byte_perm(r, s, 0x7632)};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          unsigned char* o = dst + (size_t)(d[i] + 4 * k + m) * a.cap + t[i];
          if (row >= lo && row + 4 <= hi) {
            *reinterpret_cast<uint32_t*>(o) = w[m];
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (row + j >= lo && row + j < hi) o[j] = (unsigned char)(w[m] >> (8 * j));
          }
        }
      }
    }
  }
  if (tid == 0) *scale = now;
}

struct ReadArgs {
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int* lens;
  void *ok, *ov;
  int rows, layers, heads, D, cap, block, block_log2;
};

// Two codes (the low 16 bits) times a scale.
__device__ __forceinline__ float2 values2(uint32_t two, float s) {
  const uint32_t f = e4m3_lo_f16x2(two);
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&f));
  return make_float2(v.x * s, v.y * s);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float2* v) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        w[i] = pack_f16x2(v[i].x, v[i].y);
      } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[i].x, v[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One CTA per 64 tokens of a (observation, layer, head): K and V back as values [batch][layers][rows][heads * D]; rows at and behind
// the observation's length are zero. V is turned around through shared memory, words of four tokens at an index that is
// mixed with the dim so that a warp finds its words in different banks, and its rows are written whole: in pieces of 32 bytes they took
// a half longer.
constexpr int RT = 64;
template <class T>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a) {
  extern __shared__ uint32_t words[];  // [D][RT / 4], word t of row d at t ^ (d / 8 % 16)
  const int bl = blockIdx.z, h = blockIdx.y, r0 = blockIdx.x * RT, tid = threadIdx.x;
  const int len = min(min(max(a.lens[bl / a.layers], 0), a.cap), a.rows);
  const size_t hd = (size_t)bl * a.heads + h;
  const float *ks = a.ks + hd * (a.cap / a.block), *vs = a.vs + hd * (a.cap / a.block);
  const unsigned char *k = a.k + hd * a.cap * a.D, *v = a.v + hd * a.D * a.cap;
  const size_t width = (size_t)a.heads * a.D;
  T* ok = reinterpret_cast<T*>(a.ok) + (size_t)bl * a.rows * width + h * a.D;
  T* ov = reinterpret_cast<T*>(a.ov) + (size_t)bl * a.rows * width + h * a.D;
  // K: a thread has 16 dims of a row, then of the row `step` below; no division in the loop
  const int D16 = a.D / 16, step = 256 / D16, d16 = tid % D16 * 16, end = min(RT, a.rows - r0);
#pragma unroll 2
  for (int r = tid / D16; r < end && tid < step * D16; r += step) {
    float2 x[8] = {};
    if (r0 + r < len) {
      const uint4 c = __ldg(reinterpret_cast<const uint4*>(k + (size_t)(r0 + r) * a.D + d16));
      const float s = __ldg(ks + ((r0 + r) >> a.block_log2));
      x[0] = values2(c.x, s), x[1] = values2(c.x >> 16, s), x[2] = values2(c.y, s), x[3] = values2(c.y >> 16, s);
      x[4] = values2(c.z, s), x[5] = values2(c.z >> 16, s), x[6] = values2(c.w, s), x[7] = values2(c.w >> 16, s);
    }
    T* o = ok + (size_t)(r0 + r) * width + d16;
    store8<T>(o, x);
    store8<T>(o + 8, x + 4);
  }
  for (int i = tid; i < a.D * (RT / 16); i += 256) {  // the capacity is a multiple of 16: whole pieces
    const int d = i / (RT / 16), t = i % (RT / 16) * 4;
    uint4 c = make_uint4(0, 0, 0, 0);
    if (r0 + t * 4 < len) c = __ldg(reinterpret_cast<const uint4*>(v + (size_t)d * a.cap + r0 + t * 4));
    uint32_t* row = words + d * (RT / 4);
    const int mix = d / 8 % 16;
    row[t ^ mix] = c.x, row[(t + 1) ^ mix] = c.y, row[(t + 2) ^ mix] = c.z, row[(t + 3) ^ mix] = c.w;
  }
  __syncthreads();
  const int D8 = a.D / 8;
  for (int i = tid; i < D8 * (RT / 4); i += 256) {
    const int t4 = i / D8, d8 = i % D8, d = d8 * 8, r = r0 + t4 * 4;
    const float s = r < len ? __ldg(vs + (r >> a.block_log2)) : 0.f;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = words[(d + j) * (RT / 4) + (t4 ^ (d8 % 16))];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (r + t >= a.rows) break;
      float2 x[4] = {};
      if (r + t < len) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = values2(__byte_perm(w[2 * j], w[2 * j + 1], t | (t + 4) << 4), s);
      }
      store8<T>(ov + (size_t)(r + t) * width + d, x);
    }
  }
}

template <class T>
void launch_append(const AppendArgs& a, dim3 grid, cudaStream_t s) {
  // units of 4 x 8 elements: up to 1024 in a block (128 tokens of 256 dims)
  const int units = a.block / 4 * (a.D / 8);
  if (units <= 128) append_kernel<T, 128, 1><<<grid, 128, 0, s>>>(a);
  else if (units <= 256) append_kernel<T, 256, 1><<<grid, 256, 0, s>>>(a);
  else if (units <= 512) append_kernel<T, 512, 1><<<grid, 512, 0, s>>>(a);
  else append_kernel<T, 512, 2><<<grid, 512, 0, s>>>(a);
}

bool aligned16(const void* p, std::initializer_list<long long> strides, int esize) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (long long s : strides)
    if ((s * esize) % 16) return false;
  return true;
}

}  // namespace

extern "C" fa_status fa_kv8_append(const fa_kv8* c, int layer, int rows, const fa_rows* k, const fa_rows* v,
                                   fa_dtype dtype, const int* start, const int* count, fa_stream stream) {
  fa_status st = kv8_check(c);
  if (st != FA_OK) return st;
  if (layer < 0 || layer >= c->layers) return fail(nullptr, FA_ERR_INVALID, "layer %d of %d", layer, c->layers);
  if (rows < 0) return fail(nullptr, FA_ERR_INVALID, "rows=%d", rows);
  if (dtype != FA_DT_F32 && dtype != FA_DT_BF16 && dtype != FA_DT_F16)
    return fail(nullptr, FA_ERR_INVALID, "unsupported dtype %d", (int)dtype);
  if (!k || !v) return fail(nullptr, FA_ERR_INVALID, "null rows");
  const int es = (int)dtype_size(dtype);
  if (reinterpret_cast<uintptr_t>(k->ptr) % es || reinterpret_cast<uintptr_t>(v->ptr) % es)
    return fail(nullptr, FA_ERR_INVALID, "the new rows are not aligned to their type");
  if (rows == 0) return FA_OK;
  if ((st = kv8_check_pointers(c)) != FA_OK) return st;
  if ((st = check_pointers({{"k", k->ptr}, {"v", v->ptr}, {"start", start}})) != FA_OK) return st;
  if (count && (st = check_pointers({{"count", count}})) != FA_OK) return st;
  AppendArgs a{c->k, c->v, c->k_scale, c->v_scale, k->ptr, v->ptr, k->batch, k->token, k->head, v->batch, v->token,
               v->head, start, count, rows, c->layers, layer, c->heads, c->head_dim, c->capacity, c->block,
               aligned16(k->ptr, {k->batch, k->token, k->head}, es), aligned16(v->ptr, {v->batch, v->token, v->head}, es)};
  const int touched = std::min((int)(((long long)rows + c->block - 2) / c->block + 1), c->capacity / c->block);
  const dim3 grid(2 * touched, c->heads, c->batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FA_DT_F32) launch_append<float>(a, grid, s);
  else if (dtype == FA_DT_BF16) launch_append<bf16>(a, grid, s);
  else launch_append<__half>(a, grid, s);
  FA_CUDA(nullptr, cudaGetLastError());
  return FA_OK;
}

extern "C" fa_status fa_kv8_read(const fa_kv8* c, const int* lens, int rows, void* k, void* v, fa_dtype dtype,
                                 fa_stream stream) {
  fa_status st = kv8_check(c);
  if (st != FA_OK) return st;
  if (rows < 0) return fail(nullptr, FA_ERR_INVALID, "rows=%d", rows);
  if (dtype != FA_DT_F32 && dtype != FA_DT_BF16 && dtype != FA_DT_F16)
    return fail(nullptr, FA_ERR_INVALID, "unsupported dtype %d", (int)dtype);
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16)
    return fail(nullptr, FA_ERR_INVALID, "the outputs must be 16-byte aligned");
  if ((long long)c->batch * c->layers > 65535)
    return fail(nullptr, FA_ERR_INVALID, "batch x layers = %lld is over 65535", (long long)c->batch * c->layers);
  if (rows == 0) return FA_OK;
  if ((st = kv8_check_pointers(c)) != FA_OK) return st;
  if ((st = check_pointers({{"lens", lens}, {"k", k}, {"v", v}})) != FA_OK) return st;
  ReadArgs a{c->k, c->v, c->k_scale, c->v_scale, lens, k, v, rows, c->layers, c->heads, c->head_dim, c->capacity,
             c->block, __builtin_ctz(c->block)};
  const size_t smem = (size_t)c->head_dim * RT;
  const dim3 grid((rows + RT - 1) / RT, c->heads, c->batch * c->layers);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FA_DT_F32) read_kernel<float><<<grid, 256, smem, s>>>(a);
  else if (dtype == FA_DT_BF16) read_kernel<bf16><<<grid, 256, smem, s>>>(a);
  else read_kernel<__half><<<grid, 256, smem, s>>>(a);
  FA_CUDA(nullptr, cudaGetLastError());
  return FA_OK;
}
