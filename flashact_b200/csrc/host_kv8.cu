// The 8-bit KV cache behind fa_kv8_append and fa_kv8_read: tokens quantised into blocks with a
// power-of-two scale for each block and head, and the values read back as the prefix that
// fa_bind_prefix_kv takes.
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

__device__ __forceinline__ float finite_abs(float x) {
  x = fabsf(x);
  return x <= 3.402823466e38f ? x : 0.0f;  // NaN and infinities do not set the scale
}
// E4M3 code of x (already divided by the scale): nearest even, saturating; NaN has no code and becomes 0.
__device__ __forceinline__ uint32_t code_of(float x) {
  return x == x ? (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0u;
}

template <class T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float(float v) { return v; }
template <>
__device__ __forceinline__ float as_float(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// Eight consecutive elements (D is a multiple of 8): one or two 16-byte loads when aligned.
template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&v)[8]) {
  if (vec) {
    alignas(16) T t[8];
    const uint4* s = reinterpret_cast<const uint4*>(p);
    uint4* d = reinterpret_cast<uint4*>(t);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) d[i] = __ldg(s + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = as_float<T>(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = as_float<T>(p[i]);
  }
}

struct AppendArgs {
  unsigned char *k, *v;
  float *ks, *vs;
  const void *nk, *nv;
  long long kb, kt, kh, vb, vt, vh;  // element strides of the new rows: batch, token, head
  const int *start, *count;
  int rows, layers, layer, heads, D, cap, block;
  int veck, vecv;
};

// One CTA per (touched block, K or V; head; observation). Pass 1 takes the largest finite
// magnitude of the block's new rows, pass 2 reads them again (they are in L1 by then) and writes
// codes. Rows that are already in the block keep their values: where the new scale is larger
// their codes are rounded again, which is exact but for codes that become subnormal, because the
// scales are powers of two.
template <class T>
__global__ void append_kernel(AppendArgs a) {
  extern __shared__ unsigned char tile[];  // V: codes [D][block + 16]
  __shared__ float red[8];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const bool is_v = blockIdx.x & 1;
  const int start = min(max(a.start[b], 0), a.cap);
  const int n = min(a.count ? min(max(a.count[b], 0), a.rows) : a.rows, a.cap - start);
  const int blk = start / a.block + (blockIdx.x >> 1);
  const int base = blk * a.block;
  const int lo = max(start, base), hi = min(start + n, base + a.block);
  if (lo >= hi) return;
  const long long st = is_v ? a.vt : a.kt;
  const T* src = is_v ? reinterpret_cast<const T*>(a.nv) + b * a.vb + h * a.vh + (lo - start) * a.vt
                      : reinterpret_cast<const T*>(a.nk) + b * a.kb + h * a.kh + (lo - start) * a.kt;
  const bool vec = is_v ? a.vecv : a.veck;
  const size_t hd = ((size_t)b * a.layers + a.layer) * a.heads + h;
  float* scale = (is_v ? a.vs : a.ks) + hd * (a.cap / a.block) + blk;
  const int D8 = a.D / 8, work = (hi - lo) * D8;

  float m = 0.f;
  for (int i = tid; i < work; i += blockDim.x) {
    float v[8];
    load8(src + (i / D8) * st + (i % D8) * 8, vec, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[j]));
  }
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) red[tid >> 5] = m;
  const float had = lo > base ? *scale : 0.f;
  __syncthreads();
  m = red[0];
  for (int i = 1; i < (int)blockDim.x / 32; ++i) m = fmaxf(m, red[i]);
  const int e = scale_exp(m);
  const float now = fmaxf(pow2(e), had), inv = 1.0f / now, ratio = had / now;
  const bool again = lo > base && now != had;  // the rows that are there go to the larger scale

  if (!is_v) {
    unsigned char* dst = a.k + (hd * a.cap + base) * a.D;
    if (again)
      for (int i = tid; i < (lo - base) * D8; i += blockDim.x) {
        uint2 c = *reinterpret_cast<uint2*>(dst + i * 8);
        unsigned char* p = reinterpret_cast<unsigned char*>(&c);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (unsigned char)code_of(e4m3_value(p[j]) * ratio);
        *reinterpret_cast<uint2*>(dst + i * 8) = c;
      }
    for (int i = tid; i < work; i += blockDim.x) {
      float v[8];
      const int r = i / D8, d = (i % D8) * 8;
      load8(src + r * st + d, vec, v);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j >> 2] |= code_of(v[j] * inv) << (8 * (j & 3));
      *reinterpret_cast<uint2*>(dst + (size_t)(lo - base + r) * a.D + d) = make_uint2(w[0], w[1]);
    }
  } else {
    unsigned char* dst = a.v + hd * a.D * a.cap + base;  // [D][cap]
    const int pitch = a.block + 16;
    for (int i = tid; i < work; i += blockDim.x) {
      float v[8];
      const int r = i / D8, d = (i % D8) * 8;
      load8(src + r * st + d, vec, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) tile[(d + j) * pitch + lo - base + r] = (unsigned char)code_of(v[j] * inv);
    }
    const int from = again ? 0 : lo - base;  // first token of the block to write
    if (again)
      for (int i = tid; i < a.D * (lo - base); i += blockDim.x) {
        const int d = i / (lo - base), t = i % (lo - base);
        tile[d * pitch + t] = (unsigned char)code_of(e4m3_value(dst[(size_t)d * a.cap + t]) * ratio);
      }
    __syncthreads();
    const int to = hi - base;
    if (from == 0 && to == a.block) {
      const int B16 = a.block / 16;
      for (int i = tid; i < a.D * B16; i += blockDim.x) {
        const int d = i / B16, t = (i % B16) * 16;
        *reinterpret_cast<uint4*>(dst + (size_t)d * a.cap + t) = *reinterpret_cast<const uint4*>(tile + d * pitch + t);
      }
    } else {
      const int w = to - from;
      for (int i = tid; i < a.D * w; i += blockDim.x) {
        const int d = i / w, t = from + i % w;
        dst[(size_t)d * a.cap + t] = tile[d * pitch + t];
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
  int rows, layers, heads, D, cap, block;
};

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_float(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half(v); }

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  alignas(16) T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_float<T>(v[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
}

// One CTA per 64 tokens of a (observation, layer, head): K and V back as values
// [batch][layers][rows][heads * D], V turned around through shared memory; rows at and behind
// the observation's length are zero.
constexpr int RT = 64;
template <class T>
__global__ void read_kernel(ReadArgs a) {
  extern __shared__ unsigned char tile[];  // [D][RT + 4]
  const int bl = blockIdx.z, h = blockIdx.y, r0 = blockIdx.x * RT, tid = threadIdx.x;
  const int len = min(min(max(a.lens[bl / a.layers], 0), a.cap), a.rows);
  const size_t hd = (size_t)bl * a.heads + h;
  const float *ks = a.ks + hd * (a.cap / a.block), *vs = a.vs + hd * (a.cap / a.block);
  const unsigned char *k = a.k + hd * a.cap * a.D, *v = a.v + hd * a.D * a.cap;
  const size_t width = (size_t)a.heads * a.D;
  T* ok = reinterpret_cast<T*>(a.ok) + (size_t)bl * a.rows * width + h * a.D;
  T* ov = reinterpret_cast<T*>(a.ov) + (size_t)bl * a.rows * width + h * a.D;
  const int D8 = a.D / 8, n = min(RT, a.rows - r0);
  constexpr int P = RT + 4;
  for (int i = tid; i < a.D * (RT / 16); i += blockDim.x) {  // cap is a multiple of 16: whole or none
    const int d = i / (RT / 16), t = (i % (RT / 16)) * 16;
    uint4 c = make_uint4(0, 0, 0, 0);
    if (r0 + t < len) c = __ldg(reinterpret_cast<const uint4*>(v + (size_t)d * a.cap + r0 + t));
    uint32_t* w = reinterpret_cast<uint32_t*>(tile + d * P + t);
    w[0] = c.x, w[1] = c.y, w[2] = c.z, w[3] = c.w;
  }
  for (int i = tid; i < n * D8; i += blockDim.x) {
    const int r = r0 + i / D8, d = (i % D8) * 8;
    float x[8] = {};
    if (r < len) {
      const uint2 c = __ldg(reinterpret_cast<const uint2*>(k + (size_t)r * a.D + d));
      const float s = ks[r / a.block];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = e4m3_value((unsigned char)((j < 4 ? c.x : c.y) >> (8 * (j & 3)))) * s;
    }
    store8<T>(ok + (size_t)r * width + d, x);
  }
  __syncthreads();
  for (int i = tid; i < n * D8; i += blockDim.x) {
    const int t = i / D8, d = (i % D8) * 8, r = r0 + t;
    float x[8] = {};
    if (r < len) {
      const float s = vs[r / a.block];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = e4m3_value(tile[(d + j) * P + t]) * s;
    }
    store8<T>(ov + (size_t)r * width + d, x);
  }
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
  const size_t smem = (size_t)c->head_dim * (c->block + 16);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FA_DT_F32) append_kernel<float><<<grid, 256, smem, s>>>(a);
  else if (dtype == FA_DT_BF16) append_kernel<bf16><<<grid, 256, smem, s>>>(a);
  else append_kernel<__half><<<grid, 256, smem, s>>>(a);
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
             c->block};
  const dim3 grid((rows + RT - 1) / RT, c->heads, c->batch * c->layers);
  const size_t smem = (size_t)c->head_dim * (RT + 4);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == FA_DT_F32) read_kernel<float><<<grid, 256, smem, s>>>(a);
  else if (dtype == FA_DT_BF16) read_kernel<bf16><<<grid, 256, smem, s>>>(a);
  else read_kernel<__half><<<grid, 256, smem, s>>>(a);
  FA_CUDA(nullptr, cudaGetLastError());
  return FA_OK;
}
