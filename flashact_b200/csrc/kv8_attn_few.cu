// Attention over the 8-bit cache for few query rows of a key head (one token of grouped heads),
// bound by the cache's bytes; and the merge of the splits.
//
// o = sum_j p_j vs_j V_j / sum_j p_j with p_j = 2^(s_j - max s), s_j = log2(e) scale ks_j (q . K_j):
// the codes K_j, V_j go to the matrix instruction as f16 (exact), the block scales ks and vs multiply
// the scores and the probabilities, which a thread holds for 16 consecutive keys of a 64-key chunk
// and so, with blocks of 16 or more, one factor each. q is scaled per row by a power of two into f16
// (exact: f16 has more bits than bf16, and what falls below 2^-24 of the row's largest element is
// below the scores' own rounding).
//
// Each warp works alone on every fourth 64-key chunk of the CTA's split, with its own running
// maximum and sum. The matrix instruction's operand order along d and along the keys is free as long as
// both operands share it: lane (g, t) owns bytes [16 t, 16 t + 16) of a row, so K and V are fetched in
// 16-byte pieces by the lane that uses them, through a ring of shared memory that no other lane
// reads (cp.async groups, no barrier in the loop).
#include "kv8_attn.cuh"

namespace {

using namespace fa;
using namespace fa::kv8;

constexpr int WARPS = 4, DEPTH = 6, CHUNK = 64, ROWS = 16;
constexpr float kPOff = 12.0f;  // probabilities are held as p * 2^12 in f16: down to 2^-36 of the largest

template <int D>
struct Few {
  static constexpr int NK = (D + 63) / 64;      // K pieces of 64 dims (the last may be 32)
  static constexpr int NV = (D + 63) / 64;      // V pieces of 64 dims
  static constexpr int NSUB = NK + NV;
  static constexpr int KSTEPS = D / 16;
  static constexpr int SLOT = 4096;             // 8 pieces x 32 lanes x 16 bytes
  static constexpr int RING = WARPS * DEPTH * SLOT;
  static constexpr int MERGE = WARPS * ROWS * D * 4;
  static constexpr int QF = KSTEPS * 32 * 16;
  static constexpr int BODY = RING > MERGE ? RING : MERGE;
  static constexpr int SMEM = QF + BODY + 1024;
};

template <int D>
__global__ void __launch_bounds__(WARPS * 32) few_kernel(const AttnArgs a) {
  using F = Few<D>;
  extern __shared__ __align__(16) unsigned char smem[];
  uint4* qf = reinterpret_cast<uint4*>(smem);
  unsigned char* body = smem + F::QF;
  float* rowscale = reinterpret_cast<float*>(smem + F::QF + F::BODY);  // [16]
  int* rowlim = reinterpret_cast<int*>(rowscale + ROWS);               // [16]
  float* red = reinterpret_cast<float*>(rowlim + ROWS);                // [WARPS]
  float2* wml = reinterpret_cast<float2*>(red + WARPS);                // [WARPS][16]

  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit, h = blockIdx.y, b = blockIdx.z;
  const int n = a.mask.len(b), nq = a.mask.q_len(b), pre = a.mask.prefix ? a.mask.prefix[b] : 0;
  const int row0 = tile * ROWS, nrows = min(ROWS, nq * a.group - row0);
  if (nrows <= 0) return;
  // limits grow with the token: the tile's last row sees the most
  const int top = a.mask.limit(n, nq, pre, (row0 + nrows - 1) / a.group);
  const int low = a.mask.limit(n, nq, pre, row0 / a.group);
  const int chunks = (top + CHUNK - 1) / CHUNK;
  const int c0 = split * a.split_chunks, c1 = min(chunks, c0 + a.split_chunks);
  if (c0 >= c1 && split > 0) return;  // split 0 writes the empty rows

  const size_t hd = ((size_t)b * a.layers + a.layer) * a.heads + h;
  const unsigned char* kp = a.k + hd * a.cap * D;
  const unsigned char* vp = a.v + hd * a.cap * D;
  const float *ks = a.ks + hd * (a.cap / a.block), *vs = a.vs + hd * (a.cap / a.block);
  unsigned char* ring = body + w * (DEPTH * F::SLOT) + lane * 16;

  auto issue = [&](int chunk, int sub, int slot) {
    unsigned char* dst = ring + slot * F::SLOT;
    if (chunk < c1) {
      if (sub < F::NK) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = chunk * CHUNK + 16 * (g >> 1) + 2 * i + (g & 1);
          if (D % 64 && sub == F::NK - 1)
            cp_async8_zfill(dst + i * 512, kp + (key < top ? (size_t)key * D + sub * 64 + t * 8 : 0), key < top);
          else
            cp_async16_zfill(dst + i * 512, kp + (key < top ? (size_t)key * D + sub * 64 + t * 16 : 0), key < top);
        }
      } else {
        const int key = chunk * CHUNK + 16 * t;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = (sub - F::NK) * 64 + i * 8 + g;
          if (D % 64 == 0 || d < D)
            cp_async16_zfill(dst + i * 512, vp + (key < top ? (size_t)d * a.cap + key : 0), key < top);
        }
      }
    }
    cp_async_commit();
  };
  // first pieces on their way before anything else is read
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) issue(c0 + w + (i / F::NSUB) * WARPS, i % F::NSUB, i);

  // queries: limits, power-of-two row scales, f16 fragments
  for (int r = w; r < ROWS; r += WARPS) {
    const int row = row0 + r, tok = row / a.group;
    const bool on = r < nrows;
    const long long qo = b * a.qb + tok * a.qt + (h * a.group + row % a.group) * a.qh;
    float x[D / 32], m = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      x[i] = on ? load16(a.q, qo + i * 32 + lane, a.half) : 0.f;
      m = fmaxf(m, fabsf(x[i]));
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float p2 = row_pow2(m), inv = 1.0f / p2;
    if (lane == 0) {
      rowscale[r] = p2 * a.scale_log2;
      rowlim[r] = on ? a.mask.limit(n, nq, pre, tok) : 0;
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      // element d = 64 c + 16 tq + 4 s + j (tail of 32 dims: 64 c + 8 tq + 4 s + j) of fragment step 4 c + s
      const int d = i * 32 + lane, c = d / 64, r64 = d % 64;
      const bool tail = D % 64 && c == F::NK - 1;
      const int tq = tail ? r64 / 8 : r64 / 16, s = tail ? (r64 / 4) % 2 : (r64 / 4) % 4, j = d % 4;
      // registers a0: row g, j 0..1; a1: row g + 8, j 0..1; a2: row g, j 2..3; a3: row g + 8, j 2..3
      __half* f = reinterpret_cast<__half*>(qf + (c * 4 + s) * 32 + (r & 7) * 4 + tq);
      f[((j >> 1) * 2 + (r >> 3)) * 2 + (j & 1)] = __float2half(x[i] * inv);
    }
  }
  // largest V scale of the split: the probabilities carry vs / vref <= 1
  float vref = 0.f;
  for (int i = (c0 * CHUNK) / a.block + tid; i < a.cap / a.block && i * a.block < min(top, c1 * CHUNK); i += WARPS * 32)
    vref = fmaxf(vref, vs[i]);
  for (int o = 16; o > 0; o >>= 1) vref = fmaxf(vref, __shfl_xor_sync(0xffffffffu, vref, o));
  if (lane == 0) red[w] = vref;
  __syncthreads();
  vref = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float vinv = vref > 0.f ? 1.0f / vref : 0.f;
  const float rs0 = rowscale[g], rs1 = rowscale[g + 8];
  const int lim0 = rowlim[g], lim1 = rowlim[g + 8];

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  int slot = 0;
  // a lane's 16 keys lie in one block: one K and one V scale each chunk, fetched a chunk ahead
  float kn = 0.f, vn = 0.f;
  auto scales = [&](int chunk) {
    const int key = chunk * CHUNK + 16 * t;
    const bool live = chunk < c1 && key < top;  // whole 16-key pieces lie below the capacity
    kn = live ? ks[key / a.block] : 0.f;
    vn = live ? vs[key / a.block] : 0.f;
  };
  scales(c0 + w);
  auto next = [&](int chunk, int sub) {  // piece `sub` of `chunk` has landed; fetch the one DEPTH - 1 ahead
    cp_async_wait_group<DEPTH - 2>();
    const int ahead = sub + DEPTH - 1;
    issue(chunk + (ahead / F::NSUB) * WARPS, ahead % F::NSUB, slot == 0 ? DEPTH - 1 : slot - 1);
    const unsigned char* src = ring + slot * F::SLOT;
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
    return src;
  };

  for (int chunk = c0 + w; chunk < c1; chunk += WARPS) {
    const int key0 = chunk * CHUNK + 16 * t;  // this lane's first key
    const float kscale = kn, vfac = vn * vinv;
    scales(chunk + WARPS);
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int sub = 0; sub < F::NK; ++sub) {
      const unsigned char* src = next(chunk, sub);
      const bool tail = D % 64 && sub == F::NK - 1;
      uint4 kr[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (tail) {
          const uint2 x = *reinterpret_cast<const uint2*>(src + i * 512);
          kr[i] = make_uint4(x.x, x.y, 0, 0);
        } else {
          kr[i] = *reinterpret_cast<const uint4*>(src + i * 512);
        }
      }
#pragma unroll
      for (int st = 0; st < (tail ? 2 : 4); ++st) {
        const uint4 qa = qf[(sub * 4 + st) * 32 + lane];
        const uint32_t qr[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t x = st == 0 ? kr[i].x : st == 1 ? kr[i].y : st == 2 ? kr[i].z : kr[i].w;
          mma_f16(s[i], qr, e4m3x2_f16x2(x), e4m3x2_f16x2_hi(x));
        }
      }
    }
    // scores in log2 units, masked
    const float f0 = rs0 * kscale, f1 = rs1 * kscale;
    float mx0 = -INFINITY, mx1 = -INFINITY;
    const bool whole = chunk * CHUNK + CHUNK <= low;  // seen by every row (rows behind the last are not stored)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = key0 + 2 * i + j;
        s[i][j] = whole || key < lim0 ? s[i][j] * f0 : -INFINITY;
        s[i][2 + j] = whole || key < lim1 ? s[i][2 + j] * f1 : -INFINITY;
        mx0 = fmaxf(mx0, s[i][j]);
        mx1 = fmaxf(mx1, s[i][2 + j]);
      }
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
    }
    const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
    const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
    if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
      const float r0 = exp2_approx(m0 - b0), r1 = exp2_approx(m1 - b1);
      l0 *= r0;
      l1 *= r1;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= r0;
        o[i][1] *= r0;
        o[i][2] *= r1;
        o[i][3] *= r1;
      }
      m0 = n0;
      m1 = n1;
    }
    uint32_t p[4][4];
    const float pf = vfac * 4096.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[i][j] = exp2_approx(s[i][j] - b0);
        s[i][2 + j] = exp2_approx(s[i][2 + j] - b1);
        l0 += s[i][j];
        l1 += s[i][2 + j];
      }
      p[i >> 1][(i & 1) * 2] = pack_f16x2(s[i][0] * pf, s[i][1] * pf);
      p[i >> 1][(i & 1) * 2 + 1] = pack_f16x2(s[i][2] * pf, s[i][3] * pf);
    }
    const int past = top - key0;  // V bytes from here on are behind every row's limit
#pragma unroll
    for (int sub = 0; sub < F::NV; ++sub) {
      const unsigned char* src = next(chunk, F::NK + sub);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (sub * 64 + i * 8 >= D) break;
        uint4 v = *reinterpret_cast<const uint4*>(src + i * 512);
        if (past < 16) {
          uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int left = past - 4 * q;  // bytes of this word to keep
            x[q] = left >= 4 ? x[q] : left <= 0 ? 0u : x[q] & ((1u << (8 * left)) - 1u);
          }
        }
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int st = 0; st < 4; ++st) mma_f16(o[sub * 8 + i], p[st], e4m3x2_f16x2(x[st]), e4m3x2_f16x2_hi(x[st]));
      }
    }
  }
  cp_async_wait_group<0>();
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  if (t == 0) {
    wml[w * ROWS + g] = make_float2(m0, l0);
    wml[w * ROWS + g + 8] = make_float2(m1, l1);
  }
  __syncthreads();  // every warp is done with its ring
  float* mo = reinterpret_cast<float*>(body) + w * ROWS * D;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    *reinterpret_cast<float2*>(mo + g * D + i * 8 + 2 * t) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(mo + (g + 8) * D + i * 8 + 2 * t) = make_float2(o[i][2], o[i][3]);
  }
  __syncthreads();
  const size_t slot_id = (((size_t)b * a.heads + h) * a.tiles + tile) * a.nsplit + split;
  const float unit = vref * (1.0f / 4096.0f);
  for (int r = w; r < nrows; r += WARPS) {
    float m = -INFINITY, l = 0.f, f[WARPS];
#pragma unroll
    for (int i = 0; i < WARPS; ++i) m = fmaxf(m, wml[i * ROWS + r].x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float2 x = wml[i * ROWS + r];
      f[i] = exp2_approx(x.x - base);
      l += x.y * f[i];
    }
    const int row = row0 + r, lim = rowlim[r];
    const long long oo = b * a.ob + (row / a.group) * a.ot + (h * a.group + row % a.group) * a.oh;
    const float* src = reinterpret_cast<const float*>(body) + r * D;
    const float norm = a.nsplit > 1 ? unit : lim > 0 ? unit / l : 0.f;
    for (int d = lane * 2; d < D; d += 64) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        const float2 v = *reinterpret_cast<const float2*>(src + i * ROWS * D + d);
        x += v.x * f[i];
        y += v.y * f[i];
      }
      x *= norm;
      y *= norm;
      if (a.nsplit > 1) *reinterpret_cast<float2*>(a.part + (slot_id * ROWS + r) * D + d) = make_float2(x, y);
      else if (lim > 0) store16x2(a.out, oo + d, x, y, a.half);
      else store16x2(a.out, oo + d, 0.f, 0.f, a.half);
    }
    if (a.nsplit > 1 && lane == 0) a.ml[slot_id * ROWS + r] = make_float2(m, l);
  }
}

// One warp per query row: o = sum_s 2^(m_s - m) part_s / sum_s 2^(m_s - m) l_s over the splits that the
// row's tile has, in split order (the result does not depend on which split ended first).
template <int D, int R>
__global__ void merge_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z;
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int n = a.mask.len(b), nq = a.mask.q_len(b), pre = a.mask.prefix ? a.mask.prefix[b] : 0;
  if (row >= nq * a.group) return;
  const int tile = row / R, r = row % R, last = min(tile * R + R, nq * a.group) - 1;
  const int top = a.mask.limit(n, nq, pre, last / a.group), lim = a.mask.limit(n, nq, pre, row / a.group);
  const int chunks = (top + CHUNK - 1) / CHUNK;
  const int used = max(1, (chunks + a.split_chunks - 1) / a.split_chunks);
  const size_t slot = (((size_t)b * a.heads + h) * a.tiles + tile) * a.nsplit;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < used; s += 32) m = fmaxf(m, a.ml[(slot + s) * R + r].x);
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float acc[D / 32] = {};
  for (int s = 0; s < used; ++s) {
    const float2 x = a.ml[(slot + s) * R + r];
    const float f = exp2_approx(x.x - base);
    l += x.y * f;
    const float* p = a.part + ((slot + s) * R + r) * D + lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] += f * p[i * 32];
  }
  const float norm = 1.0f / l;
  const long long oo = b * a.ob + (row / a.group) * a.ot + (h * a.group + row % a.group) * a.oh + lane;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float x = lim > 0 ? acc[i] * norm : 0.f;
    if (a.half) reinterpret_cast<__half*>(a.out)[oo + i * 32] = __float2half(x);
    else reinterpret_cast<bf16*>(a.out)[oo + i * 32] = __float2bfloat16(x);
  }
}

template <int D>
fa_status launch(const AttnArgs& a, int batch, cudaStream_t s) {
  FA_CUDA(nullptr, cudaFuncSetAttribute(few_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<D>::SMEM));
  few_kernel<D><<<dim3(a.nsplit * a.tiles, a.heads, batch), WARPS * 32, Few<D>::SMEM, s>>>(a);
  FA_CUDA(nullptr, cudaGetLastError());
  if (a.nsplit > 1) {
    merge_kernel<D, ROWS><<<dim3((a.mask.tokens * a.group + 3) / 4, a.heads, batch), 128, 0, s>>>(a);
    FA_CUDA(nullptr, cudaGetLastError());
  }
  return FA_OK;
}

}  // namespace

fa_status kv8_launch_few(const AttnArgs& a, int dim, int batch, cudaStream_t s) {
  switch (dim) {
    case 64: return launch<64>(a, batch, s);
    case 96: return launch<96>(a, batch, s);
    case 128: return launch<128>(a, batch, s);
    default: return launch<256>(a, batch, s);
  }
}
