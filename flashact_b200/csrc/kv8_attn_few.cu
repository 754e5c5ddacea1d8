// Attention over the 8-bit cache for up to 16 query rows of a key head, on the tensor cores' 8-bit kind.
//
// o = sum_j p_j vs_j V_j / sum_j p_j with p_j = 2^(s_j - max s), s_j = log2(e) scale ks_j (q . K_j). The cache's codes
// are the 128-row operand of both products as TMA brings them, S^T = K Q^T (128 keys by the query rows) and O^T = V^T P^T (128
// dims by the query rows), and nothing of the cache is converted. The other operand has more bits than eight: it is given in parts, each the
// 8-bit rounding of what the parts before it left over, scaled up, and each part has its own columns of the product, so
// that a part costs no further pass over the cache:
//   queries  E4M3 parts in units 1, 1/16 (1/256 for fp16), a row scaled by a power of two to [128, 256): bf16 rows are
//            exact down to 2^-21 of their largest element, fp16 rows to 2^-25;
//   P        E5M2 parts of p_j vs_j 2^12 / 2^d: three in units 1, 1/8, 1/64 hold what f16 holds of it, 2^-11 of a product's leading power of
//            two; for fp16 a fourth in units of 1/512 holds what f16 lost, 2^-15. All end at 2^-33 of the row's largest product: E5M2's range
//            keeps what thousands of faint keys add up to next to one loud key.
// The block scales ks, vs multiply scores and probabilities: a thread of the softmax is a key, and has one of each. 2^d is a power of two
// of the row's own, near its largest p_j vs_j so far: what a row loses goes by the keys that it sees and their weights, not by the V scales
// of a block that is masked or has no weight.
//
// One CTA takes R query rows of a (observation, key head) and a split of the keys in tiles of 128: warp 0 keeps a ring
// of K and V tiles full, warp 1 issues the products (scores of tile i + 1 before P V of tile i), warps 2..5 turn scores into
// probabilities. The running maxima (of p and of p vs) move only where one of them grew by more than 2^3, the only case that touches O^T.
//
// Measured in a graph, inputs beyond L2. Bound by the cache's bytes where it is long: one token of 8 observations at 32768 keys of 8 key heads
// of 128 takes 86 to 89 us, 6.1 TB/s. A short cache is a chain of latencies: one observation, 968 keys of one key head of 256, takes 7.7 us
// (launch 2, start and queries 2, tiles 2, join 1), and a tile about 1.05 us whatever its head_dim (1.2 with 16 rows); 64 observations at up to 1736
// keys 15.3 us, 2.9 TB/s, with two CTAs on an SM and 24% of the issue slots used. 16 rows at head_dim up to 128 need more registers than two
// CTAs leave them: about 160 bytes a thread are stored in local memory and 300 read.
// Converting the codes to f16 for the 16-bit matrix instruction took 117, 34 and 29 us: the conversion costs more
// than the products. The warp-level matrix instruction's 8-bit form is carried out in many steps here and took longer still.
#include "kv8_tc.cuh"

namespace {

using namespace fa;
using namespace fa::kv8;

constexpr int THREADS = 192;
constexpr float kPTop = 12.0f;  // log2 of P where p vs = 2^d; with maxima that lag by up to kLag, 2^15 (E5M2 ends at 57344)
constexpr float kLag = 3.0f, kSlack = 0.25f;

__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// R query rows; QP, PP parts of the queries and of P; MT tiles of 128 dims.
template <int R_, bool HALF, int MT_>
struct Cfg {
  static constexpr int R = R_, MT = MT_;
  static constexpr int QP = HALF ? 3 : 2, PP = HALF ? 4 : 3;
  static constexpr int NS = align_up(R * QP, 16), NP = align_up(R * PP, 16);  // columns of S^T and of O^T
  static constexpr int SLOT = MT * 16384;                                     // one K or V tile
  static constexpr int COLS = 2 * NS + MT * NP <= 128 ? 128 : 2 * NS + MT * NP <= 256 ? 256 : 512;
  static constexpr int QBYTES = MT * NS * 128, PBYTES = NP * 128;             // PBYTES: one of two buffers
  static constexpr int STATE = 2048;                                          // barriers and row state
  static constexpr int REST = 1024 + QBYTES + 2 * PBYTES + STATE;             // 1024: alignment of the ring
  // Two CTAs on an SM where each still has three slots, so that one starts while the other works.
  static constexpr int CTAS = COLS <= 256 && (113 * 1024 - REST) / SLOT >= 3 ? 2 : 1;
  static constexpr int SLOTS = ((CTAS == 2 ? 113 : 227) * 1024 - REST) / SLOT;
  static constexpr int SMEM = REST + SLOTS * SLOT;
  static_assert(SLOTS >= 3 && SLOTS <= 16 && R % 8 == 0 && R <= 16 && 2 * NS + MT * NP <= 512, "shared or tensor memory");
  static_assert(SLOTS * 16 + 128 <= 480 && 512 + R * 8 + R * 32 + 32 + R * 8 <= STATE && R * MT * 512 <= SLOTS * SLOT, "state");
};

template <int R, bool HALF, int MT>
__global__ void __launch_bounds__(THREADS, (Cfg<R, HALF, MT>::CTAS))
    few_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<R, HALF, MT>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* ring = smem;
  unsigned char* qs = smem + C::SLOTS * C::SLOT;  // [MT][NS][128]
  unsigned char* ps = qs + C::QBYTES;             // [2][NP][128]
  unsigned char* state = ps + 2 * C::PBYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(state);  // [SLOTS] tile has landed
  uint64_t* empty = full + C::SLOTS;                    // [SLOTS] its products are done
  uint64_t* sfull = empty + C::SLOTS;                   // [2] scores are in tensor memory
  uint64_t* sfree = sfull + 2;                          // [2] and have been read
  uint64_t* pfull = sfree + 2;                          // [2] probabilities are in shared memory
  uint64_t* pvdone = pfull + 2;                         // [2] and their product is done
  uint64_t* seen = pvdone + 2;                          // [2] the four warps' maxima are in wmax
  uint64_t* drained = seen + 2;                         // all products are done, after a wait that ran out
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* err = reinterpret_cast<volatile int*>(tmem_ptr + 1);  // [2] error word, limit of a wait
  uint64_t* maxes = reinterpret_cast<uint64_t*>(state + 480);  // the four warps' maxima are in wmax
  float* rowscale = reinterpret_cast<float*>(state + 512);     // [R]
  int* rowlim = reinterpret_cast<int*>(rowscale + R);          // [R]
  float* wmax = reinterpret_cast<float*>(rowlim + R);          // [4][2][R] of a warp's scores, of its scores and log2 vs
  int* flags = reinterpret_cast<int*>(wmax + 8 * R);           // [2][4] a warp of the softmax saw a larger maximum
  float2* mls = reinterpret_cast<float2*>(flags + 8);          // [R] maximum and sum of the split, for the cluster
  float* osum = reinterpret_cast<float*>(ring);                // [R][PITCH] and its sums, once the ring is done
  constexpr int PITCH = MT * 128;

  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit, h = blockIdx.y, b = blockIdx.z;
  const int row0 = tile * R;
  const size_t hd = ((size_t)b * a.layers + a.layer) * a.heads + h;
  const float *ks = a.ks + hd * a.blocks, *vs = a.vs + hd * a.blocks;
  const int quad = w & 3, key_lane = quad * 32 + lane, st = tid - 64;  // tensor memory lane; thread of the softmax's 128
  constexpr int RW = R / 4;  // query rows of a softmax warp: quad, quad + 4, ..; a lane holds dims 128 i + 4 lane .. + 3
  uint2 q[RW][MT];
  if (w >= 2) {
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      const int row = row0 + quad + 4 * j;
      const bool in = token_of(a, row) < a.mask.tokens;
      const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q) + row_at(a, b, h, row, a.qb, a.qt, a.qh) + lane * 4;
#pragma unroll
      for (int i = 0; i < MT; ++i) q[j][i] = in && i * 128 + lane * 4 < a.dim ? ldg_row4(p + i * 128) : make_uint2(0, 0);
    }
  }
  const int n = a.mask.len(b), nq = a.mask.q_len(b), pre = a.mask.prefix ? a.mask.prefix[b] : 0;
  const int nrows = min(R, nq * a.group - row0);
  if (nrows <= 0) return;  // of all CTAs of a cluster
  // limits grow with the token: the tile's last row sees the most
  const int top = a.mask.limit(n, nq, pre, token_of(a, row0 + nrows - 1));
  const int low = a.mask.limit(n, nq, pre, token_of(a, row0));
  const int all = (top + TILE - 1) / TILE, each = a.cluster ? (all + a.nsplit - 1) / a.nsplit : a.split_chunks;
  const int t0 = split * each, nt = min(all, t0 + each) - t0;
  launch_dependents();
  const size_t first_part = ((((size_t)b * a.heads + h) * a.tiles + tile) * a.nsplit + split) * R;
  if (nt <= 0) {  // nothing left for this split
    if (a.nsplit > 1 && !a.cluster && split > 0) return;  // the merge knows
    // An SM takes no second block while one may still allocate tensor memory, and this one waits for its cluster: 57 observations of 100
    // keys planned for 156 took 14.0 us, 8.6 with this.
    if (w == 1) tmem_relinquish();
    for (int i = tid; i < R * PITCH; i += THREADS) osum[i] = 0.f;
    if (tid < R) mls[tid] = make_float2(-INFINITY, 0.f);
    finish_rows<HALF, MT, 1>(a, osum, PITCH, reinterpret_cast<const float*>(mls), 2, split, b, h, row0, nrows, n, nq, pre, first_part);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + i, 1);
      mbar_init(sfree + i, 4);
      mbar_init(pfull + i, 128);
      mbar_init(pvdone + i, 1);
      mbar_init(seen + i, 4);
    }
    mbar_init(maxes, 4);
    mbar_init(drained, 1);
    err[0] = 0, err[1] = a.spin_limit;
    fence_mbar_init();
    produce<1, C::SLOTS, MT>(ring, full, empty, &kmap, &vmap, t0, nt, (int)hd, err, 0, min(C::SLOTS, 2 * nt));
  }
  if (w == 1) {
    tmem_alloc(tmem_ptr, C::COLS);
    tmem_relinquish();
  }
  // scales of this thread's key in the first tile
  float k_first = 0.f, v_first = 0.f;
  if (w >= 2) {
    const int key = t0 * TILE + key_lane;
    if (key < top) {
      k_first = ldg_now(ks + (key >> a.block_log2));
      v_first = ldg_now(vs + (key >> a.block_log2));
    }
    // queries: limits, power-of-two row scales, E4M3 parts; rows behind the last are zero
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      const int r = quad + 4 * j;
      const bool on = r < nrows;
      float x[MT][4], m = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float2 u = pair_f32<HALF>(q[j][i].x), v = pair_f32<HALF>(q[j][i].y);
        x[i][0] = u.x, x[i][1] = u.y, x[i][2] = v.x, x[i][3] = v.y;
        m = fmaxf(m, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(v.x), fabsf(v.y))));
      }
      m = warp_max(m);
      float back;
      const float up = row_factor(m, back), mul = on ? up : 0.f;
      if (lane == 0) {
        rowscale[r] = back * a.scale_log2;
        rowlim[r] = on ? a.mask.limit(n, nq, pre, token_of(a, row0 + r)) : 0;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float y[4] = {x[i][0] * mul, x[i][1] * mul, x[i][2] * mul, x[i][3] * mul};
        split_query<C::QP>(y, 16.f, [&](int p, uint32_t e) {
          *reinterpret_cast<uint32_t*>(qs + i * C::NS * 128 + swz(p * R + r, lane * 4)) = e;
        });
      }
    }
    // columns that pad the products to 16: never read, but kept finite
#pragma unroll
    for (int i = 0; i < MT; ++i)
      for (int j = st; j < (C::NS - C::QP * R) * 8; j += 128)
        *reinterpret_cast<uint4*>(qs + i * C::NS * 128 + C::QP * R * 128 + j * 16) = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      for (int j = st; j < (C::NP - C::PP * R) * 8; j += 128)
        *reinterpret_cast<uint4*>(ps + i * C::PBYTES + C::PP * R * 128 + j * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_shared();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const uint32_t tmem_o = tmem + 2 * C::NS;
  int issued = 0;  // tiles that the producer has sent for

  if (w == 0) {
    if (lane == 0) issued = produce<1, C::SLOTS, MT>(ring, full, empty, &kmap, &vmap, t0, nt, (int)hd, err, min(C::SLOTS, 2 * nt), 2 * nt);
    __syncwarp();
  } else if (w == 1) {
    const int steps = a.dim / 32;
    constexpr uint32_t ids = idesc_f8(C::NS, false, false), idp = idesc_f8(C::NP, false, true);
    const uint32_t qb = desc_lo(qs), pb = desc_lo(ps);
    bool ok = true;
    auto scores = [&](int i) {
      const int pos = pos_k<1>(i), slot = pos % C::SLOTS;
      ok = ok && wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
      ok = ok && (i < 2 || wait_for(sfree + (i & 1), ((i >> 1) - 1) & 1, err, ERR_SFREE));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t ka = desc_lo(ring + slot * C::SLOT), d = tmem + (i & 1) * C::NS;
#pragma unroll
      for (int k = 0; k < MT * 4; ++k)
        if (k < steps) mma_f8(d, ka + (k >> 2) * 1024 + (k & 3) * 2, qb + (k >> 2) * C::NS * 8 + (k & 3) * 2, ids, k > 0);
      if (i > 0 || split != a.fault_split) tc_commit_elect(sfull + (i & 1));
      tc_commit_elect(empty + slot);
    };
    scores(0);
    for (int i = 0; i < nt && ok; ++i) {
      if (i + 1 < nt) scores(i + 1);
      const int pos = pos_v<1>(i, nt), slot = pos % C::SLOTS;
      ok = ok && wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
      ok = ok && wait_for(pfull + (i & 1), (i >> 1) & 1, err, ERR_P);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t va = desc_lo(ring + slot * C::SLOT), pi = pb + (i & 1) * (C::PBYTES / 16);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_f8(tmem_o + m * C::NP, va + m * 1024 + k * 2, pi + k * 2, idp, i > 0 || k > 0);
      tc_commit_elect(pvdone + (i & 1));
      tc_commit_elect(empty + slot);
    }
  } else {
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    // The subtracted maximum and the exponent d of p vs, a whole number (both the same in all threads), this key lane's sum.
    float m[R], d[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) m[r] = -INFINITY, d[r] = 0.f, l[r] = 0.f;
    float kn = k_first, vn = v_first;
    int grown = 0;  // times that the maximum moved
    auto scales = [&](int i) {
      const int key = (t0 + i) * TILE + key_lane;
      const bool live = i < nt && key < top;
      kn = live ? ks[key >> a.block_log2] : 0.f;
      vn = live ? vs[key >> a.block_log2] : 0.f;
    };
    bool ok = true;
    for (int i = 0; i < nt; ++i) {
      const int key = (t0 + i) * TILE + key_lane;
      const float kscale = kn, lv = log2_approx(vn);
      scales(i + 1);
      ok = wait_for(sfull + (i & 1), (i >> 1) & 1, err, ERR_S);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      float s[R];
      {
        const uint32_t ts = tmem + lanes + (i & 1) * C::NS;
        float v[C::NS];
#pragma unroll
        for (int c = 0; c < C::NS; c += 16) tmem_ld16(ts + c, v + c);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sfree + (i & 1));
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r] = v[r] + v[R + r] * 0.0625f;
          if (HALF) s[r] += v[(C::QP - 1) * R + r] * (1.0f / 256.0f);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] *= rowscale[r] * kscale;
      if ((t0 + i) * TILE + TILE > low) {  // not seen by every row
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = key < rowlim[r] ? s[r] : -INFINITY;
      }
      bool grew = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float t = s[r] - m[r];
        grew |= t > kLag || t + lv > d[r] + kLag;
      }
      grew = __any_sync(0xffffffffu, grew);
      if (lane == 0) {
        flags[(i & 1) * 4 + quad] = grew;
        mbar_arrive(seen + (i & 1));
      }
      ok = wait_for(seen + (i & 1), (i >> 1) & 1, err, ERR_SEEN);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int4 fl = *reinterpret_cast<const int4*>(flags + (i & 1) * 4);
      if (fl.x | fl.y | fl.z | fl.w) {  // the same in all 128 threads
        float x[2 * R];
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = warp_max(s[r]);
        if (a.block_log2 >= 5) {  // a warp's 32 keys are of one block
          const float lw = __shfl_sync(0xffffffffu, lv, 0);
#pragma unroll
          for (int r = 0; r < R; ++r) x[R + r] = x[r] + lw;
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) x[R + r] = warp_max(s[r] + lv);
        }
        if (lane == 0) {
#pragma unroll
          for (int r = 0; r < 2 * R; r += 4)
            *reinterpret_cast<float4*>(wmax + quad * 2 * R + r) = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
          mbar_arrive(maxes);
        }
        ok = wait_for(maxes, grown & 1, err, ERR_SEEN);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ++grown;
        float f[R];
#pragma unroll
        for (int r = 0; r < 2 * R; r += 4) {
          float4 y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = *reinterpret_cast<const float4*>(wmax + k * 2 * R + r);
          x[r] = fmaxf(fmaxf(y[0].x, y[1].x), fmaxf(y[2].x, y[3].x)), x[r + 1] = fmaxf(fmaxf(y[0].y, y[1].y), fmaxf(y[2].y, y[3].y));
          x[r + 2] = fmaxf(fmaxf(y[0].z, y[1].z), fmaxf(y[2].z, y[3].z)), x[r + 3] = fmaxf(fmaxf(y[0].w, y[1].w), fmaxf(y[2].w, y[3].w));
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float mn = fmaxf(m[r], x[r]), nv = fmaxf(m[r] + d[r], x[R + r]);
          const float down = mn == -INFINITY ? 0.f : m[r] - mn;
          const float dn = mn == -INFINITY ? 0.f : fminf(fmaxf(ceilf(nv - mn - kSlack), -114.f), 126.f);
          f[r] = exp2_approx(down + (d[r] - dn));
          l[r] *= exp2_approx(down);
          m[r] = mn, d[r] = dn;
        }
        if (i > 0) {
          ok = wait_for(pvdone + ((i - 1) & 1), ((i - 1) >> 1) & 1, err, ERR_PV);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int c = 0; c < C::NP; c += 16) {
              float v[16];
              uint32_t u[16];
              tmem_ld16(tmem_o + lanes + mt * C::NP + c, v);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(c + j < C::PP * R ? v[j] * f[(c + j) % R] : v[j]);
              tmem_st16(tmem_o + lanes + mt * C::NP + c, u);
            }
          tc_wait_st();
          tc_fence_before();
        }
      }
      if (i >= 2) {
        ok = wait_for(pvdone + (i & 1), ((i >> 1) - 1) & 1, err, ERR_PV);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      unsigned char* pb = ps + (i & 1) * C::PBYTES;
#pragma unroll
      for (int r = 0; r < R; r += 2) {
        const float x = s[r] - (m[r] == -INFINITY ? 0.f : m[r]), y = s[r + 1] - (m[r + 1] == -INFINITY ? 0.f : m[r + 1]);
        l[r] += exp2_approx(x);
        l[r + 1] += exp2_approx(y);
        const float px = exp2_approx(x + (lv + kPTop - d[r])), py = exp2_approx(y + (lv + kPTop - d[r + 1]));
        uint32_t p = pack_f16x2(px, py);
        [[maybe_unused]] const uint32_t lost = HALF ? __byte_perm(f16_lost(px, py, p, 512.f), 0, 0x1404) : 0u;
#pragma unroll
        for (int k = 0; k < C::PP; ++k) {
          const uint32_t e = k < 3 ? round_part(p) : lost;
          pb[swz(k * R + r, key_lane)] = (unsigned char)(e >> 8);
          pb[swz(k * R + r + 1, key_lane)] = (unsigned char)(e >> 24);
          if (k < 2) p = rest8(p, e);
        }
      }
      const int left = top - (t0 + i) * TILE;
      if (left < TILE) {
        // keys behind the last limit have P = 0, but their V codes may be NaN: clear them in the tile
        const int pos = pos_v<1>(i, nt), slot = pos % C::SLOTS;
        ok = wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        clear_behind(ring + slot * C::SLOT, MT * 128, left, st, 128);
      }
      fence_proxy_async_shared();
      mbar_arrive(pfull + (i & 1));
    }
    if (ok) ok = wait_for(pvdone + ((nt - 1) & 1), ((nt - 1) >> 1) & 1, err, ERR_PV);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    // sums of the rows over the 128 key lanes: through the free P buffers, a warp adds up each fourth row
    float* ls = reinterpret_cast<float*>(ps);
#pragma unroll
    for (int r = 0; r < R; ++r) ls[r * 128 + st] = l[r];
    bar_softmax();
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      const int r = quad + 4 * j;
      float x = (ls[r * 128 + lane] + ls[r * 128 + 32 + lane]) + (ls[r * 128 + 64 + lane] + ls[r * 128 + 96 + lane]);
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      float top_m = -INFINITY;
#pragma unroll
      for (int k = 0; k < R; ++k) top_m = k == r ? m[k] : top_m;
      if (lane == 0) mls[r] = make_float2(top_m, x);
    }
    float unit[R];
#pragma unroll
    for (int r = 0; r < R; ++r) unit[r] = __int_as_float(((int)d[r] - (int)kPTop + 127) << 23);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float v[C::NP];
#pragma unroll
      for (int c = 0; c < C::NP; c += 16) tmem_ld16(tmem_o + lanes + mt * C::NP + c, v + c);
      tc_wait_ld();
      const int d = mt * 128 + key_lane;
      if (d < a.dim) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= nrows) break;
          float x = v[r] + v[R + r] * 0.125f + v[2 * R + r] * (1.0f / 64.0f);
          if (HALF) x += v[(C::PP - 1) * R + r] * (1.0f / 512.0f);
          osum[r * PITCH + d] = x * unit[r];
        }
      }
      __syncwarp();
    }
    tc_fence_before();
  }
  __syncthreads();
  if (*err) give_up<C::SLOTS>(full, issued, drained, w == 1, osum, PITCH, PITCH, reinterpret_cast<float*>(mls), 2, R);
  if (w == 1) tmem_dealloc(tmem, C::COLS);
  finish_rows<HALF, MT, 1>(a, osum, PITCH, reinterpret_cast<const float*>(mls), 2, split, b, h, row0, nrows, n, nq, pre, first_part);
}

template <int R, bool HALF, int MT>
fa_status launch(const AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  constexpr int SMEM = Cfg<R, HALF, MT>::SMEM;
  return kv8_launch<few_kernel<R, HALF, MT>>(a, batch, THREADS, SMEM, km, vm, s);
}
template <int R, bool HALF, int MT>
int resident(int device, int n) {
  return kv8_resident<few_kernel<R, HALF, MT>>(device, n, THREADS, Cfg<R, HALF, MT>::SMEM);
}
template <int R>
fa_status launch_rows(const AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  if (a.dim <= 128) return a.half ? launch<R, true, 1>(a, batch, km, vm, s) : launch<R, false, 1>(a, batch, km, vm, s);
  return a.half ? launch<R, true, 2>(a, batch, km, vm, s) : launch<R, false, 2>(a, batch, km, vm, s);
}

}  // namespace

fa_status kv8_launch_few(const AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  return a.rows == 8 ? launch_rows<8>(a, batch, km, vm, s) : launch_rows<16>(a, batch, km, vm, s);
}

int kv8_resident_few(int rows, bool half, int dim, int device, int n) {
  if (rows == 8) {
    if (dim <= 128) return half ? resident<8, true, 1>(device, n) : resident<8, false, 1>(device, n);
    return half ? resident<8, true, 2>(device, n) : resident<8, false, 2>(device, n);
  }
  if (dim <= 128) return half ? resident<16, true, 1>(device, n) : resident<16, false, 1>(device, n);
  return half ? resident<16, true, 2>(device, n) : resident<16, false, 2>(device, n);
}
