// Attention over the 8-bit cache for many query rows of a key head, 128 at a time, on the tensor cores' 8-bit kind; bound
// by their rate.
//
// o = sum_j p_j vs_j V_j / sum_j p_j with p_j = 2^(s_j - max s), s_j = log2(e) scale ks_j (q . K_j). The cache's codes go into both
// products as TMA brings them, S = Q K^T and O = P V; queries and probabilities, which have more than eight bits, are
// sums of 8-bit parts, each the rounding of what the parts before it left over, and every part is one more product into the same sums:
//   queries  two E4M3 parts (three for fp16) of a row scaled by a power of two to [128, 256): off by at most 2^-10, that is 2^-17 of
//            the row's largest element, where E4M3's smallest steps end it;
//   P        E5M2 parts of p_j vs_j 2^14 / 2^d: three hold what f16 holds of it, 2^-11 of a product's leading power of two; for fp16 a
//            fourth holds what f16 lost, 2^-15. They end at 2^-29 of the row's largest product. 2^d is the row's own, near its largest p_j vs_j
//            so far: what a row loses goes by the keys that it sees and their weights, not by the V scales of a block that is masked or has no
//            weight. fp16 without the fourth part took 65.4 us instead of 76.2 (256 tokens, below), 1.3 times the plain form's error instead of 1.0.
// That is 2 + 3 products at the 8-bit rate against the 2 + 2 that one bf16 product each would cost at half that rate,
// without converting the cache or holding it in 16 bits in shared memory, whose bandwidth would bound it.
//
// P goes to tensor memory, whence the second product reads it as its first operand: shared memory then holds the queries' parts and
// five slots of K and V tiles at head_dim 256 (with P in shared memory three, and the products waited for tiles).
//
// Warp 0 keeps a ring of K and V tiles (128 keys) full, warp 1 issues the scores' products (up to two tiles ahead), warp 2
// those of P and V, warps 4..11 turn scores into probabilities: a thread has one query row and half of the tile's keys, and
// the two threads of a row exchange their maxima, those of tile i + 1 while they write P of tile i. The running maxima (of p and of
// p vs) move only where one of them grew by more than 2^1, the only case that touches O.
//
// Measured in a graph at head_dim 256 (bf16): a tile takes 2.2 to 2.6 us, its products 2560 cycles of that (64 for a score product of K = 32,
// 128 for one of P V); a CTA's start 4 us, 2 of them the queries' parts, its end 5. 16 observations of 50 tokens and 8
// query heads on one key head at 1018 keys: 25.7 us (260 TFLOP/s, each product counted once; the tensor cores are busy 16% of it, 35% of the
// issue slots are used); 4 of 256 tokens in fp16 at up to 4096: 76 us (364; 28% and 39%). With 16-bit products and converted tiles these took 74
// and 222 us. The fp16 instances hold 24 bytes a thread in local memory. Rows come here from 17 on: a tile of 128 costs the same however
// many of its rows are used; kv8_attn_few.cu, which gives each part of each row its own columns, is built for 8 and 16 (32 would fit
// its tensor memory too: 320 columns in bf16 and 448 in fp16 at head_dim 256).
#include "kv8_tc.cuh"

namespace {

using namespace fa;
using namespace fa::kv8;

constexpr int THREADS = 384, ROWS = 128, SOFT = 4;  // SOFT: first softmax warp
constexpr float kPTop = 14.0f;  // log2 of P where p vs = 2^d; with a maximum that lags by up to kLag and kSlack, 2^15.25 (E5M2 ends at 57344)
constexpr float kLag = 1.0f, kSlack = 0.25f;

template <bool HALF, int MT_>
struct Cfg {
  static constexpr int MT = MT_;
  static constexpr int QP = HALF ? 3 : 2, PP = HALF ? 4 : 3;
  static constexpr int SLOT = MT * 16384, QBYTES = QP * MT * 16384;
  static constexpr int STATE = 3072, REST = QBYTES + STATE;
  static constexpr int SLOTS_ = (227 * 1024 - REST) / SLOT, SLOTS = SLOTS_ > 8 ? 8 : SLOTS_;
  static constexpr int SMEM = REST + SLOTS * SLOT;
  static_assert(ROWS * (MT * 128 + 4) * 4 <= SLOTS * SLOT + QBYTES, "sums of a split");
  static_assert(SLOTS >= 2, "shared memory");  // K and V of a tile; scores of the next need K's slot only
};

__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <bool HALF, int MT>
__global__ void __launch_bounds__(THREADS, 1)
    rows_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HALF, MT>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* ring = smem;
  unsigned char* qs = smem + C::SLOTS * C::SLOT;  // [part][MT][128][128]
  unsigned char* state = qs + C::QBYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(state);  // [SLOTS] tile has landed
  uint64_t* empty = full + C::SLOTS;                    // [SLOTS] its products are done
  uint64_t* sfull = empty + C::SLOTS;                   // scores are in tensor memory
  uint64_t* sfree = sfull + 1;                          // and have been read
  uint64_t* pfull = sfree + 1;                          // probabilities are in tensor memory
  uint64_t* pvdone = pfull + 1;                         // and their product is done
  uint64_t* seen = pvdone + 1;                          // the eight warps' maxima are in half_max
  uint64_t* drained = seen + 1;                         // all products are done, after a wait that ran out
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* err = reinterpret_cast<volatile int*>(tmem_ptr + 1);  // [2] error word, limit of a wait
  float* half_max = reinterpret_cast<float*>(state + 512);  // [2][2][128], a tile's maxima in the one of its parity
  signed char* half_exp = reinterpret_cast<signed char*>(state + 2560);  // [2][2][128], the exponent of p vs above each of them
  float* rowscale = half_max + 2 * ROWS;                    // [128], read before the second tile's maxima
  float* osum = reinterpret_cast<float*>(smem);             // [128][PITCH] sums of the split and, behind a row, its maximum and sum
  constexpr int PITCH = MT * 128 + 4;

  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int split = blockIdx.x % a.nsplit, tile = blockIdx.x / a.nsplit, h = blockIdx.y, b = blockIdx.z;
  const int row0 = tile * ROWS;
  const size_t hd = ((size_t)b * a.layers + a.layer) * a.heads + h;
  const float *ks = a.ks + hd * a.blocks, *vs = a.vs + hd * a.blocks;
  const int n = a.mask.len(b), nq = a.mask.q_len(b), pre = a.mask.prefix ? a.mask.prefix[b] : 0;
  const int nrows = min(ROWS, nq * a.group - row0);
  if (nrows <= 0) return;  // of all CTAs of a cluster
  // limits grow with the token: the tile's last row sees the most
  const int top = a.mask.limit(n, nq, pre, token_of(a, row0 + nrows - 1));
  const int low = a.mask.limit(n, nq, pre, token_of(a, row0));
  const int all = (top + TILE - 1) / TILE, each = a.cluster ? (all + a.nsplit - 1) / a.nsplit : a.split_chunks;
  const int t0 = split * each, nt = min(all, t0 + each) - t0;
  launch_dependents();
  const size_t first_part = ((((size_t)b * a.heads + h) * a.tiles + tile) * a.nsplit + split) * ROWS;
  if (nt <= 0) {  // nothing left for this split
    if (a.nsplit > 1 && !a.cluster && split > 0) return;  // the merge knows
    for (int i = tid; i < ROWS * PITCH; i += THREADS) osum[i] = i % PITCH == MT * 128 ? -INFINITY : 0.f;
    finish_rows<HALF, MT, 4>(a, osum, PITCH, osum + MT * 128, PITCH, split, b, h, row0, nrows, n, nq, pre, first_part);
    return;
  }

  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(sfull, 1);
    mbar_init(sfree, 8);
    mbar_init(pfull, 256);
    mbar_init(pvdone, 1);
    mbar_init(seen, 8);
    mbar_init(drained, 2);
    err[0] = 0, err[1] = a.spin_limit;
    fence_mbar_init();
    produce<2, C::SLOTS, MT>(ring, full, empty, &kmap, &vmap, t0, nt, (int)hd, err, 0, min(C::SLOTS, 2 * nt));
  }
  if (w == 1) {
    tmem_alloc(tmem_ptr, 512);
    tmem_relinquish();
  }
  if (w >= SOFT) {
    // queries: power-of-two row scales and E4M3 parts; rows behind the last are zero
    constexpr int LANES = MT * 16, PER = 32 / LANES, N = 16 / PER;  // lanes of a row, rows at a time, such groups of the warp's 16 rows
    const int l8 = (lane % LANES) * 8;                              // this lane's dims, l8 .. + 7
    // row addresses by the first 16 lanes, once; zero for rows that the call does not have
    unsigned long long at = 0;
    {
      const int r = row0 + (w - SOFT) * 16 + (lane & 15);
      if (token_of(a, r) < a.mask.tokens)
        at = reinterpret_cast<unsigned long long>(reinterpret_cast<const uint16_t*>(a.q) + row_at(a, b, h, r, a.qb, a.qt, a.qh));
    }
    // A row as it is waits where its parts will be (512 bytes either way at head_dim 256): all rows are on their way at once.
    auto place = [&](int j) {
      const int r = (w - SOFT) * 16 + j * PER + lane / LANES, piece = lane % LANES;
      return reinterpret_cast<uint4*>(qs + (piece >> 3) * 16384 + swz(r, (piece & 7) * 16));
    };
    if (a.q_wide) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const unsigned long long base = __shfl_sync(0xffffffffu, at, j * PER + lane / LANES);
        const bool on = base && l8 < a.dim;
        cp_async16_zfill(place(j), on ? reinterpret_cast<const void*>(base + l8 * 2) : a.q, on);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < N; ++j) {
        const unsigned long long base = __shfl_sync(0xffffffffu, at, j * PER + lane / LANES);
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + l8;
        uint32_t u[4] = {0, 0, 0, 0};
        if (base && l8 < a.dim) {
#pragma unroll
          for (int k = 0; k < 4; ++k) u[k] = (uint32_t)__ldg(p + 2 * k) | ((uint32_t)__ldg(p + 2 * k + 1) << 16);
        }
        *place(j) = make_uint4(u[0], u[1], u[2], u[3]);
        __syncwarp();
      }
    }
    auto largest = [&](uint4 q) {
      const float2 x[4] = {pair_f32<HALF>(q.x), pair_f32<HALF>(q.y), pair_f32<HALF>(q.z), pair_f32<HALF>(q.w)};
      return max3(max3(fabsf(x[0].x), fabsf(x[0].y), fabsf(x[1].x)), max3(fabsf(x[1].y), fabsf(x[2].x), fabsf(x[2].y)),
                  fmaxf(fabsf(x[3].x), fabsf(x[3].y)));
    };
    auto split = [&](int j, uint4 q, float m) {
      const int r = (w - SOFT) * 16 + j * PER + lane / LANES;
      const float2 x[4] = {pair_f32<HALF>(q.x), pair_f32<HALF>(q.y), pair_f32<HALF>(q.z), pair_f32<HALF>(q.w)};
      float back;
      const float up = row_factor(m, back), mul = r < nrows ? copysignf(up, a.scale_log2) : 0.f;
      if (l8 == 0) rowscale[r] = back * fabsf(a.scale_log2);
      // scaled elements are f16 numbers (what is below 2^-24 is far below the parts' end), and so are the remainders
      uint32_t y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = pack_f16x2(x[k].x * mul, x[k].y * mul);
      unsigned char* dst = qs + (l8 >> 7) * 16384 + swz(r, l8 & 127);
#pragma unroll
      for (int p = 0; p < C::QP; ++p) {
        uint32_t e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          e[k] = f16x2_e4m3x2(y[k]);
          if (p + 1 < C::QP) {
            const uint32_t v = e4m3_lo_f16x2(e[k]);
            const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&y[k]), *reinterpret_cast<const __half2*>(&v));
            y[k] = *reinterpret_cast<const uint32_t*>(&d);
          }
        }
        *reinterpret_cast<uint2*>(dst + p * MT * 16384) = make_uint2(e[0] | (e[1] << 16), e[2] | (e[3] << 16));
      }
    };
    cp_async_wait_all();
    __syncwarp();
#pragma unroll 1
    for (int j0 = 0; j0 < N; j0 += 4) {  // four rows' chains side by side; all in straight code would be fetched cold
      uint4 q[4];
      float m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *place(j0 + j);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = largest(q[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (MT == 2) {
          m[j] = warp_max(m[j]);
        } else {
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], o));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) split(j0 + j, q[j], m[j]);
    }
    fence_proxy_async_shared();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_o = *tmem_ptr, tmem_s = tmem_o + 256, tmem_p = tmem_o + 384;  // O, scores, parts of P (32 columns each)
  int issued = 0;  // tiles that the producer has sent for

  if (w == 0) {
    if (lane == 0) issued = produce<2, C::SLOTS, MT>(ring, full, empty, &kmap, &vmap, t0, nt, (int)hd, err, min(C::SLOTS, 2 * nt), 2 * nt);
    __syncwarp();
  } else if (w == 1) {
    const int steps = a.dim / 32;
    const uint32_t ids = idesc_f8(TILE, false, false);
    const uint32_t qa = desc_lo(qs);
    bool ok = true;
    auto scores = [&](int i) {
      const int pos = pos_k<2>(i), slot = pos % C::SLOTS;
      ok = ok && wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
      ok = ok && (i < 1 || wait_for(sfree, (i - 1) & 1, err, ERR_SFREE));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t kb = desc_lo(ring + slot * C::SLOT);
#pragma unroll
      for (int p = 0; p < C::QP; ++p)
#pragma unroll
        for (int k = 0; k < MT * 4; ++k)
          if (k < steps) mma_f8(tmem_s, qa + (p * MT + (k >> 2)) * 1024 + (k & 3) * 2, kb + (k >> 2) * 1024 + (k & 3) * 2, ids, p > 0 || k > 0);
      if (i > 0 || split != a.fault_split) tc_commit_elect(sfull);
      tc_commit_elect(empty + slot);
    };
    for (int i = 0; i < nt && ok; ++i) scores(i);
  } else if (w == 2) {  // a warp of its own: a product is issued in about 100 cycles beside the softmax, and takes 64 or 128
    const uint32_t idp = idesc_f8(a.dim, true, false);
    bool ok = true;
    for (int i = 0; i < nt; ++i) {
      const int pos = pos_v<2>(i, nt), slot = pos % C::SLOTS;
      ok = ok && wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
      ok = ok && wait_for(pfull, i & 1, err, ERR_P);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t vb = desc_lo(ring + slot * C::SLOT);
#pragma unroll
      for (int p = 0; p < C::PP; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_f8_ts(tmem_o, tmem_p + p * 32 + k * 8, vb + k * 2, idp, i > 0 || p > 0 || k > 0);
      tc_commit_elect(pvdone);
      tc_commit_elect(empty + slot);
    }
  } else if (w >= SOFT) {
    const int half = (w - SOFT) >> 2, quad = w & 3, row = quad * 32 + lane, st = tid - SOFT * 32;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const float rs = rowscale[row];
    const int lim = row < nrows ? a.mask.limit(n, nq, pre, token_of(a, row0 + row)) : 0;

    float next = 0.f;  // lanes 0..3: K scales of this half's four 16-key groups in the next tile, lanes 4..7: V scales
    auto scales = [&](int i) {
      const int key = (t0 + i) * TILE + half * 64 + 16 * (lane & 3);
      next = lane < 8 && i < nt && key < top ? __ldg((lane < 4 ? ks : vs) + (key >> a.block_log2)) : 0.f;
    };
    scales(0);
    // the subtracted maximum and the exponent of p vs (both the same in a row's two threads), this half's sum
    float m = -INFINITY, d = 0.f, l = 0.f;
    bool ok = true;
    // Raw scores s of a tile, factors f per 16-key group (the scale's sign went into the queries, so f >= 0 and a group's maximum
    // is f times that of its scores), log2 of the groups' V scales, and this half's maximum and the exponent above it (whole, so that it
    // goes through a byte) on their way to the row's other thread. Masked scores are -inf.
    float s[64], f[4], lv[4], mx, mv;
    auto fetch = [&](int i) {
      ok = wait_for(sfull, i & 1, err, ERR_S);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 64; c += 16) tmem_ld16(tmem_s + lanes + half * 64 + c, s + c);
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sfree);
      const float next_log = log2_approx(next);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = rs * __shfl_sync(0xffffffffu, next, j);
        lv[j] = __shfl_sync(0xffffffffu, next_log, 4 + j);
      }
      if ((t0 + i) * TILE + TILE > low) {  // not seen by every row
        const int left = lim - (t0 + i) * TILE - half * 64;
#pragma unroll
        for (int c = 0; c < 64; ++c) s[c] = c < left ? s[c] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = f[j] == 0.f ? 1e-30f : f[j];  // -inf stays -inf
      }
      scales(i + 1);
      mx = -INFINITY, mv = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float g = s[16 * j];
#pragma unroll
        for (int c = 1; c < 15; c += 2) g = max3(g, s[16 * j + c], s[16 * j + c + 1]);
        g = fmaxf(g, s[16 * j + 15]) * f[j];
        mx = fmaxf(mx, g);
        mv = fmaxf(mv, g + lv[j]);
      }
      const float up = mx == -INFINITY ? 0.f : fminf(fmaxf(ceilf(mv - mx - kSlack), -126.f), 126.f);
      mv = mx + up;
      half_max[(i & 1) * 2 * ROWS + half * ROWS + row] = mx;
      half_exp[(i & 1) * 2 * ROWS + half * ROWS + row] = (signed char)up;
      __syncwarp();
      if (lane == 0) mbar_arrive(seen);
    };
    fetch(0);
    for (int i = 0; i < nt && ok; ++i) {
      ok = wait_for(seen, i & 1, err, ERR_SEEN);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      {
        const int other = (i & 1) * 2 * ROWS + (half ^ 1) * ROWS + row;
        mv = fmaxf(mv, half_max[other] + (float)half_exp[other]);
        mx = fmaxf(mx, half_max[other]);
      }
      const bool grew = mx > m + kLag || mv > m + d + kLag || (m == -INFINITY && mx > m);
      if (__any_sync(0xffffffffu, grew)) {  // the same in the row's other thread's warp
        const float x = fmaxf(m, mx), by = x == -INFINITY ? 0.f : m - x;
        const float dn = x == -INFINITY ? 0.f : fmaxf(fmaxf(m + d, mv) - x, -110.f), down = exp2_approx(by + (d - dn));
        l *= exp2_approx(by);
        m = x, d = dn;
        if (i > 0) {  // O is at rest once the tile before is done
          ok = wait_for(pvdone, (i - 1) & 1, err, ERR_PV);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          for (int c = half * 16; c < a.dim; c += 32) {
            float v[16];
            uint32_t u[16];
            tmem_ld16(tmem_o + lanes + c, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(v[j] * down);
            tmem_st16(tmem_o + lanes + c, u);
          }
          tc_wait_st();
          tc_fence_before();
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      uint32_t e[C::PP][16];  // all of P before the wait for its place, which the product of the tile before still reads
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // p vs 2^(14 - d) straight from the exponent; the sum of p is that of a group over its factor. A factor below 2^-40 counts as
        // that: such a P is 0 in f16 either way.
        float v = lv[j] + (kPTop - d);
        v = v < -40.f ? -40.f : v;
        const float cc = v - base;
        float g0 = 0.f, g1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float* x = s + 16 * j + 4 * c;
          const float x0 = exp2_approx(fmaf(x[0], f[j], cc)), x1 = exp2_approx(fmaf(x[1], f[j], cc));
          const float x2 = exp2_approx(fmaf(x[2], f[j], cc)), x3 = exp2_approx(fmaf(x[3], f[j], cc));
          g0 += x0 + x1;
          g1 += x2 + x3;
          uint32_t p = pack_f16x2(x0, x1), q = pack_f16x2(x2, x3);
          if (HALF) e[C::PP - 1][4 * j + c] = __byte_perm(f16_lost(x0, x1, p, 1.f), f16_lost(x2, x3, q, 1.f), 0x5410);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const uint32_t pr = round_part(p), qr = round_part(q);
            e[k][4 * j + c] = __byte_perm(pr, qr, 0x7531);  // the upper bytes
            if (k < 2) p = rest1(p, pr), q = rest1(q, qr);
          }
        }
        l += (g0 + g1) * exp2_approx(-v);
      }
      if (i + 1 < nt) fetch(i + 1);
      if (!ok) break;
      if (i > 0) {
        ok = wait_for(pvdone, (i - 1) & 1, err, ERR_PV);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < C::PP; ++k) tmem_st16(tmem_p + lanes + k * 32 + half * 16, e[k]);
      const int left = top - (t0 + i) * TILE;
      if (left < TILE) {
        const int pos = pos_v<2>(i, nt), slot = pos % C::SLOTS;
        ok = wait_for(full + slot, (pos / C::SLOTS) & 1, err, ERR_FULL);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        clear_behind(ring + slot * C::SLOT, MT * 128, left, st, 256);
        fence_proxy_async_shared();
      }
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(pfull);
    }
    if (ok) ok = wait_for(pvdone, (nt - 1) & 1, err, ERR_PV);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) tc_wait_st();  // stores that a wait cut off from theirs
    tc_fence_after();
    float* sums = half_max + (nt & 1) * 2 * ROWS;  // the maxima's buffer that the last tile did not use
    sums[half * ROWS + row] = l;
    bar_softmax();
    l = sums[row] + sums[ROWS + row];
    if (half == 0) *reinterpret_cast<float2*>(osum + row * PITCH + MT * 128) = make_float2(m, l);
    const float norm = exp2_approx(d - kPTop);
#pragma unroll 1
    for (int c = half * 32; c < a.dim; c += 64) {
      float v[32];
      tmem_ld16(tmem_o + lanes + c, v);
      tmem_ld16(tmem_o + lanes + c + 16, v + 16);
      tc_wait_ld();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(osum + row * PITCH + c + 4 * j) =
            make_float4(v[4 * j] * norm, v[4 * j + 1] * norm, v[4 * j + 2] * norm, v[4 * j + 3] * norm);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (*err) give_up<C::SLOTS>(full, issued, drained, w == 1 || w == 2, osum, PITCH, MT * 128, osum + MT * 128, PITCH, ROWS);
  if (w == 1) tmem_dealloc(tmem_o, 512);
  finish_rows<HALF, MT, 4>(a, osum, PITCH, osum + MT * 128, PITCH, split, b, h, row0, nrows, n, nq, pre, first_part);
}

template <bool HALF, int MT>
fa_status launch(const AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  constexpr int SMEM = Cfg<HALF, MT>::SMEM;
  return kv8_launch<rows_kernel<HALF, MT>>(a, batch, THREADS, SMEM, km, vm, s);
}

template <bool HALF, int MT>
int resident(int device, int n) {
  return kv8_resident<rows_kernel<HALF, MT>>(device, n, THREADS, Cfg<HALF, MT>::SMEM);
}

}  // namespace

fa_status kv8_launch_rows(const AttnArgs& a, int batch, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  if (a.dim <= 128) return a.half ? launch<true, 1>(a, batch, km, vm, s) : launch<false, 1>(a, batch, km, vm, s);
  return a.half ? launch<true, 2>(a, batch, km, vm, s) : launch<false, 2>(a, batch, km, vm, s);
}

int kv8_resident_rows(bool half, int dim, int device, int n) {
  if (dim <= 128) return half ? resident<true, 1>(device, n) : resident<false, 1>(device, n);
  return half ? resident<true, 2>(device, n) : resident<false, 2>(device, n);
}
