// fa_kv8_attention: checks, the split of the key axis, the choice of kernel, and the merge of the splits.
#include "kv8_tc.cuh"

namespace {

using namespace fa::kv8;

struct Plan {
  int rows, tiles, nsplit, cluster, split_chunks;
  size_t part_bytes, ml_bytes;
};

// One warp per query row: o = sum_s 2^(m_s - m) part_s / sum_s 2^(m_s - m) l_s over the splits that the
// row's tile has, in split order (the result does not depend on which split ended first).
template <int D>
__global__ void merge_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, b = blockIdx.z, R = a.rows;
  const int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  wait_for_primary();
  const int n = a.mask.len(b), nq = a.mask.q_len(b), pre = a.mask.prefix ? a.mask.prefix[b] : 0;
  if (row >= nq * a.group) return;
  const int tile = row / R, r = row % R, last = min(tile * R + R, nq * a.group) - 1;
  const int top = a.mask.limit(n, nq, pre, token_of(a, last)), lim = a.mask.limit(n, nq, pre, token_of(a, row));
  const int chunks = (top + TILE - 1) / TILE;
  const int used = max(1, (chunks + a.split_chunks - 1) / a.split_chunks);
  const size_t slot = (((size_t)b * a.heads + h) * a.tiles + tile) * a.nsplit;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < used; s += 32) m = fmaxf(m, a.ml[(slot + s) * R + r].x);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  float acc[D / 32] = {};
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const float2 x = a.ml[(slot + s) * R + r];
    const float f = exp2_approx(x.x - base);
    l += x.y * f;
    const float* p = a.part + ((slot + s) * R + r) * D + lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] += f * p[i * 32];
  }
  const float norm = 1.0f / l;
  const long long oo = row_at(a, b, h, row, a.ob, a.ot, a.oh) + lane;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store16(a.out, oo + i * 32, lim > 0 ? acc[i] * norm : 0.f, a.half);
}

// 3D byte map [outer][rows][inner] with boxes {128, box_rows, 1}, 128-byte swizzle; what lies outside reads as zero.
fa_status byte_map(CUtensorMap* m, const void* base, uint64_t inner, uint64_t rows, uint64_t outer, uint32_t box_rows) {
  auto enc = get_encode();
  if (!enc) return fail(nullptr, FA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {inner, rows, outer};
  cuuint64_t strides[2] = {inner, inner * rows};
  cuuint32_t box[3] = {128, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(nullptr, FA_ERR_CUDA, "cuTensorMapEncodeTiled (cache) failed (%d)", (int)r);
  return FA_OK;
}

// The kernel and the splits of whole 128-key tiles: the number of splits with the least time by a model of measured parts (B200, us).
// Waves come from what the device has room for, in blocks or in whole clusters of the split's size (a cluster of 8 blocks that fill an SM
// leaves many SMs idle). A wave costs its start and end and its tiles. Up to 16 rows: 6 or 7 (16 rows), a tile 1.05 or 1.2 (a chain of
// latencies, whatever head_dim); where many are read at once their bytes at the memory's rate are the longer part (lengths are mostly below max_len,
// hence 0.85), and a quarter of the shorter one is not hidden. 128 rows: 12, a tile 1.7 at head_dim 64 to 2.6 at 256. fp16 has 1.1 and 1.35
// times that a tile. Then the join: in a cluster 1 to 2.4, with 128 rows, whose sums are many, 2 to 5; by the merge kernel, where a warp reads its row's
// sums split by split, 2 and 0.29 to 0.4 a split, with 128 rows 0.8 to 3 and 0.16 to 0.36 a split.
// Over 86 shapes (1 to 100 observations, 1 to 968 tokens, 156 to 32768 keys, head_dim 64 to 256, both types) the planned number is within 10% of
// the best of 18 tried, in 79 of them within 3%.
Plan make_plan(const fa_kv8* c, int tokens, int q_heads, int max_len, int device, bool half) {
  Plan p;
  const long long all = (long long)tokens * (q_heads / c->heads);
  p.rows = all <= 8 ? 8 : all <= 16 ? 16 : 128;
  p.tiles = (int)((all + p.rows - 1) / p.rows);
  const bool few = p.rows < 128;
  const int chunks = std::max(1, (max_len + 127) / 128);
  const long long base = (long long)c->batch * c->heads * p.tiles;
  const double mb = 256e-6 * c->head_dim;  // a tile's bytes, in MB
  const double fix = few ? (p.rows == 8 ? 6 : 7) : 12;
  const double lat = few ? (p.rows == 8 ? 1.05 : 1.2) * (half ? 1.1 : 1) : (1.4 + 0.0047 * c->head_dim) * (half ? 1.35 : 1);
  const auto resident = [&](int n) {
    const int got = device < 0 ? 0 : few ? kv8_resident_few(p.rows, half, c->head_dim, device, n) : kv8_resident_rows(half, c->head_dim, device, n);
    return got > 0 ? got : std::max(1, (few && c->head_dim <= 128 ? 2 : 1) * 148 / n);
  };
  int fit[9];
  for (int n = 1; n <= 8 && n <= chunks; ++n) fit[n] = resident(n);
  double best = 1e300;
  p.nsplit = 1;
  for (int n = 1; n <= 64 && n <= chunks; ++n) {
    const int each = (chunks + n - 1) / n;
    const bool cluster = n <= 8;
    const double groups = cluster ? (double)base : (double)base * n, room = fit[cluster ? n : 1];
    const double active = std::min(groups, room) * (cluster ? n : 1);
    const double chain = each * lat, bytes = few ? active * chunks / n * mb * (0.85 / 6.5) : 0;
    const double d = c->head_dim;
    const double join = n > 8 ? (few ? 2 + n * (0.25 + d / 1700) : 3 * d / 256 + n * (0.1 + d / 1000)) : few ? (n > 1 ? 0.8 + 0.2 * n : 0) : 1 + d / 64;
    const double cost = std::ceil(groups / room) * (fix + std::max(chain, bytes) + 0.25 * std::min(chain, bytes)) + join;
    if (cost < best) best = cost, p.nsplit = n;
  }
  p.split_chunks = (chunks + p.nsplit - 1) / p.nsplit;
  p.nsplit = (chunks + p.split_chunks - 1) / p.split_chunks;
  p.cluster = p.nsplit > 1 && p.nsplit <= 8;
  const size_t slot = p.nsplit > 1 && !p.cluster ? (size_t)base * p.nsplit * p.rows : 0;
  p.part_bytes = slot * c->head_dim * sizeof(float);
  p.ml_bytes = slot * sizeof(float2);
  return p;
}

fa_status attn_check(const fa_kv8* c, int tokens, int q_heads, int max_len) {
  fa_status st = kv8_check(c);
  if (st != FA_OK) return st;
  if (tokens < 0) return fail(nullptr, FA_ERR_INVALID, "tokens=%d", tokens);
  if (q_heads < 1 || q_heads % c->heads) return fail(nullptr, FA_ERR_INVALID, "q_heads=%d is not a multiple of heads=%d", q_heads, c->heads);
  if ((long long)tokens * (q_heads / c->heads) > (1 << 24))
    return fail(nullptr, FA_ERR_INVALID, "tokens=%d with %d query heads a key head is over 2^24 rows", tokens, q_heads / c->heads);
  if (max_len < 0 || max_len > c->capacity) return fail(nullptr, FA_ERR_INVALID, "max_len=%d of capacity %d", max_len, c->capacity);
  return FA_OK;
}

std::atomic<int> fault_split{-1};
std::atomic<unsigned> spin_limit{0};

// The current device; -1 where there is none, so that a workspace can be asked for anywhere.
int current_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return dev;
}

}  // namespace

extern "C" void fa_kv8_set_fault_injection(int split, unsigned limit) {
  fault_split.store(split, std::memory_order_relaxed);
  spin_limit.store(limit, std::memory_order_relaxed);
}

extern "C" fa_status fa_kv8_attention_workspace(const fa_kv8* c, int tokens, int q_heads, int max_len, size_t* bytes) {
  fa_status st = attn_check(c, tokens, q_heads, max_len);
  if (st != FA_OK) return st;
  if (!bytes) return fail(nullptr, FA_ERR_INVALID, "null bytes");
  *bytes = 0;
  for (const bool half : {false, true}) {  // for queries of either type
    const Plan p = make_plan(c, std::max(1, tokens), q_heads, max_len ? max_len : c->capacity, current_device(), half);
    *bytes = std::max(*bytes, p.part_bytes + p.ml_bytes);
  }
  return FA_OK;
}

extern "C" fa_status fa_kv8_attention(const fa_kv8* c, int layer, int tokens, int q_heads, const fa_rows* q, fa_dtype dtype,
                                      const int* lens, const int* q_lens, const int* prefix, int causal, float scale,
                                      int max_len, const fa_rows* out, void* workspace, size_t workspace_bytes,
                                      fa_stream stream) {
  fa_status st = attn_check(c, tokens, q_heads, max_len);
  if (st != FA_OK) return st;
  if (layer < 0 || layer >= c->layers) return fail(nullptr, FA_ERR_INVALID, "layer %d of %d", layer, c->layers);
  if (dtype != FA_DT_BF16 && dtype != FA_DT_F16)
    return fail(nullptr, FA_ERR_UNSUPPORTED, "queries are bf16 or fp16 (dtype %d)", (int)dtype);
  if (!q || !out) return fail(nullptr, FA_ERR_INVALID, "null queries or output");
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!std::isfinite(scale_log2)) return fail(nullptr, FA_ERR_INVALID, "the scale is not a finite number, or its product with log2 e is none");
  if (prefix && !causal) return fail(nullptr, FA_ERR_INVALID, "a prefix belongs to a causal mask");
  if (reinterpret_cast<uintptr_t>(q->ptr) % 2 || reinterpret_cast<uintptr_t>(out->ptr) % 2)
    return fail(nullptr, FA_ERR_INVALID, "queries and output must be aligned to their type");
  if ((c->batch > 1 && !out->batch) || (tokens > 1 && !out->token) || (q_heads > 1 && !out->head))
    return fail(nullptr, FA_ERR_INVALID, "rows of the output lie on one another (a stride of 0)");
  if (tokens == 0) return FA_OK;
  const int top = max_len ? max_len : c->capacity;
  const int device = current_device();
  const Plan p = make_plan(c, tokens, q_heads, top, device, dtype == FA_DT_F16);
  if (workspace_bytes < p.part_bytes + p.ml_bytes)
    return fail(nullptr, FA_ERR_INVALID, "workspace of %zu bytes, %zu are needed", workspace_bytes, p.part_bytes + p.ml_bytes);
  if (p.part_bytes && reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(nullptr, FA_ERR_INVALID, "the workspace must be 16-byte aligned");
  if ((st = kv8_check_pointers(c)) != FA_OK) return st;
  if ((st = check_pointers({{"q", q->ptr}, {"out", out->ptr}, {"lens", lens}})) != FA_OK) return st;
  if (q_lens && (st = check_pointers({{"q_lens", q_lens}})) != FA_OK) return st;
  if (prefix && (st = check_pointers({{"prefix", prefix}})) != FA_OK) return st;
  if (p.part_bytes && (st = check_pointers({{"workspace", workspace}})) != FA_OK) return st;
  AttnArgs a;
  a.device = device;
  const unsigned limit = spin_limit.load(std::memory_order_relaxed);
  a.fault_split = fault_split.load(std::memory_order_relaxed);
  a.spin_limit = limit ? (int)std::min(limit, fa::kSpinLimit) : (int)fa::kSpinLimit;
  a.ks = c->k_scale, a.vs = c->v_scale;
  a.q = q->ptr, a.out = out->ptr;
  a.qb = q->batch, a.qt = q->token, a.qh = q->head;
  a.ob = out->batch, a.ot = out->token, a.oh = out->head;
  a.mask = Mask{lens, q_lens, prefix, causal != 0, tokens, top};
  a.layers = c->layers, a.layer = layer, a.heads = c->heads, a.group = q_heads / c->heads, a.dim = c->head_dim;
  a.blocks = c->capacity / c->block, a.block_log2 = __builtin_ctz(c->block), a.half = dtype == FA_DT_F16;
  a.q_wide = reinterpret_cast<uintptr_t>(q->ptr) % 16 == 0 && q->batch % 8 == 0 && q->token % 8 == 0 && q->head % 8 == 0;
  a.o_wide = reinterpret_cast<uintptr_t>(out->ptr) % 8 == 0 && out->batch % 4 == 0 && out->token % 4 == 0 && out->head % 4 == 0;
  a.scale_log2 = scale_log2;
  a.group_mul = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
  a.nsplit = p.nsplit, a.cluster = p.cluster, a.split_chunks = p.split_chunks, a.rows = p.rows, a.tiles = p.tiles;
  a.part = reinterpret_cast<float*>(workspace);
  a.ml = reinterpret_cast<float2*>(reinterpret_cast<char*>(workspace) + p.part_bytes);
  CUtensorMap km, vm;
  const uint64_t outer = (uint64_t)c->batch * c->layers * c->heads;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if ((st = byte_map(&km, c->k, c->head_dim, c->capacity, outer, TILE)) != FA_OK) return st;
  if ((st = byte_map(&vm, c->v, c->capacity, c->head_dim, outer, c->head_dim <= 128 ? 128 : 256)) != FA_OK) return st;
  st = p.rows == 128 ? kv8_launch_rows(a, c->batch, km, vm, s) : kv8_launch_few(a, c->batch, km, vm, s);
  if (st != FA_OK || p.nsplit == 1 || p.cluster) return st;
  // The merge is set up while the attention runs (programmatic dependent launch): its own launch costs nothing then.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((tokens * a.group + 3) / 4, c->heads, c->batch);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  switch (c->head_dim) {
    case 64: FA_CUDA(nullptr, cudaLaunchKernelEx(&cfg, merge_kernel<64>, a)); break;
    case 96: FA_CUDA(nullptr, cudaLaunchKernelEx(&cfg, merge_kernel<96>, a)); break;
    case 128: FA_CUDA(nullptr, cudaLaunchKernelEx(&cfg, merge_kernel<128>, a)); break;
    default: FA_CUDA(nullptr, cudaLaunchKernelEx(&cfg, merge_kernel<256>, a)); break;
  }
  return FA_OK;
}
