// fa_kv8_attention: checks, the split of the key axis, and the choice of kernel.
#include "kv8_attn.cuh"

namespace {

using namespace fa::kv8;

struct Plan {
  int tiles, nsplit, split_chunks;
  size_t part_bytes, ml_bytes;
};

// Few query rows (kv8_attn_few.cu): 16 rows a tile, CTAs of four warps that take 64-key chunks in turn, two CTAs
// on an SM. The split count is the one with the least rounds of chunks on the busiest SM slot, each wave
// of CTAs paying about two rounds for its start and a merge about three.
Plan plan_few(const fa_kv8* c, int tokens, int q_heads, int max_len, int sms) {
  Plan p;
  const int rows = 16, warps = 4, slots = 2 * sms;
  p.tiles = (int)(((long long)tokens * (q_heads / c->heads) + rows - 1) / rows);
  const int chunks = std::max(1, (max_len + 63) / 64);
  const long long base = (long long)c->batch * c->heads * p.tiles;
  double best = 1e300;
  p.nsplit = 1;
  for (int n = 1; n <= 64 && n <= (chunks + warps - 1) / warps; ++n) {
    const int each = (chunks + n - 1) / n, rounds = (each + warps - 1) / warps;
    const double waves = (double)((base * n + slots - 1) / slots);
    const double cost = waves * (rounds + 2) + (n > 1 ? 3 + 0.05 * n : 0);
    if (cost < best) best = cost, p.nsplit = n;
  }
  p.split_chunks = (chunks + p.nsplit - 1) / p.nsplit;
  p.nsplit = (chunks + p.split_chunks - 1) / p.split_chunks;
  const size_t slot = p.nsplit > 1 ? (size_t)base * p.nsplit * rows : 0;
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

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    n = 148;
  }
  return n;
}

}  // namespace

extern "C" fa_status fa_kv8_attention_workspace(const fa_kv8* c, int tokens, int q_heads, int max_len, size_t* bytes) {
  fa_status st = attn_check(c, tokens, q_heads, max_len);
  if (st != FA_OK) return st;
  if (!bytes) return fail(nullptr, FA_ERR_INVALID, "null bytes");
  const Plan p = plan_few(c, std::max(1, tokens), q_heads, max_len ? max_len : c->capacity, sm_count());
  *bytes = p.part_bytes + p.ml_bytes;
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
  if (!(std::fabs(scale) <= 3.0e38f)) return fail(nullptr, FA_ERR_INVALID, "the scale is not a finite number");
  if (prefix && !causal) return fail(nullptr, FA_ERR_INVALID, "a prefix belongs to a causal mask");
  if (reinterpret_cast<uintptr_t>(q->ptr) % 2 || reinterpret_cast<uintptr_t>(out->ptr) % 2)
    return fail(nullptr, FA_ERR_INVALID, "queries and output must be aligned to their type");
  if (tokens == 0) return FA_OK;
  const int top = max_len ? max_len : c->capacity;
  const Plan p = plan_few(c, tokens, q_heads, top, sm_count());
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
  a.k = c->k, a.v = c->v, a.ks = c->k_scale, a.vs = c->v_scale;
  a.q = q->ptr, a.out = out->ptr;
  a.qb = q->batch, a.qt = q->token, a.qh = q->head;
  a.ob = out->batch, a.ot = out->token, a.oh = out->head;
  a.mask = Mask{lens, q_lens, prefix, causal != 0, tokens, top};
  a.layers = c->layers, a.layer = layer, a.heads = c->heads, a.group = q_heads / c->heads, a.cap = c->capacity;
  a.block = c->block, a.half = dtype == FA_DT_F16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.nsplit = p.nsplit, a.split_chunks = p.split_chunks, a.tiles = p.tiles;
  a.part = reinterpret_cast<float*>(workspace);
  a.ml = reinterpret_cast<float2*>(reinterpret_cast<char*>(workspace) + p.part_bytes);
  return kv8_launch_few(a, c->head_dim, c->batch, reinterpret_cast<cudaStream_t>(stream));
}
