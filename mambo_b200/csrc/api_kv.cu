// C ABI of rotary positions, the append to the paged FP8 key/value cache and
// attention over it (declared in include/mambo_b200.h).
#include "kernels.cuh"
#include "kv.cuh"

using namespace mambo;

namespace {

constexpr int kSmsBound = 160;  // workspace sizes do not depend on the device: an upper bound of its SMs
constexpr int64_t kMaxTokens = (int64_t)1 << 24, kMaxHeads = 1024, kMaxBatch = 4096, kMaxPages = (int64_t)1 << 31;

bool dtype_ok(int d) { return d == MAMBO_F32 || d == MAMBO_BF16; }
bool aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }
constexpr const char* kUnaligned = "a pointer is not aligned to its elements";

int check_rotary(const MamboRotary* r, int64_t dim) {
  if (!r->turns) return api_fail(MAMBO_EINVAL, "null pointer");
  if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > dim)
    return api_fail(MAMBO_EINVAL, "the rotated part must be an even number of dimensions of the head");
  if (!aligned(r->turns, 8)) return api_fail(MAMBO_EINVAL, kUnaligned);
  return MAMBO_OK;
}

RotaryParams rotary_params(const MamboRotary* r, int inverse) {
  RotaryParams p{};
  if (r) p = {r->turns, r->rotary_dim / 2, r->interleaved != 0, r->magnitude, inverse ? -1.f : 1.f};
  return p;
}

int check_cache(const MamboKvCache* c) {
  if (!c || !c->keys || !c->values || !c->key_scales || !c->value_scales) return api_fail(MAMBO_EINVAL, "null cache field");
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return api_fail(MAMBO_EINVAL, "a page has 16, 32, 64 or 128 tokens");
  if (c->head_dim < 16 || c->head_dim % 16 || c->head_dim > kKvMaxDim)
    return api_fail(MAMBO_EINVAL, "the head size must be a multiple of 16, at most %d", kKvMaxDim);
  if (c->kv_heads < 1 || c->kv_heads > kMaxHeads) return api_fail(MAMBO_EINVAL, "1 to %d heads", (int)kMaxHeads);
  if (c->pages < 1 || c->pages > kMaxPages / c->kv_heads) return api_fail(MAMBO_EINVAL, "pages * heads must be in [1, 2^31]");
  if (!aligned(c->keys, 16) || !aligned(c->values, 16)) return api_fail(MAMBO_EINVAL, "the cache must be 16-byte aligned");
  return MAMBO_OK;
}

KvCache cache_params(const MamboKvCache* c) {
  KvCache p{};
  p.codes[0] = c->keys;
  p.codes[1] = c->values;
  p.scales[0] = c->key_scales;
  p.scales[1] = c->value_scales;
  p.pages = c->pages;
  p.heads = c->kv_heads;
  p.page = c->page_tokens;
  p.dim = c->head_dim;
  p.log_page = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
  return p;
}

int check_sequences(const MamboKvSequences* s, int64_t tokens) {
  if (!s || !s->page_table || !s->lengths) return api_fail(MAMBO_EINVAL, "null pointer");
  if (s->batch < 1 || s->batch > kMaxBatch) return api_fail(MAMBO_EINVAL, "1 to 4096 sequences");
  if (s->table_pages < 1 || s->table_pages > (1 << 24)) return api_fail(MAMBO_EINVAL, "the page table has 1 to 2^24 columns");
  if (s->table_stride < s->table_pages && s->batch > 1) return api_fail(MAMBO_EINVAL, "page table row stride smaller than the row");
  if (tokens < 1 || tokens > kMaxTokens) return api_fail(MAMBO_EINVAL, "1 to 2^24 tokens");
  if (!s->offsets && tokens != s->batch) return api_fail(MAMBO_EINVAL, "without offsets a sequence has one token");
  if (!aligned(s->page_table, 4) || !aligned(s->lengths, 4) || !aligned(s->offsets, 4)) return api_fail(MAMBO_EINVAL, kUnaligned);
  return MAMBO_OK;
}

KvSequences sequence_params(const MamboKvSequences* s, int64_t tokens) {
  return {s->page_table, s->table_stride, (int)s->table_pages, s->lengths, s->offsets, (int)s->batch, (int)tokens};
}

// Rows of a sequence (tokens times query heads of a key head) that the decode kernel takes at most: it has forms for 16
// and for 32 rows, and where the heads alone are more, none. Single tokens of 64 sequences, in the decode kernel, in the
// prompt kernel and as the cache's bytes would take them, us: 4096 to 8191 positions, 8 key heads of 16 rows 137, 275 and
// 123, 2 key heads of 20 rows 75, 87 and 31; 400 to 900 positions, 8 key heads of 16 rows 49, 82 and 13, 2 key heads of 20
// rows 32, 37 and 3.
int few_rows(int group) { return group <= 16 ? 16 : group <= 32 ? 32 : 0; }
size_t decode_bytes(int group) { return few_rows(group) ? (kv_decode_partial_bytes(group, kSmsBound) + 255) / 256 * 256 : 0; }
constexpr int kPromptCounters = 4096;  // of the split counters: the prompt kernel's, behind the decode kernel's

}  // namespace

extern "C" {

int mambo_rotary(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t stride_token,
                 int64_t stride_head, const void* positions, int positions_64, const MamboRotary* rotary, int inverse,
                 void* out, int64_t out_stride_token, int64_t out_stride_head, mambo_stream_t stream) {
  if (!x || !out || !positions || !rotary) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!dtype_ok(dtype)) return api_fail(MAMBO_EINVAL, "x must be f32 or bf16");
  if (tokens < 1 || tokens > kMaxTokens || heads < 1 || heads > kMaxHeads || dim < 2 || dim > 65536)
    return api_fail(MAMBO_EINVAL, "x must be [1..2^24 tokens, 1..1024 heads, 2..65536]");
  const int es = dtype == MAMBO_BF16 ? 2 : 4;
  if (!aligned(x, es) || !aligned(out, es) || !aligned(positions, positions_64 ? 8 : 4)) return api_fail(MAMBO_EINVAL, kUnaligned);
  int st = check_rotary(rotary, dim);
  if (st != MAMBO_OK) return st;
  if ((double)tokens * (double)heads * (double)(dim / 16 + 2) >= 2147483647.0 * 128)
    return api_fail(MAMBO_EINVAL, "the call is too large: split its tokens");
  int sms, smem;
  st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  RotaryCall p{};
  p.rot = rotary_params(rotary, inverse);
  p.x = x;
  p.out = out;
  p.bf16 = dtype == MAMBO_BF16;
  p.tokens = (int)tokens;
  p.heads = (int)heads;
  p.dim = (int)dim;
  p.xs_t = stride_token;
  p.xs_h = stride_head;
  p.os_t = out_stride_token;
  p.os_h = out_stride_head;
  p.positions = positions;
  p.positions64 = positions_64 != 0;
  const cudaError_t e = launch_rotary(p, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "rotary positions");
  return api_ok();
}

int mambo_kv_append(const MamboKvCache* cache, const void* k, int64_t k_stride_token, int64_t k_stride_head, const void* v,
                    int64_t v_stride_token, int64_t v_stride_head, int dtype, int64_t tokens, const MamboKvSequences* seq,
                    const MamboRotary* rotary, mambo_stream_t stream) {
  int st = check_cache(cache);
  if (st == MAMBO_OK) st = check_sequences(seq, tokens);
  if (st != MAMBO_OK) return st;
  if (!k || !v) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!dtype_ok(dtype)) return api_fail(MAMBO_EINVAL, "k and v must be f32 or bf16");
  if (rotary) st = check_rotary(rotary, cache->head_dim);
  if (st != MAMBO_OK) return st;
  const int es = dtype == MAMBO_BF16 ? 2 : 4;
  if (!aligned(k, es) || !aligned(v, es)) return api_fail(MAMBO_EINVAL, kUnaligned);
  int sms, smem;
  st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  KvAppendCall p{};
  p.rot = rotary_params(rotary, 0);
  p.cache = cache_params(cache);
  p.seq = sequence_params(seq, tokens);
  p.x[0] = k;
  p.x[1] = v;
  p.xs_t[0] = k_stride_token;
  p.xs_t[1] = v_stride_token;
  p.xs_h[0] = k_stride_head;
  p.xs_h[1] = v_stride_head;
  p.bf16 = dtype == MAMBO_BF16;
  const cudaError_t e = launch_kv_append(p, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "key/value append");
  return api_ok();
}

size_t mambo_kv_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int ragged) {
  if (kv_heads < 1 || kv_heads > kMaxHeads || heads < 1 || heads > kMaxHeads || heads % kv_heads) return 0;
  const int group = (int)(heads / kv_heads);
  return kWorkspaceCounterBytes + decode_bytes(group) + (ragged || !few_rows(group) ? kv_prompt_partial_bytes(kSmsBound) : 0);
}

int mambo_kv_attention(const void* q, int64_t q_stride_token, int64_t q_stride_head, int64_t tokens, int64_t heads,
                       const MamboKvCache* cache, const MamboKvSequences* seq, int64_t window, float scale, void* out,
                       int64_t out_stride_token, int64_t out_stride_head, float* lse, int64_t lse_stride_token,
                       int64_t lse_stride_head, void* workspace, size_t workspace_bytes, mambo_stream_t stream) {
  int st = check_cache(cache);
  if (st == MAMBO_OK) st = check_sequences(seq, tokens);
  if (st != MAMBO_OK) return st;
  if (!q || !out) return api_fail(MAMBO_EINVAL, "null pointer");
  if (heads < 1 || heads > kMaxHeads || heads % cache->kv_heads)
    return api_fail(MAMBO_EINVAL, "query heads must be a multiple of the cache's heads, at most %d", (int)kMaxHeads);
  if (window < 0) return api_fail(MAMBO_EINVAL, "the window must not be negative");
  if (!aligned(lse, 4)) return api_fail(MAMBO_EINVAL, kUnaligned);
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride_token % 8 || q_stride_head % 8 || out_stride_token % 8 || out_stride_head % 8)
    return api_fail(MAMBO_EINVAL, "the heads of q and out must be 16-byte aligned");
  // Rows, and tiles of 128 positions over all sequences, heads and units of rows (which count as six more), are counted in
  // 32 bits.
  const int64_t group = heads / cache->kv_heads;
  const double units = (double)tokens * group / 256 + (double)seq->batch;
  if (tokens * group > (1 << 30) ||
      units * cache->kv_heads * ((double)seq->table_pages * cache->page_tokens / 128 + 8) >= 2147483647.0)
    return api_fail(MAMBO_EINVAL, "the call is too large: split its sequences");
  if (!(scale > 0.f) || !(scale <= 3.4028234663852886e38f)) return api_fail(MAMBO_EINVAL, "the scale must be a positive number");
  const bool prompt = seq->offsets || !few_rows((int)group);
  const size_t need = mambo_kv_attention_workspace_bytes(heads, cache->kv_heads, seq->offsets != nullptr);
  if (!workspace || workspace_bytes < need)
    return api_fail(MAMBO_EWORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  if (!aligned(workspace, 256)) return api_fail(MAMBO_EINVAL, "workspace must be 256-byte aligned");
  int sms, smem;
  st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  KvAttentionCall p{};
  p.cache = cache_params(cache);
  p.seq = sequence_params(seq, tokens);
  p.q = (const uint16_t*)q;
  p.qs_t = q_stride_token;
  p.qs_h = q_stride_head;
  p.out = (uint16_t*)out;
  p.os_t = out_stride_token;
  p.os_h = out_stride_head;
  p.lse = lse;
  p.ls_t = lse_stride_token;
  p.ls_h = lse_stride_head;
  p.group = (int)(heads / cache->kv_heads);
  p.window = window <= 0x7FFFFFFF ? (int)window : 0;
  p.scale = scale;
  p.few = few_rows(p.group);
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i)
    if (!kv_page_map(p.cache, i, &maps[i])) return api_fail(MAMBO_EINVAL, "the cache has no tensor map");
  if (sms > kSmsBound) sms = kSmsBound;
  uint8_t* parts = (uint8_t*)workspace + kWorkspaceCounterBytes;
  int* counters = (int*)((uint8_t*)workspace + kWorkspaceSplitCounterOffset);
  cudaError_t e = cudaSuccess;
  if (p.few) e = launch_kv_decode(p, maps[0], maps[1], sms, smem, (float*)parts, counters, (cudaStream_t)stream);
  if (e == cudaSuccess && prompt)
    e = launch_kv_prompt(p, maps[0], maps[1], sms, (float*)(parts + decode_bytes(p.group)), counters + kPromptCounters,
                         (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "attention");
  return api_ok();
}

}  // extern "C"
