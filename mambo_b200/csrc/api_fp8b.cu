// C ABI of the FP8 block-scaled linear, its expert-grouped form, the expert
// router and the experts' path (declared in include/mambo_b200.h).
#include "fp8b.cuh"
#include "kernels.cuh"

using namespace mambo;

namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 28;   // rows of a call (32-bit row arithmetic with padding)
constexpr int64_t kMaxExtent = (int64_t)1 << 24; // N and K

bool extent_ok(int64_t v) { return v >= 1 && v <= kMaxExtent; }
bool experts_ok(int64_t v) { return v >= 1 && v <= kFbMaxExperts; }
// tokens * top choices, without forming a product that may not fit.
bool choices_ok(int64_t tokens, int64_t top) { return tokens >= 1 && top >= 1 && tokens <= kMaxRows / top; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }
bool dtype_ok(int d) { return d == MAMBO_F32 || d == MAMBO_BF16; }
int elem(int d) { return d == MAMBO_BF16 ? 2 : 4; }

// Pointers are read and written element by element at least: one off its elements' alignment would fault.
bool aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }
constexpr const char* kUnaligned = "a pointer is not aligned to its elements";

int check_weight(const MamboFp8BlockWeight* w) {
  if (!w || !w->packed || !w->scales) return api_fail(MAMBO_EINVAL, "null weight field");
  if ((uintptr_t)w->packed % 16 || (uintptr_t)w->scales % 4)
    return api_fail(MAMBO_EINVAL, "packed weight must be 16-byte aligned, its scales 4-byte");
  if (!extent_ok(w->n_rows) || !extent_ok(w->k))
    return api_fail(MAMBO_EINVAL, "weight must have N and K in [1, 2^24]");
  if (!experts_ok(w->n_experts))
    return api_fail(MAMBO_EINVAL, "a weight has 1 to %d experts", kFbMaxExperts);
  if (w->gate_up && w->n_rows % 2) return api_fail(MAMBO_EINVAL, "a gate/up weight has an even number of rows");
  return MAMBO_OK;
}

// One product's activations and partial sums in the workspace.
struct Plan {
  int nt, kblocks, row_tiles;
  int64_t slots;
  size_t x8;  // bytes
};
Plan plan(int64_t rows, int64_t experts, int64_t bound, int64_t n, int64_t k, int gate_up) {
  Plan P;
  // Tokens of a tile: what an expert may be expected to get (twice the even
  // share, never more than `bound`), so that a decode call does not load or
  // multiply empty columns and a long segment fills its tiles.
  const int64_t share = 2 * ((rows + experts - 1) / experts);
  P.nt = fb_tile_for(experts == 1 ? rows : share < bound ? share : bound);
  P.kblocks = (int)((k + 127) / 128);
  P.row_tiles = fb_row_tiles(n, gate_up);
  P.slots = fb_slots(rows, experts, P.nt);
  P.x8 = align256((size_t)P.slots * P.kblocks * fb_record_bytes(P.nt));
  return P;
}
FbActivations activations(const Plan& P, uint8_t* at) {
  return FbActivations{at, P.slots, P.kblocks, P.nt};
}

constexpr int kSmsBound = 160;  // workspace sizes do not depend on the device: an upper bound of its SMs

size_t product_bytes(const Plan& P) { return P.x8 + align256(fb_partial_bytes(P.nt, kSmsBound)); }

int check_workspace(void* ws, size_t have, size_t need) {
  if (!ws || have < need) return api_fail(MAMBO_EWORKSPACE, "workspace of %zu bytes needed, %zu given", need, have);
  if ((uintptr_t)ws % 256) return api_fail(MAMBO_EINVAL, "workspace must be 256-byte aligned");
  return MAMBO_OK;
}

FbSource source(const void* x, int x_dtype, int64_t ldx, int64_t rows, int64_t k, int group) {
  FbSource s{};
  s.x = x;
  s.bf16 = x_dtype == MAMBO_BF16;
  s.vec = (uintptr_t)x % 16 == 0 && ldx * elem(x_dtype) % 16 == 0;
  s.ldx = ldx;
  s.k = k;
  s.group = group;
  s.top = 1;
  s.last = (int)(rows - 1);
  return s;
}

// Tiles times K blocks are counted in 32 bits, and the quantizer's spans too.
int check_size(const Plan& P, int64_t rows, int64_t experts, int64_t k) {
  const double tiles = (double)(rows / P.nt + experts) * P.row_tiles;
  if (tiles * P.kblocks >= 2147483647.0 || (double)rows * (double)((k + 1023) / 1024) >= 2147483647.0)
    return api_fail(MAMBO_EINVAL, "the call is too large: split its rows");
  return MAMBO_OK;
}

// src: activations that the product quantizes itself, else act holds them.
cudaError_t run_gemm(const MamboFp8BlockWeight* w, const Plan& P, const FbSource* src, const FbActivations& act, int64_t rows,
                     const int* offsets, void* out, int out_bf16, int64_t ldo, const FbActivations* hidden, uint8_t* partials,
                     void* workspace, int sms, int smem_optin, cudaStream_t stream) {
  FbGemmParams g{};
  if (src) g.src = *src;
  g.packed = (const uint8_t*)w->packed;
  g.scales = w->scales;
  g.act = act;
  g.experts = offsets ? (int)w->n_experts : 1;
  g.rows = rows;
  g.offsets = offsets;
  g.n_rows = (int)w->n_rows;
  g.row_tiles = P.row_tiles;
  g.out = out;
  g.out_bf16 = out_bf16;
  g.ldo = ldo;
  if (hidden) g.hidden = *hidden;
  g.stages = fb_gemm_stages(P.nt, g.experts, smem_optin, hidden != nullptr);
  // Weights are read once where a call has one token tile, or as a rule an expert has (its tile holds twice the even share):
  // evict-first keeps the rest in the L2. 64 experts of 4096 x 4096 at 16 rows each 166 us with it, 174 without, of 1024 x
  // 2048 33.1 and 35.6. With all 1024 rows in one expert its weights are read by 32 tiles, 64-65 us and 19.6 either way.
  g.evict_weights = offsets ? !fb_is_pair(P.nt) : rows <= P.nt;
  g.partials = (float*)partials;
  g.counters = (int*)((uint8_t*)workspace + kWorkspaceSplitCounterOffset);
  return launch_fb_gemm(g, fb_gemm_grid(P.nt, sms < kSmsBound ? sms : kSmsBound), stream);
}

int check_linear(const void* x, int64_t m, int group, const MamboFp8BlockWeight* w, const void* out, int out_dtype,
                 int64_t ldo) {
  if (!x || !out) return api_fail(MAMBO_EINVAL, "null pointer");
  const int st = check_weight(w);
  if (st != MAMBO_OK) return st;
  if (w->gate_up) return api_fail(MAMBO_EINVAL, "a gate/up weight is for mambo_moe_experts only");
  if (m < 1 || m > kMaxRows) return api_fail(MAMBO_EINVAL, "activation must have 1 to 2^28 rows");
  if (group != 32 && group != 128) return api_fail(MAMBO_EINVAL, "activation scales are per 32 or per 128 values");
  if (!dtype_ok(out_dtype)) return api_fail(MAMBO_EINVAL, "out must be f32 or bf16");
  if (ldo < w->n_rows) return api_fail(MAMBO_EINVAL, "out row stride is smaller than N");
  if (!aligned(out, elem(out_dtype))) return api_fail(MAMBO_EINVAL, kUnaligned);
  return MAMBO_OK;
}

int linear_impl(const void* x, int x_kind, int64_t ldx, const uint8_t* xs, int64_t lds, int group, int64_t m,
                const int* offsets, const MamboFp8BlockWeight* w, void* out, int out_dtype, int64_t ldo,
                void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  int sms, smem;
  int st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  const int64_t experts = offsets ? w->n_experts : 1;
  const Plan P = plan(m, experts, m, w->n_rows, w->k, 0);
  st = check_size(P, m, experts, w->k);
  if (st != MAMBO_OK) return st;
  st = check_workspace(workspace, workspace_bytes, kWorkspaceCounterBytes + product_bytes(P));
  if (st != MAMBO_OK) return st;
  uint8_t* at = (uint8_t*)workspace + kWorkspaceCounterBytes;
  const FbActivations act = activations(P, at);
  cudaError_t e;
  if (x_kind != kFbCodes && m <= kFbQuantTokens) {
    const FbSource src = source(x, x_kind, ldx, m, w->k, group);
    e = run_gemm(w, P, &src, act, m, offsets, out, out_dtype == MAMBO_BF16, ldo, nullptr, at + P.x8, workspace, sms, smem,
                 stream);
  } else {
    FbQuantParams q{};
    q.x = x;
    q.x_kind = x_kind;
    q.xs = xs;
    q.lds = lds;
    q.ldx = ldx;
    q.rows = m;
    q.k = w->k;
    q.group = group;
    q.mode = offsets ? kFbGrouped : kFbDense;
    q.experts = (int)experts;
    q.offsets = offsets;
    q.total_rows = m;
    q.act = act;
    e = launch_fb_quant(q, stream);
    if (e != cudaSuccess) return api_cuda_fail(e, "fp8 block quantizer");
    e = run_gemm(w, P, nullptr, act, m, offsets, out, out_dtype == MAMBO_BF16, ldo, nullptr, at + P.x8, workspace, sms,
                 smem, stream);
  }
  if (e != cudaSuccess) return api_cuda_fail(e, "fp8 block product");
  return api_ok();
}

// The experts' path: regions of the workspace after the counters.
struct ExpertsPlan {
  Plan a, b;
  int64_t rows;
  size_t y, partials, total;
};
ExpertsPlan plan_experts(int64_t tokens, int64_t top, int64_t experts, int64_t h, int64_t i, int out_dtype) {
  ExpertsPlan E;
  E.rows = tokens * top;
  // A token mostly picks an expert once; where a route repeats one, its rows take several tiles.
  E.a = plan(E.rows, experts, tokens, 2 * i, h, 1);
  E.b = plan(E.rows, experts, tokens, h, i, 0);  // the same tiles: nt depends on the rows only
  E.y = align256((size_t)E.rows * h * elem(out_dtype));
  const int nt = E.a.nt > E.b.nt ? E.a.nt : E.b.nt;
  E.partials = align256(fb_partial_bytes(nt, kSmsBound));
  E.total = kWorkspaceCounterBytes + E.a.x8 + E.b.x8 + E.y + E.partials;
  return E;
}

}  // namespace

extern "C" {

size_t mambo_fp8b_packed_bytes(int64_t experts, int64_t n, int64_t k, int gate_up) {
  if (!experts_ok(experts) || !extent_ok(n) || !extent_ok(k)) return 0;
  return (size_t)experts * fb_row_tiles(n, gate_up) * ((k + 127) / 128) * kFbRecord;
}

size_t mambo_fp8b_scales_bytes(int64_t experts, int64_t n, int64_t k, int gate_up) {
  return mambo_fp8b_packed_bytes(experts, n, k, gate_up) / kFbRecord * 2 * sizeof(float);
}

int mambo_fp8b_pack(const uint8_t* values, int64_t experts, int64_t n, int64_t k, int64_t stride_expert,
                    int64_t stride_row, int64_t stride_k, const float* block_scales, int64_t scale_stride_expert,
                    int64_t scale_stride_row, int64_t scale_stride_k, int gate_up, void* packed, float* packed_scales,
                    mambo_stream_t stream) {
  if (!values || !block_scales || !packed || !packed_scales) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!experts_ok(experts)) return api_fail(MAMBO_EINVAL, "a weight has 1 to %d experts", kFbMaxExperts);
  if (!extent_ok(n) || !extent_ok(k))
    return api_fail(MAMBO_EINVAL, "weight must have N and K in [1, 2^24]");
  if (gate_up && n % 2) return api_fail(MAMBO_EINVAL, "a gate/up weight has an even number of rows");
  if (!aligned(packed, 16)) return api_fail(MAMBO_EINVAL, "packed buffer must be 16-byte aligned");
  if (!aligned(block_scales, 4) || !aligned(packed_scales, 4)) return api_fail(MAMBO_EINVAL, kUnaligned);
  FbPackParams p{};
  p.w = values;
  p.stride_e = stride_expert;
  p.stride_n = stride_row;
  p.stride_k = stride_k;
  p.s = block_scales;
  p.sstride_e = scale_stride_expert;
  p.sstride_n = scale_stride_row;
  p.sstride_k = scale_stride_k;
  p.experts = (int)experts;
  p.n = (int)n;
  p.k = (int)k;
  p.gate_up = gate_up != 0;
  p.row_tiles = fb_row_tiles(n, gate_up);
  p.kblocks = (int)((k + 127) / 128);
  if ((int64_t)p.experts * p.row_tiles * p.kblocks > 0x7FFFFFFF) return api_fail(MAMBO_EINVAL, "weight too large");
  p.packed = (uint8_t*)packed;
  p.scales = packed_scales;
  int sms, smem;
  const int st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  const cudaError_t e = launch_fb_pack(p, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "fp8 block pack");
  return api_ok();
}

int mambo_fp8b_quantize(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int group, uint8_t* q,
                        int64_t ldq, uint8_t* s, int64_t lds, mambo_stream_t stream) {
  if (!x || !q || !s) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!dtype_ok(x_dtype)) return api_fail(MAMBO_EINVAL, "activation must be f32 or bf16");
  if (m < 1 || m > kMaxRows || !extent_ok(k)) return api_fail(MAMBO_EINVAL, "activation must be [M,K] with M, K >= 1");
  if (group != 32 && group != 128) return api_fail(MAMBO_EINVAL, "activation scales are per 32 or per 128 values");
  if (ldx < k || ldq < k || lds < (k + group - 1) / group) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (!aligned(x, elem(x_dtype))) return api_fail(MAMBO_EINVAL, kUnaligned);
  if (m * ((k + 1023) / 1024) >= 2147483647) return api_fail(MAMBO_EINVAL, "the call is too large: split its rows");
  int sms, smem;
  const int st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  FbQuantParams p{};
  p.x = x;
  p.x_kind = x_dtype;
  p.ldx = ldx;
  p.rows = m;
  p.k = k;
  p.group = group;
  p.mode = kFbDense;
  p.values = q;
  p.ldv = ldq;
  p.scales = s;
  p.ldsc = lds;
  const cudaError_t e = launch_fb_quant(p, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "fp8 block quantizer");
  return api_ok();
}

size_t mambo_fp8b_linear_workspace_bytes(int64_t rows, int64_t experts, int64_t n, int64_t k) {
  if (rows < 1 || rows > kMaxRows || !experts_ok(experts) || !extent_ok(n) || !extent_ok(k)) return 0;
  return kWorkspaceCounterBytes + product_bytes(plan(rows, experts, rows, n, k, 0));
}

int mambo_fp8b_linear(const uint8_t* xq, int64_t ldxq, const uint8_t* xs, int64_t ldxs, int group, int64_t m,
                      const MamboFp8BlockWeight* w, void* out, int out_dtype, int64_t ldo, void* workspace,
                      size_t workspace_bytes, mambo_stream_t stream) {
  if (!xs) return api_fail(MAMBO_EINVAL, "null pointer");
  const int st = check_linear(xq, m, group, w, out, out_dtype, ldo);
  if (st != MAMBO_OK) return st;
  if (w->n_experts != 1) return api_fail(MAMBO_EINVAL, "a weight of several experts needs mambo_fp8b_grouped_linear");
  if (ldxq < w->k || ldxs < (w->k + group - 1) / group) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  return linear_impl(xq, kFbCodes, ldxq, xs, ldxs, group, m, nullptr, w, out, out_dtype, ldo, workspace,
                     workspace_bytes, (cudaStream_t)stream);
}

int mambo_fp8b_linear_fused(const void* x, int x_dtype, int64_t ldx, int group, int64_t m,
                            const MamboFp8BlockWeight* w, void* out, int out_dtype, int64_t ldo, void* workspace,
                            size_t workspace_bytes, mambo_stream_t stream) {
  const int st = check_linear(x, m, group, w, out, out_dtype, ldo);
  if (st != MAMBO_OK) return st;
  if (w->n_experts != 1) return api_fail(MAMBO_EINVAL, "a weight of several experts needs mambo_fp8b_grouped_linear");
  if (!dtype_ok(x_dtype)) return api_fail(MAMBO_EINVAL, "activation must be f32 or bf16");
  if (ldx < w->k) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (!aligned(x, elem(x_dtype))) return api_fail(MAMBO_EINVAL, kUnaligned);
  return linear_impl(x, x_dtype, ldx, nullptr, 0, group, m, nullptr, w, out, out_dtype, ldo, workspace,
                     workspace_bytes, (cudaStream_t)stream);
}

int mambo_fp8b_grouped_linear(const void* x, int x_dtype, int64_t ldx, int group, int64_t rows, const int32_t* offsets,
                              const MamboFp8BlockWeight* w, void* out, int out_dtype, int64_t ldo, void* workspace,
                              size_t workspace_bytes, mambo_stream_t stream) {
  if (!offsets) return api_fail(MAMBO_EINVAL, "null pointer");
  const int st = check_linear(x, rows, group, w, out, out_dtype, ldo);
  if (st != MAMBO_OK) return st;
  if (!dtype_ok(x_dtype)) return api_fail(MAMBO_EINVAL, "activation must be f32 or bf16");
  if (ldx < w->k) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (!aligned(x, elem(x_dtype)) || !aligned(offsets, 4)) return api_fail(MAMBO_EINVAL, kUnaligned);
  return linear_impl(x, x_dtype, ldx, nullptr, 0, group, rows, offsets, w, out, out_dtype, ldo, workspace,
                     workspace_bytes, (cudaStream_t)stream);
}

size_t mambo_moe_route_workspace_bytes(int64_t tokens, int64_t experts) {
  if (!choices_ok(tokens, 1) || !experts_ok(experts)) return 0;
  const int64_t chunk = fb_route_chunk(tokens);
  return kWorkspaceCounterBytes + align256((size_t)((tokens + chunk - 1) / chunk) * (experts + 1) * sizeof(int));
}

int mambo_moe_route(const void* logits, int dtype, int64_t ld, const float* bias, int64_t tokens, int64_t experts,
                    int top, int scoring, int renormalize, float scale, int32_t* ids, float* weights, int32_t* offsets,
                    int32_t* positions, int32_t* rows, void* workspace, size_t workspace_bytes,
                    mambo_stream_t stream) {
  if (!logits || !ids || !weights || !offsets || !positions) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!dtype_ok(dtype)) return api_fail(MAMBO_EINVAL, "logits must be f32 or bf16");
  if (!experts_ok(experts)) return api_fail(MAMBO_EINVAL, "1 to %d experts", kFbMaxExperts);
  if (top < 1 || top > MAMBO_MOE_MAX_TOP || top > experts)
    return api_fail(MAMBO_EINVAL, "top must be in [1, min(%d, experts)]", MAMBO_MOE_MAX_TOP);
  if (!choices_ok(tokens, top)) return api_fail(MAMBO_EINVAL, "tokens must be at least 1, tokens * top at most 2^28");
  if (ld < experts) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (scoring != MAMBO_MOE_SOFTMAX && scoring != MAMBO_MOE_SIGMOID) return api_fail(MAMBO_EINVAL, "unknown scoring %d", scoring);
  int st = check_workspace(workspace, workspace_bytes, mambo_moe_route_workspace_bytes(tokens, experts));
  if (st != MAMBO_OK) return st;
  if (!aligned(logits, elem(dtype)) || !aligned(bias, 4) || !aligned(ids, 4) || !aligned(weights, 4) || !aligned(offsets, 4) ||
      !aligned(positions, 4) || !aligned(rows, 4))
    return api_fail(MAMBO_EINVAL, kUnaligned);
  int sms, smem;
  st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  FbRouteParams p{};
  p.logits = logits;
  p.bf16 = dtype == MAMBO_BF16;
  p.ld = ld;
  p.bias = bias;
  p.tokens = (int)tokens;
  p.chunk = fb_route_chunk(tokens);
  p.experts = (int)experts;
  p.top = top;
  p.sigmoid = scoring == MAMBO_MOE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  p.ids = ids;
  p.weights = weights;
  p.offsets = offsets;
  p.positions = positions;
  p.rows = rows;
  p.chunk_counts = (int*)((uint8_t*)workspace + kWorkspaceCounterBytes);
  const cudaError_t e = launch_fb_route(p, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "expert router");
  return api_ok();
}

int mambo_moe_combine(const void* y, int y_dtype, int64_t ldy, int64_t rows, const int32_t* positions,
                      const float* weights, int64_t tokens, int top, int64_t h, void* out, int out_dtype, int64_t ldo,
                      mambo_stream_t stream) {
  if (!y || !positions || !weights || !out) return api_fail(MAMBO_EINVAL, "null pointer");
  if (!dtype_ok(y_dtype) || !dtype_ok(out_dtype)) return api_fail(MAMBO_EINVAL, "y and out must be f32 or bf16");
  if (!choices_ok(tokens, top) || rows < 1 || !extent_ok(h))
    return api_fail(MAMBO_EINVAL, "bad tokens, top, rows or width");
  if (ldy < h || ldo < h) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (!aligned(y, elem(y_dtype)) || !aligned(positions, 4) || !aligned(weights, 4) || !aligned(out, elem(out_dtype)))
    return api_fail(MAMBO_EINVAL, kUnaligned);
  int sms, smem;
  const int st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  FbCombineParams c{y, y_dtype == MAMBO_BF16, ldy, positions, weights, (int)tokens, top, (int)h, rows, out,
                    out_dtype == MAMBO_BF16, ldo};
  const cudaError_t e = launch_fb_combine(c, (cudaStream_t)stream);
  if (e != cudaSuccess) return api_cuda_fail(e, "expert combine");
  return api_ok();
}

size_t mambo_moe_experts_workspace_bytes(int64_t tokens, int top, int64_t experts, int64_t h, int64_t i,
                                         int out_dtype) {
  if (top > MAMBO_MOE_MAX_TOP || !choices_ok(tokens, top) || !experts_ok(experts) || !extent_ok(h) || !extent_ok(i)) return 0;
  return plan_experts(tokens, top, experts, h, i, out_dtype).total;
}

int mambo_moe_experts(const void* x, int x_dtype, int64_t ldx, int64_t tokens, const int32_t* ids,
                      const float* weights, const int32_t* positions, const int32_t* offsets, const int32_t* rows,
                      int top, const MamboFp8BlockWeight* gate_up, const MamboFp8BlockWeight* down, void* out, int out_dtype,
                      int64_t ldo, void* workspace, size_t workspace_bytes, mambo_stream_t stream_) {
  if (!x || !ids || !weights || !positions || !offsets || !out) return api_fail(MAMBO_EINVAL, "null pointer");
  int st = check_weight(gate_up);
  if (st == MAMBO_OK) st = check_weight(down);
  if (st != MAMBO_OK) return st;
  if (!gate_up->gate_up || down->gate_up)
    return api_fail(MAMBO_EINVAL, "gate_up must be a gate/up weight and down a plain one");
  const int64_t experts = gate_up->n_experts, h = gate_up->k, i = gate_up->n_rows / 2;
  if (down->n_experts != experts || down->n_rows != h || down->k != i)
    return api_fail(MAMBO_EINVAL, "down must be [experts, hidden size, features] to the gate/up weight's [experts, 2 * features, hidden size]");
  if (!dtype_ok(x_dtype) || !dtype_ok(out_dtype)) return api_fail(MAMBO_EINVAL, "x and out must be f32 or bf16");
  if (top < 1 || top > MAMBO_MOE_MAX_TOP) return api_fail(MAMBO_EINVAL, "top must be in [1, %d]", MAMBO_MOE_MAX_TOP);
  if (!choices_ok(tokens, top)) return api_fail(MAMBO_EINVAL, "tokens must be at least 1, tokens * top at most 2^28");
  if (ldx < h || ldo < h) return api_fail(MAMBO_EINVAL, "row stride smaller than the row");
  if (!aligned(x, elem(x_dtype)) || !aligned(ids, 4) || !aligned(weights, 4) || !aligned(positions, 4) || !aligned(offsets, 4) ||
      !aligned(rows, 4) || !aligned(out, elem(out_dtype)))
    return api_fail(MAMBO_EINVAL, kUnaligned);
  const ExpertsPlan E = plan_experts(tokens, top, experts, h, i, out_dtype);
  st = check_size(E.a, E.rows, experts, h);
  if (st == MAMBO_OK) st = check_size(E.b, E.rows, experts, i);
  if (st != MAMBO_OK) return st;
  st = check_workspace(workspace, workspace_bytes, E.total);
  if (st != MAMBO_OK) return st;
  int sms, smem;
  st = api_require_sm100(&sms, &smem);
  if (st != MAMBO_OK) return st;
  cudaStream_t stream = (cudaStream_t)stream_;
  uint8_t* at = (uint8_t*)workspace + kWorkspaceCounterBytes;
  const FbActivations xa = activations(E.a, at);
  at += E.a.x8;
  const FbActivations ha = activations(E.b, at);
  at += E.b.x8;
  void* y = at;
  at += E.y;
  uint8_t* partials = at;

  cudaError_t e;
  // Tiles of 16 tokens, the form that quantizes them: of more only where one expert has more than 16 rows of two tokens.
  if (rows && tokens <= kFbQuantTokens && E.a.nt == 16) {
    FbSource src = source(x, x_dtype, ldx, tokens, h, 32);
    src.rows = rows;
    src.top = top;
    e = run_gemm(gate_up, E.a, &src, xa, E.rows, offsets, nullptr, 0, 0, &ha, partials, workspace, sms, smem, stream);
  } else {
    FbQuantParams q{};
    q.x = x;
    q.x_kind = x_dtype;
    q.ldx = ldx;
    q.rows = tokens;
    q.k = h;
    q.group = 32;
    q.mode = kFbRouted;
    q.experts = (int)experts;
    q.offsets = offsets;
    q.ids = ids;
    q.positions = positions;
    q.top = top;
    q.total_rows = E.rows;
    q.act = xa;
    e = launch_fb_quant(q, stream);
    if (e == cudaSuccess)
      e = run_gemm(gate_up, E.a, nullptr, xa, E.rows, offsets, nullptr, 0, 0, &ha, partials, workspace, sms, smem, stream);
  }
  // An expert's row rounds once to the output type before the weighted sum, which is FP32 and rounds once more. Kept in
  // f32 for a bf16 output, the rows cost 8 % of a prompt (4096 tokens, 64 experts of 2048 x 4096, eight a token: 1,340 ->
  // 1,442 us) and 2 % of a token (28.8 -> 29.5); the error against float64 is 2.35e-3 of the norm as it is, 1.66e-3 with
  // the output's rounding alone. Who wants the latter takes an f32 output and rounds it.
  if (e == cudaSuccess)
    e = run_gemm(down, E.b, nullptr, ha, E.rows, offsets, y, out_dtype == MAMBO_BF16, h, nullptr, partials, workspace, sms,
                 smem, stream);
  if (e == cudaSuccess) {
    FbCombineParams c{y, out_dtype == MAMBO_BF16, h, positions, weights, (int)tokens, top, (int)h, E.rows, out,
                      out_dtype == MAMBO_BF16, ldo};
    e = launch_fb_combine(c, stream);
  }
  if (e != cudaSuccess) return api_cuda_fail(e, "experts");
  return api_ok();
}

}  // extern "C"
