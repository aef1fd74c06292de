// Layouts and parameter blocks of the FP8 block-scaled linear (E4M3 weights
// with one f32 scale per 128 x 128 block) and of its expert-grouped form.
//
// Weights, packed once: a 16 KB record per (128-row tile, 128-wide K block),
// the tile's bytes in the tensor core's 128-byte-swizzled K-major layout (row
// r at 128*r, its 16-byte chunk c at chunk c ^ (r & 7)), records K-block
// consecutive per row tile, row tiles consecutive per expert. A record is one
// bulk copy and needs no tensor map; rows past N and values past K are zero.
// Scales: f32 [experts][row tiles][2][K blocks]; entry 0 scales the rows of
// the tile's even 32-row quarters, entry 1 those of the odd ones (equal,
// unless the tile interleaves gate and up rows by quarters).
//
// Activations, written by the quantizer for each call: a record per (token
// tile, K block), again one bulk copy (per CTA): the tile's rows of 128 E4M3
// bytes, swizzled, then its scale codes (UE8M0, one per 32 values) as the
// tensor core's scale-factor atoms, 512 bytes per 128 tokens. For tiles of a
// CTA pair a record has a part per CTA, each with its half of either MMA's
// tokens (fb_split) and all the scale codes.
//
// Ragged segments: expert e owns rows [o_e, o_{e+1}) of R; its token tiles have
// the slots from o_e / nt + e on: since floor(a + c) - floor(a) + 1 >= ceil(c)
// in units of nt, consecutive segments never overlap, and no prefix sum over
// the experts is needed to place a row.
#pragma once

#include "common.cuh"
#include "mxfp8.cuh"

namespace mambo {

constexpr int kFbBlock = 128;                // K block, rows of a weight tile
constexpr uint32_t kFbRecord = 128u * 128u;  // bytes of a packed weight record
constexpr uint32_t kFbAtom = 512u;           // bytes of a scale-factor atom (128 rows x 4 groups)
constexpr int kFbMaxExperts = 1024;

// Tokens of a CTA pair's tile, the largest; single CTAs take tiles of 16, 32 and 64 (fb_tile_for).
constexpr int kFbPairTokens = 192;

struct FbActivations {
  uint8_t* x8;    // [slots][kblocks][record]
  int64_t slots;  // token-tile slots
  int kblocks;
  int nt;         // most tokens of a tile
};

__host__ __device__ constexpr bool fb_is_pair(int nt) { return nt > 128; }
__host__ __device__ constexpr int fb_atoms_per_tile(int nt) { return (nt + 127) / 128; }
// Bytes of a CTA's part of a record, and of a record.
__host__ __device__ constexpr uint32_t fb_part_bytes(int nt) {
  return (uint32_t)((fb_is_pair(nt) ? nt / 2 : nt) * 128) + fb_atoms_per_tile(nt) * kFbAtom;
}
__host__ __device__ constexpr uint32_t fb_record_bytes(int nt) { return (fb_is_pair(nt) ? 2 : 1) * fb_part_bytes(nt); }
__host__ __device__ inline int64_t fb_slots(int64_t rows, int64_t experts, int nt) { return rows / nt + experts; }
__host__ __device__ inline int64_t fb_slot_start(int o, int e, int nt) { return o / nt + e; }
// A pair's tile of n tokens is two MMAs: the first takes this many tokens (a multiple of 16), the second the rest.
__host__ __device__ inline int fb_split(int n) { return ((n + 15) / 16 + 1) / 2 * 16; }
// Rows that a CTA holds of a tile of n tokens, before its scale codes: alone all (in groups of 8), of a pair half of
// each MMA's N (rounded up to 16).
__host__ __device__ inline int fb_part_rows(int n, bool pair) { return pair ? (n + 15) / 16 * 8 : (n + 7) / 8 * 8; }
// A segment of `count` rows is cut into equal tiles of at most nt tokens, a multiple of 16 each.
__host__ __device__ inline int fb_tiles(int count, int nt) { return (count + nt - 1) / nt; }
__host__ __device__ inline int fb_tile_rows(int count, int tiles) {
  return tiles > 0 ? ((count + tiles - 1) / tiles + 15) / 16 * 16 : 16;
}

#ifdef __CUDACC__
// Where row `local` of expert e (o_e, count) lies: its tile's slot, its row there and the tile's tokens.
struct FbPlace {
  int64_t slot;
  int in_tile, n;
};
__device__ __forceinline__ FbPlace fb_place(int o, int count, int e, int local, int nt) {
  FbPlace pl;
  const int tiles = fb_tiles(count, nt), tr = fb_tile_rows(count, tiles);
  const int tt = local / tr;
  pl.slot = fb_slot_start(o, e, nt) + tt;
  pl.in_tile = local - tt * tr;
  pl.n = min(tr, count - tt * tr);
  return pl;
}

// Where a row goes in the records of its K blocks: its 128 bytes' address in the first one, its scale word's, and the
// swizzle of its 16-byte chunks. row is null for a row that has no place.
struct FbDst {
  uint8_t* row;
  uint8_t* sf;
  int swz;
};
__device__ __forceinline__ FbDst fb_dst(const FbActivations& a, const FbPlace& pl) {
  FbDst d;
  d.row = nullptr;
  if (pl.slot < 0 || pl.slot >= a.slots) return d;
  const bool pair = fb_is_pair(a.nt);
  uint8_t* rec = a.x8 + pl.slot * a.kblocks * fb_record_bytes(a.nt);
  int row = pl.in_tile, part = 0, half = 0, t = pl.in_tile;  // t: place among its MMA's tokens
  if (pair) {
    const int nn = (pl.n + 15) / 16 * 16, n0 = fb_split(pl.n), n1 = nn - n0;
    half = t >= n0;
    t -= half * n0;
    const int per = (half ? n1 : n0) / 2;
    part = t >= per;
    row = t - part * per + half * (n0 / 2);
  }
  d.row = rec + part * fb_part_bytes(a.nt) + row * 128;
  d.sf = rec + fb_part_rows(pl.n, pair) * 128 + half * kFbAtom + (t & 31) * 16 + (t >> 5) * 4;
  d.swz = row & 7;
  return d;
}
// 8 values of a lane, of a scale group of 4 (32 values) or 16 lanes: their E4M3 bytes, and the K block's four scale
// codes as a word.
__device__ __forceinline__ uint32_t scale_word(uint32_t code, int lane) {
  uint32_t word = code << (8 * ((lane >> 2) & 3));
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
  return word | __shfl_xor_sync(0xFFFFFFFFu, word, 8);
}
// bf16 pairs: the maximum of packed magnitudes (NaN wins) and packed multiplications.
__device__ __forceinline__ uint2 quantize8(const uint4& c, int group, int lane, uint32_t& word) {
  uint32_t a = absmax_bf16x2(absmax_bf16x2(c.x, c.y), absmax_bf16x2(c.z, c.w));
  a = absmax_bf16x2(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
  a = absmax_bf16x2(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
  if (group == 128) {
    a = absmax_bf16x2(a, __shfl_xor_sync(0xFFFFFFFFu, a, 4));
    a = absmax_bf16x2(a, __shfl_xor_sync(0xFFFFFFFFu, a, 8));
  }
  const uint32_t code = mxfp8_scale_code(__uint_as_float(max(a & 0x7FFFu, (a >> 16) & 0x7FFFu) << 16));
  const float inv = e8m0_to_float(code == 0xFFu ? 0u : 254u - code);
  const uint32_t w4[4] = {c.x, c.y, c.z, c.w};
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo, hi;
    mul2(lo, hi, __uint_as_float(w4[j] << 16), __uint_as_float(w4[j] & 0xFFFF0000u), inv, inv);
    b[j] = cvt_e4m3x2_rn(lo, hi);
  }
  word = scale_word(code, lane);
  return make_uint2(prmt(b[0], b[1], 0x5410u), prmt(b[2], b[3], 0x5410u));
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], int group, int lane, uint32_t& word) {
  // Largest magnitude as bits: NaN orders above infinity, so either gives the group the code 0xFF.
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  if (group == 128) {
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
  }
  const uint32_t code = mxfp8_scale_code(__uint_as_float(m));
  const float inv = e8m0_to_float(code == 0xFFu ? 0u : 254u - code);
  uint32_t packed[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    packed[h] = cvt_e4m3x2_rn(v[4 * h] * inv, v[4 * h + 1] * inv) |
                (cvt_e4m3x2_rn(v[4 * h + 2] * inv, v[4 * h + 3] * inv) << 16);
  word = scale_word(code, lane);
  return make_uint2(packed[0], packed[1]);
}

__device__ __forceinline__ int clamp_offset(int o, int64_t total) { return o < 0 ? 0 : o > total ? (int)total : o; }
#endif

// --- weight packing ----------------------------------------------------------
struct FbPackParams {
  const uint8_t* w;  // E4M3 [experts][N][K] with any strides (bytes)
  int64_t stride_e, stride_n, stride_k;
  const float* s;    // [experts][row blocks][K blocks] with any strides (elements)
  int64_t sstride_e, sstride_n, sstride_k;
  int experts, n, k;
  int gate_up;       // 1: rows [0, n/2) are gate, [n/2, n) up, interleaved by quarters of a tile
  int row_tiles, kblocks;
  uint8_t* packed;
  float* scales;
};
cudaError_t launch_fb_pack(const FbPackParams& p, cudaStream_t stream);
__host__ __device__ inline int fb_row_tiles(int64_t n, int gate_up) {
  // Gate and up: 64 hidden features per tile, whole 128-feature blocks.
  return gate_up ? (int)((n / 2 + 127) / 128) * 2 : (int)((n + 127) / 128);
}

// --- activation quantization ---------------------------------------------------
enum { kFbDense = 0, kFbGrouped = 1, kFbRouted = 2 };
struct FbQuantParams {
  const void* x;  // [rows][k], row stride ldx elements
  int x_kind;     // MAMBO_F32, MAMBO_BF16, or kFbCodes: already E4M3 with the scale codes of xs
  const uint8_t* xs;
  int64_t lds;
  int64_t ldx;
  int64_t rows, k;
  int group;  // 32 or 128 values per scale
  int mode;   // kFb*
  int experts;
  const int* offsets;    // [experts + 1] (kFbGrouped, kFbRouted)
  const int* ids;        // [rows][top] (kFbRouted): expert of each copy of the row, < 0 for none
  const int* positions;  // [rows][top]: its row in expert order
  int top;
  int64_t total_rows;    // rows in expert order (bounds every position)
  FbActivations act;
  // Row-major outputs instead of act (kFbDense, values != null).
  uint8_t* values;
  int64_t ldv;
  uint8_t* scales;
  int64_t ldsc;
};
constexpr int kFbCodes = 100;
cudaError_t launch_fb_quant(const FbQuantParams& p, cudaStream_t stream);

// --- the product -----------------------------------------------------------------
// Unquantized activations that the product's own warps quantize (tiles of 16 tokens, calls of at most kFbQuantTokens).
struct FbSource {
  const void* x;     // [rows][k], row stride ldx; null: none
  int bf16;          // else f32
  int vec;           // rows 16-byte aligned
  int64_t ldx, k;
  int group;         // 32 or 128 values per scale
  const int* rows;   // row r of the product is row rows[r] / top of x; null: row r
  int top, last;     // last: x's last row, which bounds the others
};
constexpr int kFbQuantTokens = 2;  // most tokens of a call that the product quantizes itself
struct FbGemmParams {
  FbSource src;
  const uint8_t* packed;
  const float* scales;
  FbActivations act;
  int experts;
  int64_t rows;        // R (dense: M); bounds the offsets
  const int* offsets;  // device [experts + 1], or null for a dense call
  int n_rows;          // valid rows of the weight (output columns)
  int row_tiles;
  void* out;           // [R][ldo]
  int out_bf16;
  int64_t ldo;
  // Gate/up weights: h = silu(gate) * up of each row, quantized (MXFP8) into the
  // next product's activations, in place of out; its tiles are cut as act's.
  FbActivations hidden;  // x8 null: none
  int stages;
  int evict_weights;   // 1: weights are mostly read once (evict-first)
  float* partials;     // [grid][2][128 * nt]
  int* counters;       // [grid][8], zero on entry and left zero
};
// Device addresses of the product kernels' status record and wait limit (the current device's).
cudaError_t fb_status_symbols(void** status, void** limit);
// The tile, of those that the kernel is built for, for a call or an expert of so many rows.
int fb_tile_for(int64_t expected_rows);
uint32_t fb_gemm_smem(int nt, int experts, int stages, bool hidden);
int fb_gemm_stages(int nt, int experts, int smem_optin, bool hidden);
int fb_gemm_grid(int nt, int sms);
size_t fb_partial_bytes(int nt, int sms);
cudaError_t launch_fb_gemm(const FbGemmParams& p, int grid, cudaStream_t stream);

// --- experts ----------------------------------------------------------------------
struct FbRouteParams {
  int chunk;  // tokens of a CTA (fb_route_chunk)
  const void* logits;
  int bf16;
  int64_t ld;
  const float* bias;
  int tokens, experts, top;
  int sigmoid, renormalize;
  float scale;
  int* ids;
  float* weights;
  int* offsets;
  int* positions;
  int* rows;
  int* chunk_counts;  // workspace [chunks][experts + 1]
};
int fb_route_chunk(int64_t tokens);
cudaError_t launch_fb_route(const FbRouteParams& p, cudaStream_t stream);

struct FbCombineParams {
  const void* y;  // [R][ldy]
  int y_bf16;
  int64_t ldy;
  const int* positions;
  const float* weights;
  int tokens, top, h;
  int64_t rows;   // R, bounds the positions
  void* out;
  int out_bf16;
  int64_t ldo;
};
cudaError_t launch_fb_combine(const FbCombineParams& p, cudaStream_t stream);

}  // namespace mambo
