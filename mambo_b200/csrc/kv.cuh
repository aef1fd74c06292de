// Layouts and parameter blocks of the paged FP8 key/value cache: rotary
// positions, the append and attention.
//
// Cache: E4M3 codes [pages][heads][page tokens][head size], keys and values
// apart, with one UE8M0 scale code per (page, head). A page is 16, 32, 64 or
// 128 tokens, so that it is a whole box of a tensor copy and whole 8-row
// groups of the tensor core's layout. Exponents are -64 .. 127 (codes 63 ..
// 254): the factors between pages then stay in the range of a float; code 255
// marks a page with a value that was NaN or infinite.
//
// A sequence's tokens lie in the pages that its row of the page table names.
// An entry outside the cache has no tokens: the append drops them, attention
// does not see them.
#pragma once

#include "common.cuh"

namespace mambo {

constexpr int kKvMaxDim = 128;
constexpr uint32_t kKvMinCode = 63;  // of the scale 2^-64

// Rotation: pair p of the first 2 * pairs dimensions turns by position * turns[p] (a 64-bit fraction of a turn, so that
// the product wraps exactly however far the position is), scaled by magnitude.
struct RotaryParams {
  const uint64_t* turns;  // null: no rotation
  int pairs;
  int interleaved;        // pair p: dimensions 2p, 2p+1; else p, p + pairs
  float magnitude;
  float sign;             // -1: the inverse rotation
};

struct RotaryCall {
  RotaryParams rot;
  const void* x;
  void* out;
  int bf16;
  int tokens, heads, dim;
  int64_t xs_t, xs_h, os_t, os_h;  // strides in elements
  const void* positions;
  int positions64;
  int units, groups;  // of a head: units of 16 dimensions, or pairs of values where rows are not made of aligned vectors; of its heads
};
cudaError_t launch_rotary(RotaryCall p, cudaStream_t stream);

struct KvCache {
  uint8_t* codes[2];   // keys, values
  uint8_t* scales[2];
  int64_t pages;
  int heads, page, dim, log_page;
};

// The sequences of a call: tokens offsets[b] .. offsets[b+1] of the call (token b alone where offsets is null) belong
// to sequence b, whose pages are table[b * table_stride ..].
struct KvSequences {
  const int* table;
  int64_t table_stride;
  int table_pages;
  const int* lengths;  // append: tokens before the call; attention: with the call's tokens
  const int* offsets;
  int batch;
  int tokens;
};

struct KvAppendCall {
  RotaryParams rot;
  KvCache cache;
  KvSequences seq;
  const void* x[2];    // keys, values [tokens][heads][dim]
  int64_t xs_t[2], xs_h[2];
  int bf16;
  int heads_each;      // heads of a CTA
  int rows_each;       // tokens of a CTA's threads at a time
  int first;           // of the launch: 0 keys (and values), 1 values
};
cudaError_t launch_kv_append(KvAppendCall p, cudaStream_t stream);

struct KvAttentionCall {
  KvCache cache;
  KvSequences seq;
  const uint16_t* q;   // bf16 [tokens][heads * group][dim]
  int64_t qs_t, qs_h;
  uint16_t* out;       // bf16
  int64_t os_t, os_h;
  float* lse;          // f32 [tokens][query heads], or null
  int64_t ls_t, ls_h;
  int group;           // query heads of a key head
  int window;          // 0: none
  float scale;         // of the scores
  int few;             // rows (tokens * group) of a sequence up to which the decode kernel has it; 0: it has none
};
bool kv_page_map(const KvCache& c, int which, CUtensorMap* map);
size_t kv_decode_partial_bytes(int group, int sms);
cudaError_t launch_kv_decode(const KvAttentionCall& p, const CUtensorMap& k, const CUtensorMap& v, int sms, int smem_optin,
                             float* partials, int* counters, cudaStream_t stream);
size_t kv_prompt_partial_bytes(int sms);
cudaError_t launch_kv_prompt(const KvAttentionCall& p, const CUtensorMap& k, const CUtensorMap& v, int sms, float* partials,
                             int* counters, cudaStream_t stream);
// Device addresses of the prompt kernel's status record and wait limit (the current device's).
cudaError_t kv_prompt_status_symbols(void** status, void** limit);

#ifdef __CUDACC__
// The call's tokens of sequence b: [first, first + count), clamped to the call.
struct KvSpan {
  int first, count;
};
__device__ __forceinline__ KvSpan kv_span(const KvSequences& s, int b) {
  KvSpan r;
  if (!s.offsets) {
    r.first = b;
    r.count = 1;
    return r;
  }
  const int o0 = min(max(__ldg(s.offsets + b), 0), s.tokens), o1 = min(max(__ldg(s.offsets + b + 1), 0), s.tokens);
  r.first = o0;
  r.count = max(o1 - o0, 0);
  return r;
}
// A sequence's length, clamped to what its row of the table can hold.
__device__ __forceinline__ int kv_length(const KvSequences& s, int b, int page) {
  const int64_t most = (int64_t)s.table_pages * page;
  const int n = max(__ldg(s.lengths + b), 0);
  return n < most ? n : (int)most;
}
#endif

}  // namespace mambo
