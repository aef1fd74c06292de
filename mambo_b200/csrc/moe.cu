// Expert routing and the weighted sum of a token's expert outputs (layouts in
// fp8b.cuh; the hidden activation is formed in the product, fp8b_gemm.cu).
#include "fp8b.cuh"
#include "kernels.cuh"
#include "mxfp8.cuh"

namespace mambo {

namespace {

// Threads of a routing CTA: as many warps as its registers allow, a token each at a time (more than 256 experts need
// more registers a thread).
constexpr int kPlaceThreads = 1024;
__host__ __device__ constexpr int route_threads(int nv) { return nv <= 8 ? 1024 : 512; }

// Monotone map of a number to an unsigned key: 0 is free (it marks masked experts), zeros of either sign have one key.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? 0u - b : b | 0x80000000u;
}

// One token, a warp: expert 32*i + lane in slot i of the lane. Experts whose
// logit is -inf or NaN are masked; +inf counts as the largest finite number.
template <int NV>
__device__ __forceinline__ void route_load(const FbRouteParams& p, int token, int lane, float (&raw)[NV]) {
  const int64_t at = (int64_t)token * p.ld + lane;
  if (p.bf16) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      raw[i] = 32 * i + lane < p.experts ? __uint_as_float((uint32_t)__ldg((const uint16_t*)p.logits + at + 32 * i) << 16)
                                         : -INFINITY;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      raw[i] = 32 * i + lane < p.experts ? __ldg((const float*)p.logits + at + 32 * i) : -INFINITY;
  }
}

// The probability of a logit, before any renormalization.
__device__ __forceinline__ float route_prob(bool sigmoid, float l, float top, float sum) {
  return sigmoid ? 1.0f / (1.0f + expf(-l)) : expf(l - top) / sum;
}

template <int NV>
__device__ __forceinline__ void route_token(const FbRouteParams& p, int token, int lane, const float (&raw)[NV],
                                            const float (&bias)[NV], int* hist) {
  uint32_t key[NV];
  float top = -INFINITY, sum = 0.f;
  float l[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float v = raw[i];
    l[i] = v == v ? fminf(v, 3.4028234663852886e38f) : -INFINITY;
    top = fmaxf(top, l[i]);
  }
  if (!p.sigmoid) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += l[i] == -INFINITY ? 0.f : expf(l[i] - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float s = (p.sigmoid ? 1.0f / (1.0f + expf(-l[i])) : l[i]) + bias[i];
    key[i] = l[i] == -INFINITY || s != s ? 0u : order_key(s);
  }
  // Each lane's best two keys and their slots (the first of equal keys: the lowest expert of the lane). A lane whose
  // best is taken goes on with the second; only one that is taken again looks through its keys anew.
  uint32_t best = 0, second = 0, taken = 0;
  int at = 0, at2 = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool b1 = key[i] > best, b2 = key[i] > second;
    second = b1 ? best : b2 ? key[i] : second;
    at2 = b1 ? at : b2 ? i : at2;
    best = b1 ? key[i] : best;
    at = b1 ? i : at;
  }
  bool have2 = true;
  int mine_id = -1;
  for (int j = 0; j < p.top; ++j) {
    const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, best);
    if (m == 0) break;  // no expert left
    const uint32_t id = __reduce_min_sync(0xFFFFFFFFu, best == m ? (uint32_t)(32 * at + lane) : 0xFFFFFFFFu);
    if (lane == j) mine_id = (int)id;
    const bool won = lane == (int)(id & 31);
    if (won) taken |= 1u << at;
    if (__any_sync(0xFFFFFFFFu, won && !have2)) {
      if (won) {
        best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (!((taken >> i) & 1u) && key[i] > best) {
            best = key[i];
            at = i;
          }
      }
    } else if (won) {
      best = second;
      at = at2;
      have2 = false;
    }
  }
  // Lane j has the j-th choice: its probability from its logit, once more.
  float w = 0.f;
  if (mine_id >= 0) {
    const int64_t from = (int64_t)token * p.ld + mine_id;
    const float v = p.bf16 ? __uint_as_float((uint32_t)__ldg((const uint16_t*)p.logits + from) << 16)
                           : __ldg((const float*)p.logits + from);
    w = route_prob(p.sigmoid, fminf(v, 3.4028234663852886e38f), top, sum);
  }
  if (p.renormalize) {
    float total = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
    w = total > 0.f ? w / total : 0.f;
  }
  if (lane < p.top) {
    p.ids[(int64_t)token * p.top + lane] = mine_id;
    p.weights[(int64_t)token * p.top + lane] = w * p.scale;
    atomicAdd(hist + (mine_id < 0 ? p.experts : mine_id), 1);  // whole numbers: the order does not matter
  }
}

// In-place exclusive scan of n counts in shared memory by warp 0.
__device__ __forceinline__ void scan_counts(int* v, int n, int lane) {
  int carry = 0;
  for (int b = 0; b < n; b += 32) {
    const int x = b + lane < n ? v[b + lane] : 0;
    int t = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, t, d);
      if (lane >= d) t += up;
    }
    if (b + lane < n) v[b + lane] = carry + t - x;
    carry += __shfl_sync(0xFFFFFFFFu, t, 31);
  }
}

// The chunk's (token, choice) pairs in order, each to its row: base[e] holds
// the first free row of expert e for this chunk (bucket `experts`: no expert).
template <int kRouteThreads>
__device__ __forceinline__ void place_chunk(const FbRouteParams& p, int first, int count, const int* base, int* wcnt,
                                            int warp, int lane) {
  constexpr int kRouteWarps = kRouteThreads / 32;
  const int n = count * p.top, buckets = p.experts + 1;
  const int per = (n + kRouteWarps * 32 - 1) / (kRouteWarps * 32) * 32;  // entries of a warp, whole groups of 32
  const int b0 = min(n, warp * per), b1 = min(n, b0 + per);
  const int* ids = p.ids + (int64_t)first * p.top;
  for (int i = threadIdx.x; i < kRouteWarps * buckets; i += kRouteThreads) wcnt[i] = 0;
  __syncthreads();
  for (int i = b0 + lane; i < b1; i += 32) {
    const int e = ids[i];
    atomicAdd(wcnt + warp * buckets + (e < 0 ? p.experts : e), 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < buckets; e += kRouteThreads) {
    int at = base[e];
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = wcnt[w * buckets + e];
      wcnt[w * buckets + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i0 = b0; i0 < b1; i0 += 32) {
    const int i = i0 + lane;
    const bool have = i < b1;
    const int id = have ? ids[i] : -2;
    const int e = id < 0 ? p.experts : id;
    const unsigned same = __match_any_sync(0xFFFFFFFFu, id);
    int* c = wcnt + warp * buckets + e;
    const int at = have ? *c + __popc(same & ((1u << lane) - 1u)) : 0;
    __syncwarp();
    if (have) {
      if ((same >> lane) == 1u) *c = at + 1;  // the group's last lane
      const int64_t slot = (int64_t)first * p.top + i;
      p.positions[slot] = id < 0 ? -1 : at;
      if (p.rows) p.rows[at] = id < 0 ? -1 : (int)slot;
    }
    __syncwarp();
  }
}

}  // namespace

// Selection of a chunk's tokens, a warp per token, and the chunk's counts per
// expert; with one chunk also the placement. Latency-bound in decode.
template <int NV>
__global__ void __launch_bounds__(route_threads(NV), 1) moe_route_kernel(const __grid_constant__ FbRouteParams p) {
  constexpr int kRouteThreads = route_threads(NV), kRouteWarps = kRouteThreads / 32;
  extern __shared__ int route_sm[];
  int* hist = route_sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, buckets = p.experts + 1;
  const int first = blockIdx.x * p.chunk, count = min(p.chunk, p.tokens - first);
  for (int i = threadIdx.x; i < buckets; i += kRouteThreads) hist[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  float bias[NV], raw[NV], next[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) bias[i] = p.bias && 32 * i + lane < p.experts ? __ldg(p.bias + 32 * i + lane) : 0.f;
  if (warp < count) route_load<NV>(p, first + warp, lane, next);
  for (int t = warp; t < count; t += kRouteWarps) {
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = next[i];
    if (t + kRouteWarps < count) route_load<NV>(p, first + t + kRouteWarps, lane, next);  // while this one is ranked
    route_token<NV>(p, first + t, lane, raw, bias, hist);
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int i = threadIdx.x; i < buckets; i += kRouteThreads) p.chunk_counts[(int64_t)blockIdx.x * buckets + i] = hist[i];
    return;
  }
  if (warp == 0) scan_counts(hist, buckets, lane);
  __syncthreads();
  for (int i = threadIdx.x; i < buckets; i += kRouteThreads) p.offsets[i] = hist[i];
  place_chunk<kRouteThreads>(p, first, count, hist, hist + buckets, warp, lane);
}

// Placement of one chunk: every CTA sums the chunks' counts itself (the counts
// of a 16384-token call are 128 x 257 numbers in L2), so there is no third launch.
__global__ void __launch_bounds__(kPlaceThreads, 1) moe_place_kernel(const __grid_constant__ FbRouteParams p) {
  constexpr int kRouteThreads = kPlaceThreads, kRouteWarps = kRouteThreads / 32;
  extern __shared__ int route_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, buckets = p.experts + 1;
  int* base = route_sm;            // totals, then first rows
  int* before = base + buckets;    // counts of earlier chunks
  int* wcnt = before + buckets;
  const int first = blockIdx.x * p.chunk, count = min(p.chunk, p.tokens - first);
  pdl_wait();
  pdl_launch_dependents();
  // Warps take (32 buckets, part of the chunks), so that the loads of all are in flight.
  for (int e = threadIdx.x; e < 2 * buckets; e += kRouteThreads) base[e] = 0;
  __syncthreads();
  const int groups = (buckets + 31) / 32, parts = max(1, kRouteWarps / groups), chunks = (int)gridDim.x;
  for (int job = warp; job < groups * parts; job += kRouteWarps) {
    const int e = job % groups * 32 + lane, part = job / groups;
    const int c0 = part * chunks / parts, c1 = (part + 1) * chunks / parts;
    int all = 0, prior = 0;
    if (e < buckets) {
#pragma unroll 16
      for (int c = c0; c < c1; ++c) {
        const int v = __ldg(p.chunk_counts + (int64_t)c * buckets + e);
        all += v;
        prior += c < (int)blockIdx.x ? v : 0;
      }
      atomicAdd(base + e, all);  // whole numbers: the order does not matter
      atomicAdd(before + e, prior);
    }
  }
  __syncthreads();
  if (warp == 0) scan_counts(base, buckets, lane);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < buckets; i += kRouteThreads) p.offsets[i] = base[i];
  for (int e = threadIdx.x; e < buckets; e += kRouteThreads) before[e] += base[e];
  __syncthreads();
  place_chunk<kRouteThreads>(p, first, count, before, wcnt, warp, lane);
}

// Tokens of a chunk, one CTA: up to 32 tokens are one chunk and one launch; beyond that at most 128 chunks, so that
// each has an SM (a token's ranking is a chain of some 2000 clocks) and the placement sums few counts: 16384 tokens
// over 256 experts take 30 us, with 256 chunks of half the warps 35 (64 tokens in one chunk 13, in two 11).
int fb_route_chunk(int64_t tokens) {
  const int64_t per = (tokens + 127) / 128;
  return per < 32 ? 32 : (int)per;
}

cudaError_t launch_fb_route(const FbRouteParams& p, cudaStream_t stream) {
  const int chunks = (p.tokens + p.chunk - 1) / p.chunk, buckets = p.experts + 1;
  const int nv = (p.experts + 31) / 32, threads = route_threads(nv);
  const size_t smem = (size_t)buckets * (1 + threads / 32) * sizeof(int);
  const void* k = nv <= 2   ? (const void*)moe_route_kernel<2>
                  : nv <= 4 ? (const void*)moe_route_kernel<4>
                  : nv <= 8 ? (const void*)moe_route_kernel<8>
                  : nv <= 16 ? (const void*)moe_route_kernel<16>
                             : (const void*)moe_route_kernel<32>;
  cudaError_t e = ensure_smem_attribute(k, smem);
  if (e == cudaSuccess) e = launch_pdl(k, dim3(chunks), dim3(threads), smem, stream, p);
  if (e != cudaSuccess || chunks == 1) return e;
  const size_t place = (size_t)buckets * (2 + kPlaceThreads / 32) * sizeof(int);
  e = ensure_smem_attribute((const void*)moe_place_kernel, place);
  return e != cudaSuccess ? e : launch_pdl((const void*)moe_place_kernel, dim3(chunks), dim3(kPlaceThreads), place, stream, p);
}

// --------------------------------------------------------------------------
// out[t] = sum_j weights[t, j] * y[positions[t, j]], FP32 in the order of j,
// rounded once; a token without experts gets zeros.
// --------------------------------------------------------------------------
template <bool kIn16, bool kVec>
__global__ void __launch_bounds__(256) moe_combine_kernel(const __grid_constant__ FbCombineParams p) {
  const int t = blockIdx.y + blockIdx.z * 65535;
  if (t >= p.tokens) return;
  const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
  pdl_wait();
  pdl_launch_dependents();
  if (c >= p.h) return;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (int j = 0; j < p.top; ++j) {
    const int pos = __ldg(p.positions + (int64_t)t * p.top + j);
    if (pos < 0 || pos >= p.rows) continue;
    const float w = __ldg(p.weights + (int64_t)t * p.top + j);
    if constexpr (kIn16) {
      const uint16_t* y = (const uint16_t*)p.y + (int64_t)pos * p.ldy + c;
      if (kVec) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(y));
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[2 * i] = fmaf(w, __uint_as_float(u[i] << 16), acc[2 * i]);
          acc[2 * i + 1] = fmaf(w, __uint_as_float(u[i] & 0xFFFF0000u), acc[2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.h) acc[i] = fmaf(w, __uint_as_float((uint32_t)__ldg(y + i) << 16), acc[i]);
      }
    } else {
      const float* y = (const float*)p.y + (int64_t)pos * p.ldy + c;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (kVec || c + i < p.h) acc[i] = fmaf(w, __ldg(y + i), acc[i]);
    }
  }
  if (p.out_bf16) {
    __nv_bfloat16* o = (__nv_bfloat16*)p.out + (int64_t)t * p.ldo + c;
    if (kVec) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(acc[2 * i], acc[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(o) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < p.h) o[i] = __float2bfloat16_rn(acc[i]);
    }
  } else {
    float* o = (float*)p.out + (int64_t)t * p.ldo + c;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (kVec || c + i < p.h) o[i] = acc[i];
  }
}

cudaError_t launch_fb_combine(const FbCombineParams& p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.h + 2047) / 2048), (unsigned)(p.tokens < 65535 ? p.tokens : 65535),
                  (unsigned)((p.tokens + 65534) / 65535));
  const int ys = p.y_bf16 ? 2 : 4, os = p.out_bf16 ? 2 : 4;
  const bool vec = p.h % 8 == 0 && (uintptr_t)p.y % 16 == 0 && p.ldy * ys % 16 == 0 && (uintptr_t)p.out % 16 == 0 &&
                   p.ldo * os % 16 == 0;
  const void* k = p.y_bf16 ? (vec ? (const void*)moe_combine_kernel<true, true> : (const void*)moe_combine_kernel<true, false>)
                           : (vec ? (const void*)moe_combine_kernel<false, true> : (const void*)moe_combine_kernel<false, false>);
  return launch_pdl(k, grid, dim3(256), 0, stream, p);
}

}  // namespace mambo
