// Attention over the paged FP8 cache: a warp of a query row's four takes every fourth position; a running maximum and
// sum per warp, joined at the end.
#include <cuda_fp8.h>

#include "kernels.cuh"
#include "kv.cuh"

namespace mambo {

namespace {

__device__ __forceinline__ float e4m3_value(uint8_t c) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"((uint32_t)c));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}

__global__ void __launch_bounds__(128) kv_attention_simple_kernel(const __grid_constant__ KvAttentionCall p) {
  __shared__ float so[4][kKvMaxDim], sm[4], sl[4];
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvCache& cache = p.cache;
  pdl_wait();
  pdl_launch_dependents();
  int b = t, at = 0, count = 1;
  if (p.seq.offsets) {
    for (b = 0; b < p.seq.batch; ++b) {
      const KvSpan s = kv_span(p.seq, b);
      if (t >= s.first && t < s.first + s.count) {
        at = t - s.first;
        count = s.count;
        break;
      }
    }
    if (b == p.seq.batch) return;
  }
  if (count * p.group <= p.few) return;
  const int64_t place = (int64_t)kv_length(p.seq, b, cache.page) - count + at;
  const int64_t first = p.window ? max(place - p.window + 1, (int64_t)0) : 0;
  const int kv = h / p.group, dim = cache.dim;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < dim ? __uint_as_float((uint32_t)p.q[t * p.qs_t + h * p.qs_h + d] << 16) : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = first + warp; j <= place; j += 4) {
    const int64_t page = __ldg(p.seq.table + b * p.seq.table_stride + (j >> cache.log_page));
    if (page < 0 || page >= cache.pages) continue;
    const int64_t row = page * cache.heads + kv;
    const int64_t from = (row * cache.page + (j & (cache.page - 1))) * dim;
    const uint32_t kc = cache.scales[0][row], vc = cache.scales[1][row];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < dim) s = fmaf(q[i], e4m3_value(cache.codes[0][from + d]), s);
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, i);
    s *= p.scale * (kc == 255u ? NAN : e8m0_to_float(kc));
    const float top = fmaxf(m, s), f = expf(m - top), e = expf(s - top);
    m = top;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      if (d < dim) o[i] = fmaf(e, e4m3_value(cache.codes[1][from + d]) * (vc == 255u ? NAN : e8m0_to_float(vc)), o[i] * f);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) so[warp][lane + 32 * i] = o[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float total = 0.f, sum = 0.f;
  const int d = threadIdx.x;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (sl[w] == 0.f) continue;
    const float f = expf(sm[w] - top);
    total += sl[w] * f;
    sum += so[w][d] * f;
  }
  if (d < dim) {
    const __nv_bfloat16 v = __float2bfloat16_rn(total == 0.f ? 0.f : sum / total);
    p.out[t * p.os_t + h * p.os_h + d] = *reinterpret_cast<const uint16_t*>(&v);
  }
  if (p.lse && threadIdx.x == 0) p.lse[t * p.ls_t + h * p.ls_h] = total == 0.f ? -INFINITY : top + logf(total);
}

}  // namespace

cudaError_t launch_kv_attention_simple(const KvAttentionCall& p, cudaStream_t stream) {
  return launch_pdl((const void*)kv_attention_simple_kernel, dim3(p.seq.tokens, p.cache.heads * p.group), dim3(128), 0, stream, p);
}

}  // namespace mambo
