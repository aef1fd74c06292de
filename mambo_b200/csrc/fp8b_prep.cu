// Weight packing and activation quantization of the FP8 block-scaled linear
// (layouts in fp8b.cuh).
#include "fp8b.cuh"
#include "kernels.cuh"
#include "mxfp8.cuh"

namespace mambo {

// --------------------------------------------------------------------------
// Packing: one CTA per record, a thread per (row, 16-byte chunk). Run once per
// weight, so it takes any strides byte by byte.
// --------------------------------------------------------------------------
__global__ void __launch_bounds__(256) fb_pack_kernel(const FbPackParams p) {
  const int64_t rec = blockIdx.x;
  const int kb = (int)(rec % p.kblocks);
  const int rt = (int)(rec / p.kblocks % p.row_tiles);
  const int e = (int)(rec / p.kblocks / p.row_tiles);
  const uint8_t* w = p.w + e * p.stride_e;
  uint8_t* dst = p.packed + rec * kFbRecord;
  const int half = p.n / 2;
  for (int i = threadIdx.x; i < 1024; i += 256) {
    const int r = i >> 3, c = i & 7;
    int row;  // source row, or -1
    if (p.gate_up) {
      // Quarter q of tile rt: gate (q even) or up (q odd) of features 64*rt + 32*(q/2) ...
      const int q = r >> 5, f = 64 * rt + 32 * (q >> 1) + (r & 31);
      row = f < half ? f + (q & 1) * half : -1;
    } else {
      row = 128 * rt + r < p.n ? 128 * rt + r : -1;
    }
    uint32_t b[4] = {0, 0, 0, 0};
    if (row >= 0) {
      const uint8_t* src = w + row * p.stride_n;
      const int64_t k0 = (int64_t)kb * 128 + c * 16;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k0 + j < p.k) b[j >> 2] |= (uint32_t)__ldg(src + (k0 + j) * p.stride_k) << (8 * (j & 3));
    }
    *reinterpret_cast<uint4*>(dst + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(b[0], b[1], b[2], b[3]);
  }
  if (threadIdx.x < 2) {
    // Row block of the scale: gate blocks first, then up blocks, counted anew.
    const int blk = p.gate_up ? rt / 2 + (int)threadIdx.x * ((half + 127) / 128) : rt;
    p.scales[(((int64_t)e * p.row_tiles + rt) * 2 + threadIdx.x) * p.kblocks + kb] =
        __ldg(p.s + e * p.sstride_e + blk * p.sstride_n + kb * p.sstride_k);
  }
}

cudaError_t launch_fb_pack(const FbPackParams& p, cudaStream_t stream) {
  const int64_t records = (int64_t)p.experts * p.row_tiles * p.kblocks;
  fb_pack_kernel<<<(unsigned)records, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

// --------------------------------------------------------------------------
// Quantization: 8 values per thread (one 16-byte load of bf16), a quad (16
// lanes) per 32 (128) values, 2048 values of a row per CTA. Every row goes to
// each of its places: one in expert order (kFbGrouped), up to `top` when its
// token was routed, so that x is read once.
// --------------------------------------------------------------------------
template <int kIn, bool kVec>
__global__ void __launch_bounds__(256) fb_quant_kernel(const __grid_constant__ FbQuantParams p) {
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= p.rows) return;
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;  // 8-value chunk of the row
  const int64_t chunks = (p.k + 127) / 128 * 16;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  // Whole 16-lane groups are in range together (chunks is a multiple of 16).
  const bool in = c < chunks;
  uint2 q = make_uint2(0, 0);
  uint32_t word = 0;
  if (kIn == kFbCodes) {
    if (in) {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.x) + row * p.ldx + c * 8;
      if (kVec && c * 8 + 8 <= p.k) {
        q = __ldg(reinterpret_cast<const uint2*>(src));
      } else {
        uint32_t b[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c * 8 + i < p.k) b[i >> 2] |= (uint32_t)__ldg(src + i) << (8 * (i & 3));
        q = make_uint2(b[0], b[1]);
      }
      const uint8_t* s = p.xs + row * p.lds;
      if (p.group == 128) {
        word = (uint32_t)__ldg(s + (c >> 4)) * 0x01010101u;
      } else {
        const int64_t g0 = (c >> 4) * 4, groups = (p.k + 31) / 32;
#pragma unroll
        for (int j = 0; j < 4; ++j) word |= (uint32_t)(g0 + j < groups ? __ldg(s + g0 + j) : 127) << (8 * j);
      }
    }
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (in) {
      if constexpr (kIn == MAMBO_BF16) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx + c * 8;
        if (kVec && c * 8 + 8 <= p.k) {
          const uint4 raw = __ldg(reinterpret_cast<const uint4*>(src));
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c * 8 + i < p.k) v[i] = __uint_as_float((uint32_t)__ldg(src + i) << 16);
        }
      } else {
        const float* src = reinterpret_cast<const float*>(p.x) + row * p.ldx + c * 8;
        if (kVec && c * 8 + 8 <= p.k) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(src));
          const float4 b = __ldg(reinterpret_cast<const float4*>(src) + 1);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
          v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c * 8 + i < p.k) v[i] = __ldg(src + i);
        }
      }
    }
    // Largest magnitude as bits: NaN orders above infinity, so either gives the group the code 0xFF.
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    if (p.group == 128) {
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
    q = make_uint2(packed[0], packed[1]);
    word = code << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
  }
  // Grouped: the row's expert, by whole warps: how many segments end at or before it.
  int expert = 0;
  if (p.mode == kFbGrouped) {
    for (int b = 0; b < p.experts; b += 32) {
      const int end = b + lane < p.experts ? __ldg(p.offsets + b + lane + 1) : 0x7FFFFFFF;
      expert += __popc(__ballot_sync(0xFFFFFFFFu, end <= row));
    }
  }
  if (!in) return;
  if (p.mode == kFbDense) {
    if (p.values) {
      uint8_t* d = p.values + row * p.ldv + c * 8;
      if (c * 8 + 8 <= p.k && (uintptr_t)d % 8 == 0) {
        *reinterpret_cast<uint2*>(d) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c * 8 + i < p.k) d[i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
      }
      if (p.group == 128) {
        if ((c & 15) == 0) p.scales[row * p.ldsc + (c >> 4)] = (uint8_t)word;
      } else if ((c & 3) == 0 && c * 8 < p.k) {
        p.scales[row * p.ldsc + (c >> 2)] = (uint8_t)(word >> (8 * ((c >> 2) & 3)));
      }
      return;
    }
    fb_store(p.act, fb_place(0, (int)p.rows, 0, (int)row, p.act.nt), c, q, word);
  } else if (p.mode == kFbGrouped) {
    const int e = expert;
    if (e >= p.experts) return;  // past the last segment
    const int o = clamp_offset(__ldg(p.offsets + e), p.total_rows);
    const int end = clamp_offset(__ldg(p.offsets + e + 1), p.total_rows);
    const int local = (int)row - o;
    if (local < 0 || end <= o) return;
    fb_store(p.act, fb_place(o, end - o, e, local, p.act.nt), c, q, word);
  } else {
    for (int j = 0; j < p.top; ++j) {
      const int e = __ldg(p.ids + row * p.top + j);
      const int pos = __ldg(p.positions + row * p.top + j);
      if (e < 0 || e >= p.experts || pos < 0 || pos >= p.total_rows) continue;
      const int o = clamp_offset(__ldg(p.offsets + e), p.total_rows);
      const int end = clamp_offset(__ldg(p.offsets + e + 1), p.total_rows);
      if (pos < o || pos >= end) continue;
      fb_store(p.act, fb_place(o, end - o, e, pos - o, p.act.nt), c, q, word);
    }
  }
}

cudaError_t launch_fb_quant(const FbQuantParams& p, cudaStream_t stream) {
  const int64_t chunks = (p.k + 127) / 128 * 16;
  const dim3 grid((unsigned)((chunks + 255) / 256), (unsigned)(p.rows < 65535 ? p.rows : 65535),
                  (unsigned)((p.rows + 65534) / 65535));
  const int esize = p.x_kind == MAMBO_F32 ? 4 : p.x_kind == MAMBO_BF16 ? 2 : 1;
  const int align = p.x_kind == kFbCodes ? 8 : 16;
  const bool vec = (uintptr_t)p.x % align == 0 && (p.ldx * esize) % align == 0;
  const void* k;
  if (p.x_kind == MAMBO_BF16)
    k = vec ? (const void*)fb_quant_kernel<MAMBO_BF16, true> : (const void*)fb_quant_kernel<MAMBO_BF16, false>;
  else if (p.x_kind == MAMBO_F32)
    k = vec ? (const void*)fb_quant_kernel<MAMBO_F32, true> : (const void*)fb_quant_kernel<MAMBO_F32, false>;
  else
    k = vec ? (const void*)fb_quant_kernel<kFbCodes, true> : (const void*)fb_quant_kernel<kFbCodes, false>;
  return launch_pdl(k, grid, dim3(256), 0, stream, p);
}

}  // namespace mambo
