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
// Quantization, bound by the bytes it moves. A warp takes kSpan values of one
// row, kSteps loads in flight (a lane holds 8 values, a quad or 16 lanes a
// scale group), and finds the row's places once for all of them: one place in
// expert order (kFbGrouped), up to `top` when the row's token was routed, so
// that x is read once. 4096 x 28672 bf16 values take 75 us, 4.7 TB/s read and
// written (0.72 of the measured bandwidth); one step of 256 values a warp with
// the place found by every thread took 180 us under ncu where this takes 99.
// --------------------------------------------------------------------------
namespace {

constexpr int kSteps = 4, kSpan = 256 * kSteps;

}  // namespace

// One item's loads: a row's span, 8 values a lane and step.
template <int kIn, bool kVec>
__device__ __forceinline__ void quant_load(const FbQuantParams& p, int64_t row, int64_t c0, uint4 (&raw)[kSteps],
                                           uint4 (&raw2)[kIn == MAMBO_F32 ? kSteps : 1]) {
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int64_t k0 = (c0 + 32 * i) * 8;
    raw[i] = make_uint4(0, 0, 0, 0);
    if constexpr (kIn == MAMBO_F32) raw2[i] = make_uint4(0, 0, 0, 0);
    if (k0 >= p.k) continue;
    if constexpr (kIn == MAMBO_BF16) {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx + k0;
      if (kVec && k0 + 8 <= p.k) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < p.k) w[j >> 1] |= (uint32_t)__ldg(src + j) << (16 * (j & 1));
        raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else if constexpr (kIn == MAMBO_F32) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.x) + row * p.ldx + k0;
      if (kVec && k0 + 8 <= p.k) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(src));
        raw2[i] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
      } else {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = k0 + j < p.k ? __ldg(src + j) : 0u;
        raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
        raw2[i] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    } else {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.x) + row * p.ldx + k0;
      if (kVec && k0 + 8 <= p.k) {
        const uint2 t = __ldg(reinterpret_cast<const uint2*>(src));
        raw[i] = make_uint4(t.x, t.y, 0, 0);
      } else {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k0 + j < p.k) w[j >> 2] |= (uint32_t)__ldg(src + j) << (8 * (j & 3));
        raw[i] = make_uint4(w[0], w[1], 0, 0);
      }
    }
  }
}

template <int kIn, bool kVec>
__global__ void __launch_bounds__(256, 5) fb_quant_kernel(const __grid_constant__ FbQuantParams p) {
  const int lane = threadIdx.x & 31;
  const uint32_t spans = (uint32_t)((p.k + kSpan - 1) / kSpan);
  const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);  // the host keeps rows * spans below 2^31
  pdl_wait();
  pdl_launch_dependents();
  if (item >= (uint32_t)p.rows * spans) return;
  const uint32_t r32 = item / spans;
  const int64_t row = r32;
  const int c0 = (int)(item - r32 * spans) * (kSpan / 8) + lane;  // first 8-value chunk of the lane
  const int chunks = (int)((p.k + 127) / 128 * 16);               // whole K blocks
  uint4 raw[kSteps], raw2[kIn == MAMBO_F32 ? kSteps : 1];
  quant_load<kIn, kVec>(p, row, c0, raw, raw2);
  // The row's places.
  int copies = 1, expert = 0;
  FbDst dst;
  dst.row = nullptr;
  if (p.mode == kFbDense) {
    if (!p.values) dst = fb_dst(p.act, fb_place(0, (int)p.rows, 0, (int)row, p.act.nt));
  } else if (p.mode == kFbGrouped) {
    // The row's expert: how many segments end at or before it.
    for (int b = 0; b < p.experts; b += 32) {
      const int end = b + lane < p.experts ? __ldg(p.offsets + b + lane + 1) : 0x7FFFFFFF;
      expert += __popc(__ballot_sync(0xFFFFFFFFu, end <= row));
    }
    if (expert < p.experts) {
      const int o = clamp_offset(__ldg(p.offsets + expert), p.total_rows);
      const int end = clamp_offset(__ldg(p.offsets + expert + 1), p.total_rows);
      if (row >= o && end > o) dst = fb_dst(p.act, fb_place(o, end - o, expert, (int)row - o, p.act.nt));
    }
  } else {
    copies = p.top;
  }
  uint2 q[kSteps];
  uint32_t word[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if constexpr (kIn == kFbCodes) {
      q[i] = make_uint2(raw[i].x, raw[i].y);
      const int kb = (c0 + 32 * i) >> 4;
      const uint8_t* s = p.xs + row * p.lds;
      word[i] = 0;
      if (c0 + 32 * i < chunks) {
        if (p.group == 128) {
          word[i] = (uint32_t)__ldg(s + kb) * 0x01010101u;
        } else {
          const int64_t groups = (p.k + 31) / 32;
#pragma unroll
          for (int j = 0; j < 4; ++j) word[i] |= (uint32_t)(kb * 4 + j < groups ? __ldg(s + kb * 4 + j) : 127) << (8 * j);
        }
      }
    } else {
      if constexpr (kIn == MAMBO_BF16) {
        q[i] = quantize8(raw[i], p.group, lane, word[i]);
      } else {
        const float v[8] = {__uint_as_float(raw[i].x),  __uint_as_float(raw[i].y),  __uint_as_float(raw[i].z),
                            __uint_as_float(raw[i].w),  __uint_as_float(raw2[i].x), __uint_as_float(raw2[i].y),
                            __uint_as_float(raw2[i].z), __uint_as_float(raw2[i].w)};
        q[i] = quantize8(v, p.group, lane, word[i]);
      }
    }
  }
  if (p.mode == kFbDense && p.values) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int64_t c = c0 + 32 * i;
      if (c * 8 >= p.k) continue;
      uint8_t* d = p.values + row * p.ldv + c * 8;
      if (c * 8 + 8 <= p.k && (uintptr_t)d % 8 == 0) {
        *reinterpret_cast<uint2*>(d) = q[i];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c * 8 + j < p.k) d[j] = (uint8_t)((j < 4 ? q[i].x : q[i].y) >> (8 * (j & 3)));
      }
      if (p.group == 128) {
        if ((c & 15) == 0) p.scales[row * p.ldsc + (c >> 4)] = (uint8_t)word[i];
      } else if ((c & 3) == 0) {
        p.scales[row * p.ldsc + (c >> 2)] = (uint8_t)(word[i] >> (8 * ((c >> 2) & 3)));
      }
    }
    return;
  }
  for (int j = 0; j < copies; ++j) {
    if (p.mode == kFbRouted) {
      dst.row = nullptr;
      const int e = __ldg(p.ids + row * p.top + j);
      const int pos = __ldg(p.positions + row * p.top + j);
      if (e >= 0 && e < p.experts && pos >= 0 && pos < p.total_rows) {
        const int o = clamp_offset(__ldg(p.offsets + e), p.total_rows);
        const int end = clamp_offset(__ldg(p.offsets + e + 1), p.total_rows);
        if (pos >= o && pos < end) dst = fb_dst(p.act, fb_place(o, end - o, e, pos - o, p.act.nt));
      }
    }
    if (!dst.row) continue;
    // The lane's chunk of its K block is the same in every step, two blocks on.
    const uint32_t rec = fb_record_bytes(p.act.nt);
    const int64_t at = (int64_t)(c0 >> 4) * rec;
    uint8_t* d = dst.row + at + ((((c0 & 15) >> 1) ^ dst.swz) << 4) + (c0 & 1) * 8;
    uint8_t* sf = dst.sf + at;
    const bool first = (c0 & 15) == 0, pair = fb_is_pair(p.act.nt);
    const uint32_t other = fb_part_bytes(p.act.nt);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (c0 + 32 * i < chunks) {
        *reinterpret_cast<uint2*>(d) = q[i];
        if (first) {
          *reinterpret_cast<uint32_t*>(sf) = word[i];
          if (pair) *reinterpret_cast<uint32_t*>(sf + other) = word[i];  // both CTAs' parts
        }
      }
      d += 2 * rec;
      sf += 2 * rec;
    }
  }
}

cudaError_t launch_fb_quant(const FbQuantParams& p, cudaStream_t stream) {
  const int64_t items = p.rows * ((p.k + kSpan - 1) / kSpan);
  if (items >= (int64_t)1 << 31) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((items + 7) / 8));
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
