// Rotary positions, and the append of keys and values to the paged FP8 cache.
//
// Both are bound by memory: each value is read once and written once. The
// rotation's angle is position * frequency as a 64-bit fraction of a turn, an
// integer product that drops whole turns exactly, so that a position of 2^20
// is as precise as the first; its cosine and sine are the Taylor polynomials
// on an eighth of a turn to either side (below). A cosine and sine serve
// several heads of the token where there is enough to do.
#include "kernels.cuh"
#include "kv.cuh"
#include "mxfp8.cuh"

namespace mambo {

namespace {

// cos and sin of phase / 2^64 turns. The nearest quarter turn is split off; on the rest, |x| <= pi/4, the Taylor
// polynomials to x^9 and x^8 are off by less than 2^-25.
__device__ __forceinline__ void turn_cos_sin(uint64_t phase, float& c, float& s) {
  const uint32_t t = (uint32_t)(phase >> 32);
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float p = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);  // 1/9!, -1/7!
  p = fmaf(z, p, 8.3333333e-3f);
  p = fmaf(z, p, -1.6666667e-1f);
  const float sine = fmaf(x * z, p, x);
  float r = fmaf(z, 2.4801587e-5f, -1.3888889e-3f);  // 1/8!, -1/6!
  r = fmaf(z, r, 4.1666667e-2f);
  r = fmaf(z, r, -0.5f);
  const float cosine = fmaf(z, r, 1.0f);
  const float a = quarter & 1 ? sine : cosine, b = quarter & 1 ? cosine : sine;
  c = (quarter + 1) & 2 ? -a : a;
  s = quarter & 2 ? -b : b;
}

// Where the 16 dimensions of a unit lie in a head. Interleaved pairs: dimensions a .. a+15, of which the first `turned`
// pairs turn. Halves: dimensions a .. a+7 and b .. b+7, `turned` pairs; behind the rotated part a .. a+15, unchanged.
// n: valid dimensions from a on (adjacent units).
struct RotaryUnit {
  int a, b, n, turned;
  bool adjacent;
};
__host__ __device__ __forceinline__ int rotary_units(const RotaryParams& r, int dim) {
  const int pairs = r.turns ? r.pairs : 0;
  return r.interleaved ? (dim + 15) / 16 : (pairs + 7) / 8 + (dim - 2 * pairs + 15) / 16;
}
__device__ __forceinline__ RotaryUnit rotary_unit(const RotaryParams& r, int dim, int u) {
  RotaryUnit v;
  const int pairs = r.turns ? r.pairs : 0, first = r.interleaved ? 0 : (pairs + 7) / 8;
  v.adjacent = u >= first;
  if (v.adjacent) {
    v.a = (r.interleaved ? 0 : 2 * pairs) + 16 * (u - first);
    v.b = v.a + 8;
    v.n = min(16, dim - v.a);
    v.turned = r.interleaved ? max(min(8, pairs - 8 * u), 0) : 0;
  } else {
    v.a = 8 * u;
    v.b = pairs + 8 * u;
    v.n = 0;
    v.turned = min(8, pairs - 8 * u);
  }
  return v;
}

// 16 values of a unit: lo[i] at a + i, hi[i] at b + i. Vectors where everything is a multiple of 8 elements and 16 bytes.
template <bool kVec, bool k16>
__device__ __forceinline__ void unit_load(const void* x, int64_t at, const RotaryUnit& u, float (&lo)[8], float (&hi)[8]) {
  if constexpr (kVec && k16) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + at;
    const uint4 l = __ldg(reinterpret_cast<const uint4*>(p + u.a)), h = __ldg(reinterpret_cast<const uint4*>(p + u.b));
    const uint32_t lw[4] = {l.x, l.y, l.z, l.w}, hw[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[2 * i] = __uint_as_float(lw[i] << 16);
      lo[2 * i + 1] = __uint_as_float(lw[i] & 0xFFFF0000u);
      hi[2 * i] = __uint_as_float(hw[i] << 16);
      hi[2 * i + 1] = __uint_as_float(hw[i] & 0xFFFF0000u);
    }
  } else if constexpr (kVec) {
    const float* p = reinterpret_cast<const float*>(x) + at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 l = __ldg(reinterpret_cast<const float4*>(p + u.a) + i), h = __ldg(reinterpret_cast<const float4*>(p + u.b) + i);
      lo[4 * i] = l.x, lo[4 * i + 1] = l.y, lo[4 * i + 2] = l.z, lo[4 * i + 3] = l.w;
      hi[4 * i] = h.x, hi[4 * i + 1] = h.y, hi[4 * i + 2] = h.z, hi[4 * i + 3] = h.w;
    }
  } else {
    auto one = [&](int d) {
      if constexpr (k16) return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(x) + at + d) << 16);
      return __ldg(reinterpret_cast<const float*>(x) + at + d);
    };
    const int n0 = u.adjacent ? u.n : u.turned, n1 = u.adjacent ? u.n - 8 : u.turned;  // values from a and from b on
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = i < n0 ? one(u.a + i) : 0.f;
      hi[i] = i < n1 ? one(u.b + i) : 0.f;
    }
  }
}

// A unit's values as they come: 16 bf16, or 16 floats.
template <bool kVec, bool k16>
struct RawUnit {
  static constexpr bool kPacked = kVec && k16;
  uint4 w[kPacked ? 2 : 4];
  __device__ __forceinline__ void load(const void* x, int64_t at, const RotaryUnit& u) {
    if constexpr (kPacked) {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + at;
      w[0] = __ldg(reinterpret_cast<const uint4*>(p + u.a));
      w[1] = __ldg(reinterpret_cast<const uint4*>(p + u.b));
    } else {
      float lo[8], hi[8];
      unit_load<kVec, k16>(x, at, u, lo, hi);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = make_uint4(__float_as_uint(lo[4 * i]), __float_as_uint(lo[4 * i + 1]), __float_as_uint(lo[4 * i + 2]), __float_as_uint(lo[4 * i + 3]));
        w[2 + i] = make_uint4(__float_as_uint(hi[4 * i]), __float_as_uint(hi[4 * i + 1]), __float_as_uint(hi[4 * i + 2]), __float_as_uint(hi[4 * i + 3]));
      }
    }
  }
  __device__ __forceinline__ void get(float (&lo)[8], float (&hi)[8]) const {
    if constexpr (kPacked) {
      const uint32_t l[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, h[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[2 * i] = __uint_as_float(l[i] << 16);
        lo[2 * i + 1] = __uint_as_float(l[i] & 0xFFFF0000u);
        hi[2 * i] = __uint_as_float(h[i] << 16);
        hi[2 * i + 1] = __uint_as_float(h[i] & 0xFFFF0000u);
      }
    } else {
      const uint32_t* f = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = __uint_as_float(f[i]);
        hi[i] = __uint_as_float(f[8 + i]);
      }
    }
  }
};
// cos and sin of the unit's pairs, times the magnitude; 1 and 0 for those that do not turn.
__device__ __forceinline__ void unit_angles(const RotaryParams& r, const RotaryUnit& u, int pair0, int64_t position,
                                            float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool turns = i < u.turned;
    const uint64_t f = turns ? __ldg(reinterpret_cast<const unsigned long long*>(r.turns) + pair0 + i) : 0ull;
    turn_cos_sin((uint64_t)position * f, c[i], s[i]);  // of nothing: 1 and 0
    c[i] *= turns ? r.magnitude : 1.f;
    s[i] *= r.magnitude * r.sign;
  }
}
__device__ __forceinline__ void unit_turn(bool interleaved, const float (&c)[8], const float (&s)[8], float (&lo)[8],
                                          float (&hi)[8]) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = lo[2 * i], b = lo[2 * i + 1], d = hi[2 * i], e = hi[2 * i + 1];
      lo[2 * i] = fmaf(a, c[i], -b * s[i]);
      lo[2 * i + 1] = fmaf(a, s[i], b * c[i]);
      hi[2 * i] = fmaf(d, c[4 + i], -e * s[4 + i]);
      hi[2 * i + 1] = fmaf(d, s[4 + i], e * c[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = lo[i], b = hi[i];
      lo[i] = fmaf(a, c[i], -b * s[i]);
      hi[i] = fmaf(a, s[i], b * c[i]);
    }
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

template <bool kVec, bool k16>
__device__ __forceinline__ void unit_store(void* out, int64_t at, const RotaryUnit& u, const float (&lo)[8],
                                           const float (&hi)[8]) {
  if constexpr (kVec && k16) {
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + at;
    *reinterpret_cast<uint4*>(p + u.a) =
        make_uint4(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]), pack_bf16(lo[4], lo[5]), pack_bf16(lo[6], lo[7]));
    *reinterpret_cast<uint4*>(p + u.b) =
        make_uint4(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]), pack_bf16(hi[4], hi[5]), pack_bf16(hi[6], hi[7]));
  } else if constexpr (kVec) {
    float* p = reinterpret_cast<float*>(out) + at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      reinterpret_cast<float4*>(p + u.a)[i] = make_float4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
      reinterpret_cast<float4*>(p + u.b)[i] = make_float4(hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
    }
  } else {
    auto one = [&](int d, float v) {
      if constexpr (k16) reinterpret_cast<__nv_bfloat16*>(out)[at + d] = __float2bfloat16_rn(v);
      else reinterpret_cast<float*>(out)[at + d] = v;
    };
    const int n0 = u.adjacent ? u.n : u.turned, n1 = u.adjacent ? u.n - 8 : u.turned;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < n0) one(u.a + i, lo[i]);
      if (i < n1) one(u.b + i, hi[i]);
    }
  }
}

// A unit's angles need its first pair's number: 8 per rotated unit.
template <bool kVec, bool k16, int kPer>
__global__ void __launch_bounds__(256, kPer == 4 && kVec && k16 ? 3 : 1) rotary_kernel(const __grid_constant__ RotaryCall p) {
  const int64_t job = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_token = p.units * p.groups;
  const int64_t token = job / per_token;
  pdl_wait();
  pdl_launch_dependents();
  if (token >= p.tokens) return;
  const int in = (int)(job - token * per_token), g = in / p.units, unit = in - g * p.units;
  const RotaryUnit u = rotary_unit(p.rot, p.dim, unit);
  RawUnit<kVec, k16> raw[kPer];
  const int64_t from = token * p.xs_t, to = token * p.os_t;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int h = g + i * p.groups;
    if (h < p.heads) raw[i].load(p.x, from + h * p.xs_h, u);
  }
  float c[8], s[8];
  const bool turns = u.turned > 0;
  if (turns) {
    const int64_t position = p.positions64 ? __ldg(reinterpret_cast<const long long*>(p.positions) + token)
                                           : (int64_t)__ldg(reinterpret_cast<const int*>(p.positions) + token);
    unit_angles(p.rot, u, 8 * unit, position, c, s);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int h = g + i * p.groups;
    if (h < p.heads) {
      float lo[8], hi[8];
      raw[i].get(lo, hi);
      if (turns) unit_turn(p.rot.interleaved, c, s, lo, hi);
      unit_store<kVec, k16>(p.out, to + h * p.os_h, u, lo, hi);
    }
  }
}

template <bool kVec, bool k16>
const void* rotary_variant(int per) {
  return per == 4 ? (const void*)rotary_kernel<kVec, k16, 4> : per == 2 ? (const void*)rotary_kernel<kVec, k16, 2>
                                                                        : (const void*)rotary_kernel<kVec, k16, 1>;
}

// ---------------------------------------------------------------------------
// Append. A CTA has one page and its keys or its values of some heads, one
// after the other: it takes the head's new values into registers (turned),
// finds their largest magnitude, decides the page's scale, rescales what the
// page already holds where the scale has grown, and writes the codes. One pass
// over the input. A thread has the same tokens and dimensions in every head,
// so that it keeps their cosines and sines; the next head's values are on
// their way while one is quantized.
// ---------------------------------------------------------------------------
// Units of a thread: one in the vector form, which keeps its registers at 64 (a page of 64 tokens with two units a thread
// and 128 registers took 42 us for 16384 tokens).
template <bool kVec>
constexpr int kAppendPasses = kVec ? 1 : 2;
template <bool kVec>
constexpr int kAppendThreads = kVec ? 1024 : 640;  // most, of a CTA: 128 tokens x 8 units, or 9 where the rotated part ends inside one

// mxfp8_scale_code from a magnitude's bits, without branches; of zero 0.
__device__ __forceinline__ uint32_t f32_scale_code(uint32_t bits) {
  const int biased = (int)(bits >> 23), code = max(biased - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7), 0);
  return biased == 255 ? 255u : (uint32_t)code;
}
// The larger magnitude of three, NaN if any is.
__device__ __forceinline__ float absmax3(float m, float a, float b) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return cvt_e4m3x2_rn(a, b) | (cvt_e4m3x2_rn(c, d) << 16);
}
// Two E4M3 codes times f, rounded to E4M3 again.
__device__ __forceinline__ uint32_t rescale_e4m3x2(uint32_t codes, float f) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(codes & 0xFFFFu));
  const __half2 v = *reinterpret_cast<const __half2*>(&h);
  return cvt_e4m3x2_rn(__low2float(v) * f, __high2float(v) * f);
}

// The first slot of sequence b: sequences b and b + 1 are offsets[b+1] / page - offsets[b] / page + 2 slots apart, and
// n tokens touch at most n / page + 2 pages.
__device__ __forceinline__ int append_slot(const KvSequences& s, int b, int log_page) {
  const int o = min(max(__ldg(s.offsets + b), 0), s.tokens);
  return (o >> log_page) + 2 * b;
}

template <bool kVec, bool k16>
__global__ void __launch_bounds__(kAppendThreads<kVec>) kv_append_kernel(const __grid_constant__ KvAppendCall p) {
  __shared__ float sm_max[2][32];
  const int which = blockIdx.z, threads = blockDim.x;
  const KvCache& cache = p.cache;
  const int page = cache.page, dim = cache.dim;
  const int head0 = blockIdx.y * p.heads_each, head1 = min(head0 + p.heads_each, cache.heads);
  pdl_wait();
  pdl_launch_dependents();
  int b = blockIdx.x, at = 0;
  if (p.seq.offsets) {
    // The last sequence whose first slot is at most this one's: 32 at a time.
    const int lane = threadIdx.x & 31, slot = blockIdx.x;
    int lo = 0, hi = p.seq.batch;  // in [lo, hi)
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, mine = lo + lane * step;
      const bool before = mine < hi && append_slot(p.seq, mine, cache.log_page) <= slot;
      const int n = max(1, __popc(__ballot_sync(0xFFFFFFFFu, before)));
      const int next = lo + (n - 1) * step;
      hi = min(hi, next + step);
      lo = next;
    }
    b = lo;
    at = slot - append_slot(p.seq, b, cache.log_page);
  }
  const KvSpan span = kv_span(p.seq, b);
  const int64_t past = kv_length(p.seq, b, page), block = (past >> cache.log_page) + at;
  const int64_t t0 = max(past, block << cache.log_page), t1 = min(past + span.count, (block + 1) << cache.log_page);
  if (at < 0 || t0 >= t1 || block >= p.seq.table_pages) return;
  const int64_t where = __ldg(p.seq.table + b * p.seq.table_stride + block);
  const int begun = (int)(t0 & (page - 1)), count = (int)(t1 - t0);  // tokens before the call's, and the call's

  RotaryParams rot = p.rot;
  if (which == 1) rot = RotaryParams{nullptr, 0, 0, 1.f, 1.f};
  const int units = rotary_units(rot, dim), all = count * units;
  const int64_t xs_h = p.xs_h[which];
  constexpr int kPasses = kAppendPasses<kVec>;
  constexpr bool kAhead = kVec && k16;  // the other forms have no registers for it
  int64_t from[kPasses];  // this thread's tokens: in the input, and their codes in the page
  int to[kPasses];
  RotaryUnit u[kPasses];
  float c[kPasses][8], s[kPasses][8];
  RawUnit<kVec, k16> raw[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int f = threadIdx.x + i * threads;
    if (f < all) {
      const int row = f / units, unit = f - row * units;
      u[i] = rotary_unit(rot, dim, unit);
      from[i] = (span.first + (t0 - past) + row) * p.xs_t[which];
      to[i] = (begun + row) * dim;
      if constexpr (kAhead) raw[i].load(p.x[which], from[i] + head0 * xs_h, u[i]);
      if (u[i].turned > 0) unit_angles(rot, u[i], 8 * unit, t0 + row, c[i], s[i]);
    }
  }
  if (where < 0 || where >= cache.pages) return;  // (after the values' loads, which do not wait for the page)
  uint8_t* scale_at = cache.scales[which] + where * cache.heads + head0;
  uint8_t* codes = cache.codes[which] + (where * cache.heads + head0) * (int64_t)(page * dim);
  const int lane = threadIdx.x & 31, warps = threads / 32;
  for (int head = head0; head < head1; ++head, ++scale_at, codes += page * dim) {
    const uint32_t old = begun ? *scale_at : 0u;
    float lo[kPasses][8], hi[kPasses][8];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if ((int)threadIdx.x + i * threads < all) {
        if constexpr (!kAhead) raw[i].load(p.x[which], from[i] + head * xs_h, u[i]);
        raw[i].get(lo[i], hi[i]);
        if constexpr (kAhead) {
          if (head + 1 < head1) raw[i].load(p.x[which], from[i] + (head + 1) * xs_h, u[i]);
        }
        if (u[i].turned > 0) unit_turn(rot.interleaved, c[i], s[i], lo[i], hi[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = absmax3(top, lo[i][j], hi[i][j]);
      }
    }
    // As integers: NaN and infinity order above every number.
    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top) & 0x7FFFFFFFu);
    float* maxima = sm_max[head & 1];
    if (lane == 0) maxima[threadIdx.x >> 5] = __uint_as_float(most);
    __syncthreads();
    const uint32_t bits = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? __float_as_uint(maxima[lane]) : 0u);
    // 255 stays; zero takes the smallest scale.
    const uint32_t code = max(max(f32_scale_code(bits), kKvMinCode), old);
    if (begun && code > old && code != 255u) {
      const int d = (int)old - (int)code;  // < 0
      const float f = d < -126 ? 0.f : __uint_as_float((uint32_t)(127 + d) << 23);
      for (int i = threadIdx.x; i < begun * dim / 16; i += threads) {
        uint4 v = reinterpret_cast<uint4*>(codes)[i];
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = rescale_e4m3x2(w[j], f) | (rescale_e4m3x2(w[j] >> 16, f) << 16);
        reinterpret_cast<uint4*>(codes)[i] = v;
      }
    }
    const float inv = code == 255u ? 0.f : e8m0_to_float(254u - code);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int f = threadIdx.x + i * threads;
      if (f < all) {
        uint8_t* at = codes + to[i];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w[j] = e4m3x4(lo[i][4 * j] * inv, lo[i][4 * j + 1] * inv, lo[i][4 * j + 2] * inv, lo[i][4 * j + 3] * inv);
          w[2 + j] = e4m3x4(hi[i][4 * j] * inv, hi[i][4 * j + 1] * inv, hi[i][4 * j + 2] * inv, hi[i][4 * j + 3] * inv);
        }
        if (code == 255u) w[0] = w[1] = w[2] = w[3] = 0u;  // zero times NaN has a code of its own
        if constexpr (kVec) {
          *reinterpret_cast<uint2*>(at + u[i].a) = make_uint2(w[0], w[1]);
          *reinterpret_cast<uint2*>(at + u[i].b) = make_uint2(w[2], w[3]);
        } else {
          const int n0 = u[i].adjacent ? u[i].n : u[i].turned, n1 = u[i].adjacent ? u[i].n - 8 : u[i].turned;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j < n0) at[u[i].a + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
            if (j < n1) at[u[i].b + j] = (uint8_t)(w[2 + (j >> 2)] >> (8 * (j & 3)));
          }
        }
      }
    }
    if (threadIdx.x == 0) *scale_at = (uint8_t)code;
  }
}

}  // namespace

cudaError_t launch_rotary(RotaryCall p, cudaStream_t stream) {
  const int es = p.bf16 ? 2 : 4;
  p.units = rotary_units(p.rot, p.dim);
  const bool vec = p.dim % 16 == 0 && (p.rot.interleaved || p.rot.pairs % 8 == 0) && (uintptr_t)p.x % 16 == 0 &&
                   (uintptr_t)p.out % 16 == 0 && p.xs_t * es % 16 == 0 && p.xs_h * es % 16 == 0 && p.os_t * es % 16 == 0 &&
                   p.os_h * es % 16 == 0;
  const int64_t head_units = (int64_t)p.tokens * p.heads * p.units;
  // Heads of a thread, which share its cosines and sines: four or two where that leaves 512 threads an SM.
  const int per = head_units >= 4 * 148 * 512 ? 4 : head_units >= 2 * 148 * 512 ? 2 : 1;
  p.groups = (p.heads + per - 1) / per;
  const int64_t jobs = (int64_t)p.tokens * p.groups * p.units;
  const void* k = p.bf16 ? (vec ? rotary_variant<true, true>(per) : rotary_variant<false, true>(per))
                         : (vec ? rotary_variant<true, false>(per) : rotary_variant<false, false>(per));
  return launch_pdl(k, dim3((unsigned)((jobs + 255) / 256)), dim3(256), 0, stream, p);
}

cudaError_t launch_kv_append(KvAppendCall p, cudaStream_t stream) {
  const int es = p.bf16 ? 2 : 4;
  bool vec = !p.rot.turns || p.rot.interleaved || p.rot.pairs % 8 == 0;
  for (int i = 0; i < 2; ++i)
    vec = vec && (uintptr_t)p.x[i] % 16 == 0 && p.xs_t[i] * es % 16 == 0 && p.xs_h[i] * es % 16 == 0;
  const int slots = p.seq.offsets ? (p.seq.tokens >> p.cache.log_page) + 2 * p.seq.batch : p.seq.batch;
  // One token a sequence is at most 9 units and needs a warp.
  const int units = max(rotary_units(p.rot, p.cache.dim), (p.cache.dim + 15) / 16), page_units = p.cache.page * units;
  const int threads = !p.seq.offsets ? 32 : ((vec ? page_units : (page_units + 1) / 2) + 31) / 32 * 32;
  // Heads of a CTA: as many as leave six CTAs an SM.
  p.heads_each = max(1, min(p.cache.heads, (int)((int64_t)slots * p.cache.heads * 2 / (148 * 6))));
  const unsigned groups = (unsigned)((p.cache.heads + p.heads_each - 1) / p.heads_each);
  const void* k = p.bf16 ? (vec ? (const void*)kv_append_kernel<true, true> : (const void*)kv_append_kernel<false, true>)
                         : (vec ? (const void*)kv_append_kernel<true, false> : (const void*)kv_append_kernel<false, false>);
  return launch_pdl(k, dim3((unsigned)slots, groups, 2), dim3(threads), 0, stream, p);
}

}  // namespace mambo
