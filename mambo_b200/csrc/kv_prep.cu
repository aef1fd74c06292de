// Rotary positions, and the append of keys and values to the paged FP8 cache.
//
// Both are bound by memory: each value is read once and written once. The
// rotation's angle is position * frequency as a 64-bit fraction of a turn, an
// integer product that drops whole turns exactly, so that a position of 2^20
// is as precise as the first; its cosine and sine are the Taylor polynomials
// on an eighth of a turn to either side (below). A cosine and sine serve
// several heads of the token where there is enough to do. 8192 tokens x 32
// heads of 128 in bf16: 23.5 us, 0.87 of a measured copy. Append of 17059
// tokens x 8 heads of 128: 28 us, 0.57 of a copy's rate: 260 instructions a
// unit of 16 values for the turn, the largest magnitude and the conversions.
#include "kernels.cuh"
#include "kv.cuh"
#include "mxfp8.cuh"

#include <type_traits>

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
struct RotaryUnit {
  int a, b, turned;
};
__host__ __device__ __forceinline__ int rotary_units(const RotaryParams& r, int dim) {
  const int pairs = r.turns ? r.pairs : 0;
  return r.interleaved ? (dim + 15) / 16 : (pairs + 7) / 8 + (dim - 2 * pairs + 15) / 16;
}
__device__ __forceinline__ RotaryUnit rotary_unit(const RotaryParams& r, int u) {
  RotaryUnit v;
  const int pairs = r.turns ? r.pairs : 0, first = r.interleaved ? 0 : (pairs + 7) / 8;
  if (u >= first) {
    v.a = (r.interleaved ? 0 : 2 * pairs) + 16 * (u - first);
    v.b = v.a + 8;
    v.turned = r.interleaved ? max(min(8, pairs - 8 * u), 0) : 0;
  } else {
    v.a = 8 * u;
    v.b = pairs + 8 * u;
    v.turned = min(8, pairs - 8 * u);
  }
  return v;
}

// The 16 values of a unit as they come: eight from a on, eight from b on. Everything is a multiple of 8 elements and 16 bytes.
template <bool k16>
struct RawUnit {
  uint4 w[k16 ? 2 : 4];
  __device__ __forceinline__ void load(const void* x, int64_t at, const RotaryUnit& u) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(x) + at * (k16 ? 2 : 4);
    constexpr int kHalf = k16 ? 1 : 2;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      w[i] = __ldg(reinterpret_cast<const uint4*>(p + u.a * (k16 ? 2 : 4)) + i);
      w[kHalf + i] = __ldg(reinterpret_cast<const uint4*>(p + u.b * (k16 ? 2 : 4)) + i);
    }
  }
  __device__ __forceinline__ void get(float (&lo)[8], float (&hi)[8]) const {
    if constexpr (k16) {
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
// A pair of values of a row that is not made of aligned vectors: pairs that turn, then neighbours that do not.
struct RotaryPair {
  int a, b;
  bool turns, halves;
};
__host__ __device__ __forceinline__ int rotary_pairs(const RotaryParams& r, int dim) {
  const int pairs = r.turns ? r.pairs : 0;
  return r.interleaved ? (dim + 1) / 2 : pairs + (dim - 2 * pairs + 1) / 2;
}
__device__ __forceinline__ RotaryPair rotary_pair(const RotaryParams& r, int i) {
  const int pairs = r.turns ? r.pairs : 0;
  RotaryPair v;
  v.turns = i < pairs;
  v.halves = v.turns && !r.interleaved;
  v.a = v.halves ? i : r.interleaved ? 2 * i : 2 * pairs + 2 * (i - pairs);
  v.b = v.halves ? i + pairs : v.a + 1;
  return v;
}
template <bool k16>
__device__ __forceinline__ float one_value(const void* x, int64_t at) {
  if constexpr (k16) return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(x) + at) << 16);
  else return __ldg(reinterpret_cast<const float*>(x) + at);
}
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

// The words of the pairs that turn (all eight, or the first of an interleaved unit's, whose pair i is word i in 16 bits and
// words 2 i and 2 i + 1 in 32) from lo and hi, the others as they came: bit for bit, whatever their neighbours are.
template <bool k16>
__device__ __forceinline__ void unit_store(void* out, int64_t at, const RotaryUnit& u, const RawUnit<k16>& raw,
                                           const float (&lo)[8], const float (&hi)[8]) {
  constexpr int kWords = k16 ? 8 : 16, kHalf = kWords / 8;
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const float* v = i < kWords / 2 ? lo : hi;
    const int k = i % (kWords / 2);
    w[i] = k16 ? pack_bf16(v[(2 * k) % 8], v[(2 * k + 1) % 8]) : __float_as_uint(v[k]);
  }
  if (u.turned < 8) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(raw.w);
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = i / kHalf < u.turned ? w[i] : r[i];
  }
  uint8_t* p = reinterpret_cast<uint8_t*>(out) + at * (k16 ? 2 : 4);
#pragma unroll
  for (int i = 0; i < kHalf; ++i) {
    const int j = 4 * i, k = 4 * (kHalf + i);
    reinterpret_cast<uint4*>(p + u.a * (k16 ? 2 : 4))[i] = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
    reinterpret_cast<uint4*>(p + u.b * (k16 ? 2 : 4))[i] = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
  }
}

// A unit's angles need its first pair's number: 8 per rotated unit.
template <bool k16, int kPer>
__global__ void __launch_bounds__(256, kPer == 4 && k16 ? 3 : 1) rotary_kernel(const __grid_constant__ RotaryCall p) {
  const int64_t job = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_token = p.units * p.groups;
  const int64_t token = job / per_token;
  pdl_wait();
  pdl_launch_dependents();
  if (token >= p.tokens) return;
  const int in = (int)(job - token * per_token), g = in / p.units, unit = in - g * p.units;
  const RotaryUnit u = rotary_unit(p.rot, unit);
  RawUnit<k16> raw[kPer];
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
      unit_store<k16>(p.out, to + h * p.os_h, u, raw[i], lo, hi);
    }
  }
}

// The same where rows are not made of aligned vectors (a half of odd size, an odd address): a thread has one pair of
// values of its heads, neighbours in the row for neighbours in the warp. 10926 tokens x 24 heads of 80, 34 of them turned
// in halves: 38 us; 16 dimensions a thread as above, value by value, took 116.
template <bool k16, int kPer>
__global__ void __launch_bounds__(256) rotary_pairs_kernel(const __grid_constant__ RotaryCall p) {
  using T = typename std::conditional<k16, uint16_t, float>::type;
  const int64_t job = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_token = p.units * p.groups;
  const int64_t token = job / per_token;
  pdl_wait();
  pdl_launch_dependents();
  if (token >= p.tokens) return;
  const int in = (int)(job - token * per_token), g = in / p.units, pair = in - g * p.units;
  const RotaryPair at = rotary_pair(p.rot, pair);
  const int a = at.a, b = at.b;
  const bool turns = at.turns;
  const bool two = b < p.dim;  // of an odd number of dimensions the last is alone
  const T* x = reinterpret_cast<const T*>(p.x) + token * p.xs_t;
  T lo[kPer], hi[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int h = g + i * p.groups;
    if (h < p.heads) {
      lo[i] = __ldg(x + h * p.xs_h + a);
      if (two) hi[i] = __ldg(x + h * p.xs_h + b);
    }
  }
  float c = 1.f, s = 0.f;
  if (turns) {
    const int64_t position = p.positions64 ? __ldg(reinterpret_cast<const long long*>(p.positions) + token)
                                           : (int64_t)__ldg(reinterpret_cast<const int*>(p.positions) + token);
    turn_cos_sin((uint64_t)position * __ldg(reinterpret_cast<const unsigned long long*>(p.rot.turns) + pair), c, s);
    c *= p.rot.magnitude;
    s *= p.rot.magnitude * p.rot.sign;
  }
  T* out = reinterpret_cast<T*>(p.out) + token * p.os_t;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int h = g + i * p.groups;
    if (h >= p.heads) continue;
    if (turns) {
      float u, v;
      if constexpr (k16) u = __uint_as_float((uint32_t)lo[i] << 16), v = __uint_as_float((uint32_t)hi[i] << 16);
      else u = lo[i], v = hi[i];
      const float first = fmaf(u, c, -v * s), second = fmaf(u, s, v * c);
      if constexpr (k16) {
        const uint32_t both = pack_bf16(first, second);
        lo[i] = (uint16_t)both, hi[i] = (uint16_t)(both >> 16);
      } else {
        lo[i] = first, hi[i] = second;
      }
    }
    out[h * p.os_h + a] = lo[i];
    if (two) out[h * p.os_h + b] = hi[i];
  }
}

template <bool k16>
const void* rotary_variant(bool vec, int per) {
  if (vec)
    return per == 4 ? (const void*)rotary_kernel<k16, 4> : per == 2 ? (const void*)rotary_kernel<k16, 2> : (const void*)rotary_kernel<k16, 1>;
  return per == 4 ? (const void*)rotary_pairs_kernel<k16, 4>
                  : per == 2 ? (const void*)rotary_pairs_kernel<k16, 2> : (const void*)rotary_pairs_kernel<k16, 1>;
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
// In the vector form a thread has one unit, which keeps its registers at 64 (a page of 64 tokens with two units a thread
// and 128 registers took 42 us for 17059 tokens). Otherwise it has one pair of values of every `rows_each`th token.
constexpr int kAppendThreads = 1024;  // most, of a CTA: 128 tokens x 8 units
constexpr int kAppendRows = 8;        // most, of a thread: 128 tokens x 64 pairs

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
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ KvAppendCall p) {
  __shared__ float sm_max[2][32];
  const int which = p.first + blockIdx.z, threads = blockDim.x;
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
  const int64_t xs_h = p.xs_h[which], xs_t = p.xs_t[which];
  const int units = kVec ? rotary_units(rot, dim) : rotary_pairs(rot, dim);
  const int row = threadIdx.x / units, unit = threadIdx.x - row * units;
  const int64_t from = (span.first + (t0 - past) + row) * xs_t;  // this thread's token: in the input, and its codes in the page
  const int to = (begun + row) * dim;
  constexpr bool kAhead = kVec && k16;  // the other forms have no registers for it
  RotaryUnit u{};
  RotaryPair pair{};
  RawUnit<k16> raw;
  float c[8], s[8];  // of the unit's pairs, or of the pair for each token
  const int rows = row < p.rows_each ? (count - row + p.rows_each - 1) / p.rows_each : 0;  // of this thread
  if constexpr (kVec) {
    if (rows > 0) {
      u = rotary_unit(rot, unit);
      if constexpr (kAhead) raw.load(p.x[which], from + head0 * xs_h, u);
      if (u.turned > 0) unit_angles(rot, u, 8 * unit, t0 + row, c, s);
    }
  } else {
    pair = rotary_pair(rot, unit);
    const uint64_t f = pair.turns ? __ldg(reinterpret_cast<const unsigned long long*>(rot.turns) + unit) : 0ull;
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
      if (i < rows && pair.turns) {
        turn_cos_sin((uint64_t)(t0 + row + i * p.rows_each) * f, c[i], s[i]);
        c[i] *= rot.magnitude;
        s[i] *= rot.magnitude;
      }
    }
  }
  if (where < 0 || where >= cache.pages) return;  // (after the values' loads, which do not wait for the page)
  uint8_t* scale_at = cache.scales[which] + where * cache.heads + head0;
  uint8_t* codes = cache.codes[which] + (where * cache.heads + head0) * (int64_t)(page * dim);
  const int lane = threadIdx.x & 31, warps = threads / 32;
  for (int head = head0; head < head1; ++head, ++scale_at, codes += page * dim) {
    const uint32_t old = begun ? *scale_at : 0u;
    float lo[8], hi[8];
    float top = 0.f;
    if constexpr (kVec) {
      if (rows > 0) {
        if constexpr (!kAhead) raw.load(p.x[which], from + head * xs_h, u);
        raw.get(lo, hi);
        if constexpr (kAhead) {
          if (head + 1 < head1) raw.load(p.x[which], from + (head + 1) * xs_h, u);
        }
        if (u.turned > 0) unit_turn(rot.interleaved, c, s, lo, hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = absmax3(top, lo[j], hi[j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAppendRows; ++i) {
        if (i < rows) {
          const int64_t at = from + head * xs_h + i * p.rows_each * xs_t;
          lo[i] = one_value<k16>(p.x[which], at + pair.a);
          hi[i] = one_value<k16>(p.x[which], at + pair.b);
        }
      }
#pragma unroll
      for (int i = 0; i < kAppendRows; ++i) {
        if (i < rows) {
          if (pair.turns) {
            const float a = lo[i], b2 = hi[i];
            lo[i] = fmaf(a, c[i], -b2 * s[i]);
            hi[i] = fmaf(a, s[i], b2 * c[i]);
          }
          top = absmax3(top, lo[i], hi[i]);
        }
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
    if constexpr (kVec) {
      if (rows > 0) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w[j] = e4m3x4(lo[4 * j] * inv, lo[4 * j + 1] * inv, lo[4 * j + 2] * inv, lo[4 * j + 3] * inv);
          w[2 + j] = e4m3x4(hi[4 * j] * inv, hi[4 * j + 1] * inv, hi[4 * j + 2] * inv, hi[4 * j + 3] * inv);
        }
        if (code == 255u) w[0] = w[1] = w[2] = w[3] = 0u;  // zero times NaN has a code of its own
        *reinterpret_cast<uint2*>(codes + to + u.a) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(codes + to + u.b) = make_uint2(w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAppendRows; ++i) {
        if (i < rows) {
          uint8_t* at = codes + to + i * p.rows_each * dim;
          const uint32_t w = code == 255u ? 0u : cvt_e4m3x2_rn(lo[i] * inv, hi[i] * inv);
          if (pair.halves) {
            at[pair.a] = (uint8_t)w;
            at[pair.b] = (uint8_t)(w >> 8);
          } else {
            *reinterpret_cast<uint16_t*>(at + pair.a) = (uint16_t)w;
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
  const bool vec = p.dim % 16 == 0 && (p.rot.interleaved || p.rot.pairs % 8 == 0) && (uintptr_t)p.x % 16 == 0 &&
                   (uintptr_t)p.out % 16 == 0 && p.xs_t * es % 16 == 0 && p.xs_h * es % 16 == 0 && p.os_t * es % 16 == 0 &&
                   p.os_h * es % 16 == 0;
  p.units = vec ? rotary_units(p.rot, p.dim) : rotary_pairs(p.rot, p.dim);
  const int64_t head_units = (int64_t)p.tokens * p.heads * p.units;
  // Heads of a thread, which share its cosines and sines: four or two where that leaves 512 threads an SM.
  const int per = head_units >= 4 * 148 * 512 ? 4 : head_units >= 2 * 148 * 512 ? 2 : 1;
  p.groups = (p.heads + per - 1) / per;
  const int64_t jobs = (int64_t)p.tokens * p.groups * p.units;
  const void* k = p.bf16 ? rotary_variant<true>(vec, per) : rotary_variant<false>(vec, per);
  return launch_pdl(k, dim3((unsigned)((jobs + 255) / 256)), dim3(256), 0, stream, p);
}

cudaError_t launch_kv_append(KvAppendCall p, cudaStream_t stream) {
  const int es = p.bf16 ? 2 : 4;
  bool vec[2];
  for (int i = 0; i < 2; ++i)
    vec[i] = (i == 1 || !p.rot.turns || p.rot.interleaved || p.rot.pairs % 8 == 0) && (uintptr_t)p.x[i] % 16 == 0 &&
             p.xs_t[i] * es % 16 == 0 && p.xs_h[i] * es % 16 == 0;
  const int slots = p.seq.offsets ? (p.seq.tokens >> p.cache.log_page) + 2 * p.seq.batch : p.seq.batch;
  // Keys and values in one launch where both have the same form.
  for (int i = 0; i < 2; ++i) {
    const bool both = vec[0] == vec[1];
    if (both && i == 1) break;
    const int units = vec[i] ? p.cache.dim / 16 : p.cache.dim / 2, page = p.seq.offsets ? p.cache.page : 1;
    p.rows_each = vec[i] ? page : (page + kAppendRows - 1) / kAppendRows;
    p.first = i;
    const int threads = (p.rows_each * units + 31) / 32 * 32;
    // A CTA has all heads of its page, for which it forms the cosines and sines once, where that leaves 1536 threads an SM,
    // and fewer otherwise. 17059 tokens, 8 heads: all eight 28 us, four 32, one 56; 64 single tokens: one 2.9, all 5.7.
    const int64_t page_threads = (int64_t)slots * 2 * threads;
    const int most = (int)min((int64_t)p.cache.heads, (148 * 1536 + page_threads - 1) / page_threads);
    p.heads_each = (p.cache.heads + most - 1) / most;
    const unsigned groups = (unsigned)((p.cache.heads + p.heads_each - 1) / p.heads_each);
    const void* k = p.bf16 ? (vec[i] ? (const void*)kv_append_kernel<true, true> : (const void*)kv_append_kernel<false, true>)
                           : (vec[i] ? (const void*)kv_append_kernel<true, false> : (const void*)kv_append_kernel<false, false>);
    const cudaError_t e = launch_pdl(k, dim3((unsigned)slots, groups, both ? 2 : 1), dim3(threads), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mambo
