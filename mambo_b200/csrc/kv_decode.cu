// Attention of few query rows over the paged FP8 cache: a token or a few of
// each sequence (decoding). With g query heads to a key head and n tokens, g n
// rows read the same keys and values; up to 16 or 32 of them are one unit.
//
// Bound by the cache's bytes, read once: 2 * head size per position and key
// head (64 sequences of 4096 to 8191 positions, 8 key heads of 128, 32 query
// heads: 133 us, 6.03 TB/s, 0.92 of a measured copy; one of 131072, 64 query
// heads: 59 us, 0.69, the rest its start and the join of 37 parts a head).
// With head size 64 (113 us, 0.55) or 17 to 32 rows (20 rows of 2 key heads:
// 75 us, 0.41) by a tile's chain of scores, vote, weights and their terms.
// So keys and values go from memory through tensor copies into shared
// memory and from there straight into the tensor core, 8 bits as they are:
//   S^T [128 positions x rows] = K Q^T        (keys: A, along K)
//   O^T [head size x rows]    += V^T W^T      (values: A, along M)
// with the rows as the MMA's N, and 128 positions or the head size as its M.
// Queries are two E4M3 terms (kv_tc.cuh). Weights are three, each of what the
// one before leaves, at 1, 2^4 and 2^8 times its size: columns of their own in
// one MMA of N = 3 times the rows, so that the values are read from shared
// memory once, and added up with their factors where a unit ends. A thread of
// the softmax has one position and all rows; S^T goes to it through TMEM, the
// weights go back through shared memory, 16 bytes a term.
//
// The softmax works with x = score * log2(e) + (exponent of the position's
// value scale), so that the value scale needs no multiplication anywhere:
//   w = 2^(x - m), O += w * code, l += w * 2^-exponent.
// m need not be the maximum: it is moved (and O rescaled in TMEM) only when a
// weight would pass 2^8.7, which a vote of the four warps finds out, so that
// the common tile has no reduction over positions. A row's m is moved to its
// maximum less 6, so that its largest weight is at least 2^6.
//
// A weight's error is 2^-11 of it (f16, on the way to its terms) or, of the
// smallest, 2^-18 (half the last term's step, 2^-9 of 2^-8): 2^-24 of the row's
// largest weight. It must be that small because weights add up: beside a
// position that has half of the mass, as the first one often does, each of n
// others has 1/n of it, and 2^-24 n is the most that they lose together. (Two
// terms of one size, with steps of 2^-9, lost up to a third of the result at
// 32768 positions.)
//
// Work: the 128-position tiles of all (sequence, head) units in a row, cut into
// one equal range per SM whatever the lengths are (they are on the device).
// A unit that several CTAs share is joined by whichever arrives last, in the
// order of the positions: nothing waits, and results do not depend on who.
//
// Warps 0-3 softmax, 4 copies, 5 MMA, 6 queries of the units to come, 7 the pages' scales, 32 pages ahead (each is
// two dependent loads from memory; a softmax thread that fetched its own a tile ahead spent most of its time on them).
#include "iq3s_tm.cuh"
#include "kernels.cuh"
#include "kv_tc.cuh"

namespace mambo {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxStages = 8;
constexpr float kNone = -3e38f;      // m of a row that has seen nothing
constexpr float kHeadroom = 8.7f;    // 2^8.7 < 448
constexpr float kStart = 6.f;
constexpr int kTerms = 3;            // of a weight, each 2^4 times as large as it counts beside the one before
constexpr uint32_t kTermStep = 0x4C004C00u;  // 2^4, twice in f16

template <int N>
struct Cfg {
  static constexpr int kCtas = N == 16 ? 2 : 1;       // of an SM
  static constexpr uint32_t kStage = 2 * kKvTileBytes;
  static constexpr uint32_t kQ = N * 128u;            // bytes of a term of the queries
  static constexpr uint32_t kW = 128u * N;            // of a term of the weights: [N / 16][128 positions][16]
  static constexpr uint32_t kTmem = N == 16 ? 128 : 256;  // O: N columns for each term of the weights, S: two of N
  static constexpr uint32_t kMeta = 2 * N * 16;       // two units' row factors, places, tokens and heads
  static constexpr uint32_t kScales = 2 * 32 * 8;     // two batches of pages
  static constexpr uint32_t kRed = (4 * N + 16) * 4;  // maxima or sums of the warps; the first tile, a flag
  static constexpr int kNumBars = 3 * kMaxStages + 15;
  static constexpr uint32_t kFixed = 1024 + 4 * kQ + kTerms * kW + kMeta + kScales + kRed + kNumBars * 8 + 16;
  static constexpr int kPart = N * 130;               // floats of a part: O [N][128], m, l
};

// The tiles [x, x1) of a CTA, unit by unit: sequence b, head h, tile t of `tiles` from tile `start` of the sequence on.
struct Walk {
  const KvAttentionCall& p;
  int rows, x, x1, b, h, t, tiles, start;
  bool first;  // of the CTA's part of the unit
  // Tiles of sequence b for each head, and the first of them: none where its rows are too many.
  static __device__ __forceinline__ int tiles_of(const KvAttentionCall& p, int rows, int b, int& start) {
    const KvSpan s = kv_span(p.seq, b);
    start = 0;
    if (s.count < 1 || (int64_t)s.count * p.group > rows) return 0;
    const int64_t len = kv_length(p.seq, b, p.cache.page);
    const int64_t low = p.window ? len - s.count + 1 - (int64_t)p.window : 0;
    start = low > 0 ? (int)(low / kKvTile) : 0;
    const int end = (int)((len + kKvTile - 1) / kKvTile);
    return end > start ? end - start : 1;  // one (of masked positions) where nothing is seen
  }
  // at: the first tile's sequence, head, tile, tiles and start.
  __device__ __forceinline__ Walk(const KvAttentionCall& call, int rows_, int x0, int end, const int* at)
      : p(call), rows(rows_), x(x0), x1(end), b(at[0]), h(at[1]), t(at[2]), tiles(at[3]), start(at[4]), first(true) {}
  __device__ __forceinline__ bool valid() const { return x < x1; }
  __device__ __forceinline__ bool last() const { return t == tiles - 1 || x == x1 - 1; }
  __device__ __forceinline__ void next() {
    ++x;
    first = false;
    if (++t < tiles) return;
    t = 0;
    first = true;
    if (++h < p.cache.heads || x >= x1) return;
    h = 0;
    do tiles = tiles_of(p, rows, ++b, start); while (tiles == 0);  // x < x1: there is one
  }
};

// O^T += V^T W^T over the 128 positions of a tile: values along M (128-byte swizzle, 32 positions in 4096 bytes), all terms of
// the weights along N (no swizzle, 32 positions in 512 bytes); and the arrivals once it is done.
__device__ __forceinline__ void mma_values(uint32_t d, uint32_t v, uint32_t w, uint32_t idesc, uint32_t acc, uint32_t done0,
                                           uint32_t done1) {
  asm volatile(
      "{\n\t.reg .pred p, t;\n\t.reg .b32 a, x;\n\t.reg .b64 da, dx;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 dx, {%2, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, dx, %3, p;\n\t"
      "add.u32 a, %1, 256;\n\tadd.u32 x, %2, 32;\n\tmov.b64 da, {a, %5};\n\tmov.b64 dx, {x, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, dx, %3, t;\n\t"
      "add.u32 a, %1, 512;\n\tadd.u32 x, %2, 64;\n\tmov.b64 da, {a, %5};\n\tmov.b64 dx, {x, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, dx, %3, t;\n\t"
      "add.u32 a, %1, 768;\n\tadd.u32 x, %2, 96;\n\tmov.b64 da, {a, %5};\n\tmov.b64 dx, {x, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, dx, %3, t;\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%8];\n\t}" ::"r"(d),
      "r"(v), "r"(w), "r"(idesc), "r"(acc), "r"(desc_high(1024, true)), "r"(desc_high(2048, false)), "r"(done0), "r"(done1)
      : "memory");
}

// The reduction of N columns over the warp, each lane with a value of each: every step halves the columns that a lane
// goes on with, N - 1 + 32 / N shuffles in all. The result is that of column `column_of(lane)`.
template <int N, typename Op>
__device__ __forceinline__ float reduce_columns(float (&v)[N], int lane, Op op) {
#pragma unroll
  for (int w = N / 2, bit = 1; w >= 1; w >>= 1, bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float other = __shfl_xor_sync(0xFFFFFFFFu, up ? v[i] : v[i + w], bit);
      v[i] = op(up ? v[i + w] : v[i], other);
    }
  }
  if constexpr (N == 16) v[0] = op(v[0], __shfl_xor_sync(0xFFFFFFFFu, v[0], 16));
  return v[0];
}
template <int N>
__device__ __forceinline__ int column_of(int lane) {
  return (int)(__brev((uint32_t)lane) >> (N == 16 ? 28 : 27));
}

}  // namespace

template <int N>
__global__ void __launch_bounds__(kThreads, Cfg<N>::kCtas)
    kv_decode_kernel(const __grid_constant__ KvAttentionCall p, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, int stages, float* partials, int* counters) {
  using C = Cfg<N>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* tiles0 = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* qs = tiles0 + (size_t)stages * C::kStage;  // [2 units][hi, lo][N][128]
  uint8_t* ws = qs + 4 * C::kQ;                       // [terms][N / 16][128][16]
  float* factors = reinterpret_cast<float*>(ws + kTerms * C::kW);  // [2][N]
  int* places = reinterpret_cast<int*>(factors + 2 * N);       // [2][N]
  int2* owners = reinterpret_cast<int2*>(places + 2 * N);      // [2][N]: the row's token and query head
  float2* scales = reinterpret_cast<float2*>(owners + 2 * N);  // [2][32]: key factor, value exponent (minus infinity: no page)
  float* red = reinterpret_cast<float*>(scales + 2 * 32);      // [4][N]
  int* begin = reinterpret_cast<int*>(red + 4 * N);            // the first tile: sequence, head, tile, tiles, start; a flag
  int* warp_sums = begin + 8;                                  // [8]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + C::kRed);
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  const uint32_t kFullK = smem_u32(bars), kFullV = kFullK + 8 * kMaxStages, kEmpty = kFullV + 8 * kMaxStages;
  const uint32_t kSfull = kEmpty + 8 * kMaxStages, kSfree = kSfull + 16, kQfull = kSfree + 16, kQfree = kQfull + 16;
  const uint32_t kMfull = kQfree + 16, kMfree = kMfull + 16, kWfull = kMfree + 16, kWfree = kWfull + 8, kOfree = kWfree + 8;
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(kFullK + 8 * s, 1);
      mbar_init(kFullV + 8 * s, 1);
      mbar_init(kEmpty + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(kSfull + 8 * i, 1);
      mbar_init(kSfree + 8 * i, 4);
      mbar_init(kQfull + 8 * i, 1);
      mbar_init(kQfree + 8 * i, 5);  // the MMAs and the softmax warps
      mbar_init(kMfull + 8 * i, 1);
      mbar_init(kMfree + 8 * i, 4);
    }
    mbar_init(kWfull, 4);
    mbar_init(kWfree, 1);
    mbar_init(kOfree, 4);
    fence_barrier_init();
  }
  if (warp == 5) {
    tc::alloc(smem_u32(slot), C::kTmem);
    tc::relinquish();
  }
  if (threadIdx.x == 128) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_wait();
  pdl_launch_dependents();
  // All tiles, and where this CTA's first one lies: a thread has a run of sequences.
  const int each = (p.seq.batch + kThreads - 1) / kThreads, mine0 = min(p.seq.batch, (int)threadIdx.x * each);
  const int mine1 = min(p.seq.batch, mine0 + each);
  int sum = 0, unused;
  for (int b = mine0; b < mine1; ++b) sum += Walk::tiles_of(p, N, b, unused) * p.cache.heads;
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += up;
  }
  if (lane == 31) warp_sums[warp] = upto;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = (uint32_t)__shfl_sync(0xFFFFFFFFu, (int)*slot, 0);
  int total = 0, before = upto - sum;
  for (int w = 0; w < kThreads / 32; ++w) {
    total += warp_sums[w];
    before += w < warp ? warp_sums[w] : 0;
  }
  // Each of the CTAs that take part has a tile at least: those of a unit's parts are all that the join waits for.
  const int ctas = max(1, min((int)gridDim.x, total));
  const bool has = (int)blockIdx.x < ctas;
  const int x0 = has ? (int)((int64_t)blockIdx.x * total / ctas) : 0;
  const int x1 = has ? (int)(((int64_t)blockIdx.x + 1) * total / ctas) : 0;
  if (x0 < x1 && x0 >= before && x0 < before + sum) {
    int b = mine0, start, n;
    while (x0 >= before + (n = Walk::tiles_of(p, N, b, start)) * p.cache.heads) {
      before += n * p.cache.heads;
      ++b;
    }
    begin[0] = b;
    begin[1] = (x0 - before) / n;
    begin[2] = (x0 - before) % n;
    begin[3] = n;
    begin[4] = start;
  }
  __syncthreads();
  Walk walk(p, N, x0, x1, begin);
  const int log_page = p.cache.log_page, per_tile = kKvTile >> log_page, batch = 32 / per_tile;

  if (warp == 4) {
    // -------------------------------------------------------------- copies
    KvRing ring;
    bool ok = true;
    auto page_of = [&](const Walk& w) {
      const int64_t i = (int64_t)(w.start + w.t) * per_tile + lane;
      return w.valid() && lane < per_tile && i < p.seq.table_pages ? __ldg(p.seq.table + w.b * p.seq.table_stride + i) : -1;
    };
    const uint64_t policy = l2_policy_evict_first();
    Walk ahead = walk;
    int page = page_of(ahead);
    for (int it = 0; walk.valid(); ++it) {
      ahead.next();
      const int next_page = page_of(ahead);
      if (it >= stages && !(ok = kv_warp_wait(kEmpty + 8 * ring.at, ring.phase ^ 1, kSiteKvEmpty))) break;
      const uint32_t kbar = kFullK + 8 * ring.at, vbar = kFullV + 8 * ring.at;
      const uint32_t dst = smem_u32(tiles0) + ring.at * C::kStage + lane * (128u << log_page);
      if (lane == 0) {
        mbar_arrive_expect_tx(kbar, kKvTileBytes);
        mbar_arrive_expect_tx(vbar, kKvTileBytes);
      }
      __syncwarp();
      if (lane < per_tile) {
        // A page outside the cache: a box outside the tensor, which reads zeros.
        const int row = page >= 0 && page < p.cache.pages ? page * p.cache.heads + walk.h : -1;
        tma_load_3d(dst, &kmap, 0, 0, row, kbar, policy);
        tma_load_3d(dst + kKvTileBytes, &vmap, 0, 0, row, vbar, policy);
      }
      page = next_page;
      walk.next();
      ring.next(stages);
    }
    if (!ok) kv_settle();
  } else if (warp == 5) {
    // -------------------------------------------------------------- MMA
    if (walk.valid() && tm::elect_one()) {
      constexpr uint32_t kIdS = tc::idesc_e4m3_f32(128, N);
      constexpr uint32_t kIdO = tc::idesc_e4m3_f32(128, kTerms * N) | kIdescAlongM | kIdescAlongN;
      const bool wide = p.cache.dim > 64;
      const uint32_t stage0 = smem_u32(tiles0), q0 = smem_u32(qs), w0 = smem_u32(ws);
      KvRing kr, vr, sr, qr;
      uint32_t ophase = 0, wphase = 0;
      bool ok = true, first_unit = true, v_first = false;
      // The scores of a tile are formed before the weights of the one before it are waited for.
      auto scores = [&](const Walk& w) {
        uint32_t d = tmem + kTerms * N + sr.at * N, a = desc_low(stage0 + kr.at * C::kStage, 16);
        uint32_t b = desc_low(q0 + qr.at * 2 * C::kQ, 16);
        asm volatile("" : "+r"(d), "+r"(a), "+r"(b));  // before the waits
        if (w.first && !kv_wait(kQfull + 8 * qr.at, qr.phase, kSiteKvFull)) return false;
        if (!kv_wait(kFullK + 8 * kr.at, kr.phase, kSiteKvFull)) return false;
        if (!kv_wait(kSfree + 8 * sr.at, sr.phase ^ 1, kSiteKvEmpty)) return false;
        tc::fence_after_sync();
        mma_along_k_2x2(d, a, b, b + (C::kQ >> 4), kIdS, 0);
        if (wide) mma_along_k_2x2(d, a + 4, b + 4, b + 4 + (C::kQ >> 4), kIdS, 1);
        tc::commit(kSfull + 8 * sr.at);
        if (w.last()) {
          tc::commit(kQfree + 8 * qr.at);
          qr.next(2);
        }
        kr.next(stages);
        sr.next(2);
        return true;
      };
      auto values = [&](bool first) {
        uint32_t v = desc_low(stage0 + vr.at * C::kStage + kKvTileBytes, 1024), w = desc_low(w0, 128);
        asm volatile("" : "+r"(v), "+r"(w));
        if (!kv_wait(kFullV + 8 * vr.at, vr.phase, kSiteKvFull)) return false;
        if (!kv_wait(kWfull, wphase, kSiteKvFull)) return false;
        wphase ^= 1;
        if (first) {
          if (!first_unit) {
            if (!kv_wait(kOfree, ophase, kSiteKvEmpty)) return false;
            ophase ^= 1;
          }
          first_unit = false;
        }
        tc::fence_after_sync();
        mma_values(tmem, v, w, kIdO, !first, kWfree, kEmpty + 8 * vr.at);
        vr.next(stages);
        return true;
      };
      while (ok && walk.valid()) {
        const bool f = walk.first, more = walk.x > x0;
        ok = scores(walk) && (!more || values(v_first));
        v_first = f;
        walk.next();
      }
      if (ok) ok = values(v_first);
      if (!ok) kv_settle();
    }
  } else if (warp == 6) {
    // -------------------------------------------------------------- queries
    KvRing ring;
    bool ok = true;
    const int half = lane >> 4, d0 = 8 * (lane & 15);  // two rows at a time, 8 dimensions a lane
    for (int unit = 0; walk.valid(); ++unit) {
      const KvSpan span = kv_span(p.seq, walk.b);
      const int place0 = kv_length(p.seq, walk.b, p.cache.page) - span.count, rows = span.count * p.group;
      if (unit >= 2 && !(ok = kv_warp_wait(kQfree + 8 * ring.at, ring.phase ^ 1, kSiteKvEmpty))) break;
      // Rows behind the last keep whatever is there: their columns are not read, and their factor is 0.
      if (lane < N) {
        const int t = min(lane, rows - 1) / p.group;
        factors[ring.at * N + lane] = 0.f;
        places[ring.at * N + lane] = place0 + t;
        owners[ring.at * N + lane] = make_int2(span.first + t, walk.h * p.group + lane - t * p.group);
      }
      __syncwarp();
      uint8_t* hi = qs + ring.at * 2 * C::kQ;
      // A loop, four rows a step, and not unrolled: code that runs once is paced by the fetch of its instructions.
#pragma unroll 1
      for (int n0 = 0; n0 < rows; n0 += 4) {
        uint4 raw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 2 * i + half;
          raw[i] = make_uint4(0, 0, 0, 0);
          if (n < rows && d0 < p.cache.dim) {
            const int2 own = owners[ring.at * N + n];
            const uint16_t* q = p.q + own.x * p.qs_t + own.y * p.qs_h + d0;
            raw[i] = __ldg(reinterpret_cast<const uint4*>(q));
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + 2 * i + half;
          uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          uint32_t top = absmax_bf16x2(absmax_bf16x2(w[0], w[1]), absmax_bf16x2(w[2], w[3]));
#pragma unroll
          for (int o = 8; o; o >>= 1) top = absmax_bf16x2(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
          const uint32_t code = bf16_scale_code(max(top & 0x7FFFu, (top >> 16) & 0x7FFFu));
          const float inv = code == 255u ? 0.f : e8m0_to_float(254u - code);
          uint32_t h[2], l[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float v[4] = {__uint_as_float(w[2 * k] << 16) * inv, __uint_as_float(w[2 * k] & 0xFFFF0000u) * inv,
                                __uint_as_float(w[2 * k + 1] << 16) * inv, __uint_as_float(w[2 * k + 1] & 0xFFFF0000u) * inv};
            split_e4m3x4(v, h[k], l[k]);
            if (code == 255u) h[k] = l[k] = 0u;
          }
          if (n < rows) {
            const uint32_t to = n * 128 + (((lane & 15) >> 1 ^ (n & 7)) << 4) + (lane & 1) * 8;
            *reinterpret_cast<uint2*>(hi + to) = make_uint2(h[0], h[1]);
            *reinterpret_cast<uint2*>(hi + C::kQ + to) = make_uint2(l[0], l[1]);
            if (d0 == 0)
              factors[ring.at * N + n] = code == 255u ? NAN : p.scale * 1.4426950408889634f * e8m0_to_float(code);
          }
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(kQfull + 8 * ring.at);
      ring.next(2);
      do walk.next(); while (walk.valid() && !walk.first);
    }
  } else if (warp == 7) {
    // -------------------------------------------------------------- scales: lane `mine` tiles on, page `which` of the tile
    KvRing ring;
    bool ok = true;
    const int mine = lane / per_tile, which = lane - mine * per_tile;
    for (int step = 0; walk.valid(); ++step) {
      int64_t at = -1;
      int h = 0;
      for (int i = 0; i < batch && walk.valid(); ++i) {
        if (i == mine) {
          const int64_t k = (int64_t)(walk.start + walk.t) * per_tile + which;
          at = k < p.seq.table_pages ? walk.b * p.seq.table_stride + k : -1;
          h = walk.h;
        }
        walk.next();
      }
      const int page = at >= 0 ? __ldg(p.seq.table + at) : -1;
      float2 v = make_float2(0.f, -INFINITY);
      if (page >= 0 && page < p.cache.pages) {
        const int64_t row = (int64_t)page * p.cache.heads + h;
        const uint32_t kc = max((uint32_t)__ldg(p.cache.scales[0] + row), kKvMinCode);
        const uint32_t vc = max((uint32_t)__ldg(p.cache.scales[1] + row), kKvMinCode);
        v = make_float2(kc == 255u ? NAN : e8m0_to_float(kc), vc == 255u ? NAN : (float)((int)vc - 127));
      }
      if (step >= 2 && !(ok = kv_warp_wait(kMfree + 8 * ring.at, ring.phase ^ 1, kSiteKvEmpty))) break;
      scales[ring.at * 32 + lane] = v;
      __syncwarp();
      if (lane == 0) mbar_arrive(kMfull + 8 * ring.at);
      ring.next(2);
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int j = threadIdx.x, column = column_of<N>(lane);
    const uint32_t tq = tmem + ((uint32_t)(32 * warp) << 16);
    KvRing sr, vr, qr;
    uint32_t wphase = 1;  // of the last tile's MMAs on the values: a fresh barrier's previous phase counts as over
    KvRing mr;
    int in_batch = 0;
    float m[N], l[N];
    int place_lo = 0, place_hi = 0;
    bool failed = false;
    while (walk.valid()) {
      const bool first = walk.first;
      const int* pl = places + qr.at * N;
      if (first) {
        failed |= !kv_warp_wait(kQfull + 8 * qr.at, qr.phase, kSiteKvFull);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          m[n] = kNone;
          l[n] = 0.f;
        }
        place_lo = pl[0];
        place_hi = pl[N - 1];
      }
      if (in_batch == 0) failed |= !kv_warp_wait(kMfull + 8 * mr.at, mr.phase, kSiteKvFull);
      const float2 sc = scales[mr.at * 32 + in_batch * per_tile + (j >> log_page)];
      const float ck = sc.x, ev = sc.y;
      const bool there = ev != -INFINITY;
      const float back = there ? e8m0_to_float((uint32_t)(127 - (int)ev)) : 1.f;  // 2^-ev; of a NaN 1
      if (++in_batch == batch) {
        in_batch = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(kMfree + 8 * mr.at);
        mr.next(2);
      }
      failed |= !kv_warp_wait(kSfull + 8 * sr.at, sr.phase, kSiteKvFull);
      tc::fence_after_sync();
      uint32_t raw[N];
      kv_ld<N>(tq + kTerms * N + sr.at * N, raw);
      kv_wait_ld();
      kv_tie(raw);
      tc::fence_before_sync();
      if (lane == 0) mbar_arrive(kSfree + 8 * sr.at);
      sr.next(2);

      const int64_t j0 = (int64_t)(walk.start + walk.t) * kKvTile, jj = j0 + j;
      const bool edge = j0 + kKvTile - 1 > place_lo || (p.window && j0 <= (int64_t)place_hi - p.window);
      // The rows' factors from shared memory: in registers they made the form of 16 rows spill (64 x 1 token 138 us for 129).
      float x[N];
#pragma unroll
      for (int n = 0; n < N; n += 4) {
        const float4 c = *reinterpret_cast<const float4*>(factors + qr.at * N + n);
        // The factors' product first: large queries over small keys have scores that a product with one of them alone may pass.
        x[n] = fmaf(__uint_as_float(raw[n]), c.x * ck, ev), x[n + 1] = fmaf(__uint_as_float(raw[n + 1]), c.y * ck, ev);
        x[n + 2] = fmaf(__uint_as_float(raw[n + 2]), c.z * ck, ev), x[n + 3] = fmaf(__uint_as_float(raw[n + 3]), c.w * ck, ev);
      }
      if (edge || !__all_sync(0xFFFFFFFFu, there)) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int at = pl[n];
          if (!there || jj > at || (p.window && jj <= (int64_t)at - p.window)) x[n] = -INFINITY;
        }
      }
      bool up = failed;
#pragma unroll
      for (int n = 0; n < N; ++n) up |= x[n] - m[n] > kHeadroom;  // m + kHeadroom may round to 16 more than m, of scores near 2^27
      if (kv_bar_any(1, 128, up)) {
        if (kv_bar_any(1, 128, failed)) break;  // all four warps leave together
        float f[N];
#pragma unroll
        for (int n = 0; n < N; ++n) f[n] = x[n];
        red[warp * N + column] = reduce_columns<N>(f, lane, [](float a, float b) { return fmaxf(a, b); });
        kv_bar_sync(1, 128);
#pragma unroll
        for (int n = 0; n < N; n += 4) {
          float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 r = *reinterpret_cast<const float4*>(red + w * N + n);
            t[0] = fmaxf(t[0], r.x), t[1] = fmaxf(t[1], r.y), t[2] = fmaxf(t[2], r.z), t[3] = fmaxf(t[3], r.w);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // Only where the row itself asks for it: its bits must not depend on the others', of which those behind the last
            // one hold whatever was in shared memory.
            f[n + k] = 1.f;
            if (t[k] - m[n + k] > kHeadroom) {
              f[n + k] = ex2(m[n + k] - (t[k] - kStart));
              m[n + k] = t[k] - kStart;
              l[n + k] *= f[n + k];
            }
          }
        }
        if (!first) {
          // O holds all tiles before once the last one's MMAs are done.
          failed |= !kv_warp_wait(kWfree, wphase, kSiteKvFull);
          tc::fence_after_sync();
#pragma unroll 1
          for (uint32_t to = tq; to < tq + kTerms * N; to += N) {
            kv_ld<N>(to, raw);
            kv_wait_ld();
            kv_tie(raw);
#pragma unroll
            for (int n = 0; n < N; ++n) raw[n] = __float_as_uint(__uint_as_float(raw[n]) * f[n]);
            tc::st_cols<N>(to, raw);
          }
          tc::wait_st();
          tc::fence_before_sync();
        }
        kv_bar_sync(1, 128);  // before red is used again
      }
      // A position that no row sees: its value may be anything, and zero times NaN is NaN.
      if (edge && (jj > place_hi || (p.window && jj <= (int64_t)place_lo - p.window))) {
        failed |= !kv_wait(kFullV + 8 * vr.at, vr.phase, kSiteKvFull);
        uint4* v = reinterpret_cast<uint4*>(tiles0 + vr.at * C::kStage + kKvTileBytes + j * 128);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
      failed |= !kv_warp_wait(kWfree, wphase, kSiteKvEmpty);
      wphase ^= 1;
      uint8_t* w = ws + j * 16;
#pragma unroll
      for (int g = 0; g < N / 16; ++g) {
        uint32_t term[kTerms][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 16 * g + 4 * i;
          float e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            e[k] = ex2(x[n + k] - m[n + k]);
            l[n + k] = fmaf(e[k], back, l[n + k]);
          }
          uint32_t a = f16x2_of(e[0], e[1]), b = f16x2_of(e[2], e[3]);
#pragma unroll
          for (int t = 0;; ++t) {
            const uint32_t ha = e4m3x2_of_f16x2(a), hb = e4m3x2_of_f16x2(b);
            term[t][i] = ha | (hb << 16);
            if (t == kTerms - 1) break;
            a = mul_f16x2(sub_f16x2(a, f16x2_of_e4m3x2(ha)), kTermStep);  // exact, both
            b = mul_f16x2(sub_f16x2(b, f16x2_of_e4m3x2(hb)), kTermStep);
          }
        }
#pragma unroll
        for (int t = 0; t < kTerms; ++t)
          *reinterpret_cast<uint4*>(w + t * C::kW + g * 2048) = make_uint4(term[t][0], term[t][1], term[t][2], term[t][3]);
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(kWfull);
      vr.next(stages);

      if (walk.last()) {
        // The unit's end, or this CTA's part of it: O^T has a dimension of the head a lane, a row a column.
        const int2* own = owners + qr.at * N;
        const int rows = kv_span(p.seq, walk.b).count * p.group;
        const int unit0 = walk.x - walk.t, unit1 = unit0 + walk.tiles - 1;  // the unit's tiles
        auto result = [&](int n, int d, float sum, float total_, float top) {  // of row n, dimension d
          const int2 to = own[n];
          const __nv_bfloat16 v = __float2bfloat16_rn(total_ == 0.f ? 0.f : sum / total_);
          if (d < p.cache.dim) p.out[to.x * p.os_t + to.y * p.os_h + d] = *reinterpret_cast<const uint16_t*>(&v);
          if (p.lse && d == 0)
            p.lse[to.x * p.ls_t + to.y * p.ls_h] = total_ == 0.f ? -INFINITY : (top + log2f(total_)) * 0.6931471805599453f;
        };
        red[warp * N + column] = reduce_columns<N>(l, lane, [](float a, float b) { return a + b; });
        failed |= !kv_warp_wait(kWfree, wphase, kSiteKvFull);
        tc::fence_after_sync();
        // The terms' sums with their factors, the smallest first.
        kv_ld<N>(tq + (kTerms - 1) * N, raw);
        kv_wait_ld();
        kv_tie(raw);
#pragma unroll
        for (int t = kTerms - 2; t >= 0; --t) {
          uint32_t more[N];
          kv_ld<N>(tq + t * N, more);
          kv_wait_ld();
          kv_tie(more);
#pragma unroll
          for (int n = 0; n < N; ++n) raw[n] = __float_as_uint(fmaf(__uint_as_float(raw[n]), 0.0625f, __uint_as_float(more[n])));
        }
        tc::fence_before_sync();
        if (lane == 0) mbar_arrive(kOfree);
        kv_bar_sync(1, 128);
        if (unit0 >= x0 && unit1 < x1) {
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n < rows) result(n, j, __uint_as_float(raw[n]), (red[n] + red[N + n]) + (red[2 * N + n] + red[3 * N + n]), m[n]);
        } else {
          // Published: O [N][128], m [N], l [N]. The last to arrive joins all parts, in the order of the positions.
          const int cta0 = kv_owner(unit0, total, ctas), cta1 = kv_owner(unit1, total, ctas);
          auto part = [&](int cta) { return partials + (int64_t)(cta * 2 + (cta == cta0)) * C::kPart; };
          float* mine = part(blockIdx.x);
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n < rows) __stcg(mine + n * 128 + j, __uint_as_float(raw[n]));
          if (j < N) __stcg(mine + N * 129 + j, (red[j] + red[N + j]) + (red[2 * N + j] + red[3 * N + j]));
          if (j == 32) {
#pragma unroll
            for (int n = 0; n < N; n += 4)
              __stcg(reinterpret_cast<float4*>(mine + N * 128 + n), make_float4(m[n], m[n + 1], m[n + 2], m[n + 3]));
          }
          kv_bar_sync(1, 128);  // orders the warps' stores before the counting thread's release
          if (j == 0) {
            begin[5] = atomic_add_acq_rel_gpu(counters + cta0, 1) == cta1 - cta0;
            if (begin[5]) counters[cta0] = 0;  // all parts are in: zero again for the next launch
          }
          kv_bar_sync(1, 128);
          if (begin[5]) {
            // Rows' maxima and sums, 128 / N threads a row (over the weights' buffer: the MMAs are done with it).
            constexpr int kSplit = 128 / N;
            float* tops = reinterpret_cast<float*>(ws);  // [kSplit][N], then [kSplit][N] sums
            const int n = j % N;
            float top = kNone, sum = 0.f;
#pragma unroll 4
            for (int c = cta0 + j / N; c <= cta1; c += kSplit) top = fmaxf(top, __ldcg(part(c) + N * 128 + n));
            tops[j] = top;
            kv_bar_sync(1, 128);
            for (int i = 0; i < kSplit; ++i) top = fmaxf(top, tops[i * N + n]);
#pragma unroll 4
            for (int c = cta0 + j / N; c <= cta1; c += kSplit)
              sum = fmaf(ex2(__ldcg(part(c) + N * 128 + n) - top), __ldcg(part(c) + N * 129 + n), sum);
            tops[128 + j] = sum;
            kv_bar_sync(1, 128);
            if (j < N) {
              float all = 0.f;
              for (int i = 0; i < kSplit; ++i) all += tops[128 + i * N + n];
              red[n] = top;
              red[N + n] = all;
            }
            kv_bar_sync(1, 128);
            // A warp a row, four dimensions a lane: many parts' loads are in flight at once.
#pragma unroll 1
            for (int r = warp; r < rows; r += 4) {
              const float at = red[r], all = red[N + r];
              float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
              for (int c = cta0; c <= cta1; ++c) {
                const float4 v = __ldcg(reinterpret_cast<const float4*>(part(c) + r * 128) + lane);
                const float f = ex2(__ldcg(part(c) + N * 128 + r) - at);
                o[0] = fmaf(f, v.x, o[0]), o[1] = fmaf(f, v.y, o[1]), o[2] = fmaf(f, v.z, o[2]), o[3] = fmaf(f, v.w, o[3]);
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) result(r, 4 * lane + k, o[k], all, at);
            }
          }
        }
        kv_bar_sync(1, 128);  // before red and the weights' buffer are used again
        if (lane == 0) mbar_arrive(kQfree + 8 * qr.at);
        qr.next(2);
      }
      walk.next();
    }
    __syncwarp();
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 5) {
    tc::fence_after_sync();
    tc::dealloc(tmem, C::kTmem);
  }
}

namespace {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                   q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeFn>(ptr)
               : nullptr;
  }();
  return fn;
}

template <int N>
cudaError_t launch_decode(const KvAttentionCall& p, const CUtensorMap& k, const CUtensorMap& v, int sms, int smem_optin,
                          float* partials, int* counters, cudaStream_t stream) {
  using C = Cfg<N>;
  // As many stages as fit the SM's shared memory, of which each CTA has 1 KB besides: of two CTAs three each, with 376 bytes
  // to spare, of one six.
  const uint32_t room = ((uint32_t)smem_optin + 1024) / C::kCtas - 1024;
  const int stages = min(kMaxStages, (int)((room - C::kFixed) / C::kStage));
  const uint32_t smem = C::kFixed + stages * C::kStage;
  const void* kernel = (const void*)kv_decode_kernel<N>;
  const cudaError_t e = ensure_smem_attribute(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(sms * C::kCtas), dim3(kThreads), smem, stream, p, k, v, stages, partials, counters);
}

}  // namespace

// A page of a head as a box: rows of 128 bytes, zero behind the head size.
bool kv_page_map(const KvCache& c, int which, CUtensorMap* map) {
  const EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)c.dim, (cuuint64_t)c.page, (cuuint64_t)c.pages * c.heads};
  const cuuint64_t strides[2] = {(cuuint64_t)c.dim, (cuuint64_t)c.dim * c.page};
  const cuuint32_t box[3] = {128, (cuuint32_t)c.page, 1}, one[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.codes[which], dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t kv_decode_partial_bytes(int group, int sms) {
  return (size_t)sms * 2 * (group <= 16 ? Cfg<16>::kCtas * Cfg<16>::kPart : Cfg<32>::kCtas * Cfg<32>::kPart) * sizeof(float);
}

cudaError_t launch_kv_decode(const KvAttentionCall& p, const CUtensorMap& k, const CUtensorMap& v, int sms, int smem_optin,
                             float* partials, int* counters, cudaStream_t stream) {
  return p.group <= 16 ? launch_decode<16>(p, k, v, sms, smem_optin, partials, counters, stream)
                       : launch_decode<32>(p, k, v, sms, smem_optin, partials, counters, stream);
}

}  // namespace mambo
