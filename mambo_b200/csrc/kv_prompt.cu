// Attention of many query rows over the paged FP8 cache: prompts and chunks of
// prompts, and any sequence whose rows (tokens times the query heads of a key
// head) are more than the decode kernel takes.
//
// A unit is 256 rows of one key head (row r of a sequence: token r / group,
// query head r % group) as two MMA tiles of 128, which share the keys and
// values that pass by. For each 128 positions and tile:
//   S [128 x 128] = Q K^T       8-bit MMAs, the queries in two exact terms (kv_tc.cuh)
//   O [128 x D]  += W V         f16 MMAs, the weights W from TMEM (over S, which they replace)
// Two 8-bit terms cost what one 16-bit product does and need no conversion of
// the keys. The values are converted to f16 (exactly) by a warpgroup of their
// own: weights in f16 have 11 bits, where two more terms would have cost the
// softmax, the busiest part, more instructions than the conversion is.
//
// A softmax thread has a row: no reductions over lanes. As in the decode kernel
// x = score * log2(e) + exponent of the position's value scale, w = 2^(x - m),
// l += w * 2^-exponent, and m moves (O is rescaled) only when a weight would
// pass 2^8. What paces the kernel: the tensor core (2048 clocks for both tiles
// and 128 positions of head size 128), then the softmax, whose 2^x take as long
// on the special function unit alone.
//
// Work: all units' tiles in a row, one equal range per SM (units have unequal
// lengths under the causal mask, and there may be few of them). A unit that
// several CTAs share is joined by the last to arrive, in the order of the
// positions.
//
// Warps 0-3 and 4-7 softmax of either tile, 8-11 queries and values, 12 copies,
// 13 MMA, 14 the pages' scales. Compiled as a whole program of its own, for
// setmaxnreg; so it has its own device status.
#define MAMBO_OWN_DEVICE_STATUS
#include "iq3s_tm.cuh"
#include "kernels.cuh"
#include "kv_tc.cuh"

namespace mambo {

namespace {

constexpr int kThreads = 512;
constexpr int kRows = 128;            // of an MMA tile
constexpr int kUnitRows = 2 * kRows;
constexpr int kKStages = 3, kVStages = 2;
constexpr float kNone = -1e30f;       // m of a row that has seen nothing
constexpr float kHeadroom = 8.f;

// Shared memory: queries [2 tiles][hi, lo][128][128], keys, values as they come and in f16 [2 halves of D][128][128 bytes].
constexpr uint32_t kQ = 4 * kKvTileBytes, kVf = 2 * kKvTileBytes;
constexpr uint32_t kAtK = kQ, kAtV = kAtK + kKStages * kKvTileBytes, kAtVf = kAtV + kVStages * kKvTileBytes;
constexpr uint32_t kAtFactors = kAtVf + 2 * kVf, kAtScales = kAtFactors + kUnitRows * 4, kAtBegin = kAtScales + 2 * 32 * 16;
constexpr uint32_t kAtBars = kAtBegin + 128;
constexpr int kNumBars = 2 * kKStages + 2 * kVStages + 4 + 8 + 2 + 4;
constexpr uint32_t kSmem = 1024 + kAtBars + kNumBars * 8 + 16;
constexpr int kPart = kRows * 130;    // floats of a tile's part: O [32][128][4], m, l

// The unit that a CTA is at, and its tiles. b, h: sequence and key head; u: the unit's number in them.
struct Walk {
  const KvAttentionCall& p;
  int x, x1, b, h, u, t, tiles, start;
  int first_token, place0, rows;  // of the sequence: its first token, the position of that, its rows
  bool first;                     // tile of the CTA's part of the unit
  __device__ __forceinline__ void sequence() {
    const KvSpan s = kv_span(p.seq, b);
    first_token = s.first;
    rows = (int64_t)s.count * p.group > p.few ? s.count * p.group : 0;
    place0 = kv_length(p.seq, b, p.cache.page) - s.count;
  }
  __device__ __forceinline__ int units() const { return (rows + kUnitRows - 1) / kUnitRows; }
  __device__ __forceinline__ int place(int row) const { return place0 + min(row, rows - 1) / p.group; }
  // Tiles of unit i, at least one.
  __device__ __forceinline__ int tiles_of(int i, int& at) const {
    const int64_t low = p.window ? place(kUnitRows * i) + 1 - (int64_t)p.window : 0;
    at = low > 0 ? (int)(low / kKvTile) : 0;
    const int high = place(kUnitRows * i + kUnitRows - 1);
    const int end = high >= 0 ? high / kKvTile + 1 : 0;
    return max(end - at, 1);
  }
  __device__ __forceinline__ Walk(const KvAttentionCall& call, int x0, int end, const int* at)
      : p(call), x(x0), x1(end), b(at[0]), h(at[1]), u(at[2]), t(at[3]), tiles(1), start(0), first(true) {
    if (x >= x1) return;
    sequence();
    tiles = tiles_of(u, start);
  }
  __device__ __forceinline__ bool valid() const { return x < x1; }
  __device__ __forceinline__ bool last() const { return t == tiles - 1 || x == x1 - 1; }
  __device__ __forceinline__ void next() {
    ++x;
    first = false;
    if (++t < tiles) return;
    t = 0;
    first = true;
    if (x >= x1) return;
    if (++u == units()) {
      u = 0;
      if (++h == p.cache.heads) {
        h = 0;
        do {
          ++b;
          sequence();
        } while (rows == 0);  // x < x1: there is one
      }
    }
    tiles = tiles_of(u, start);
  }
  // Places of a tile's first and last rows (lo > hi: it has no rows), and whether its rows see any of the 128 positions
  // from j0 on: what the MMA and the softmax both go by.
  __device__ __forceinline__ void bounds(int q, int& lo, int& hi) const {
    const int r = kUnitRows * u + kRows * q;
    lo = r < rows ? place(r) : 0;
    hi = r < rows ? place(r + kRows - 1) : -1;
  }
  __device__ __forceinline__ int64_t j0() const { return (int64_t)(start + t) * kKvTile; }
  __device__ __forceinline__ bool sees(int lo, int hi) const {
    return j0() <= hi && (p.window == 0 || j0() + kKvTile - 1 > (int64_t)lo - p.window);
  }
};

// One tile's S = Q K^T: head size up to 64 or 128, two terms of A.
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b, bool wide, uint32_t done) {
  constexpr uint32_t kId = tc::idesc_e4m3_f32(kRows, kKvTile);
  asm volatile(
      "{\n\t.reg .pred p, t, w;\n\t.reg .b32 x, y, z;\n\t.reg .b64 dx, dy, db;\n\t"
      "setp.ne.b32 p, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\tsetp.ne.b32 w, %5, 0;\n\t"
      "add.u32 y, %1, 1024;\n\t"
      "mov.b64 dx, {%1, %4};\n\tmov.b64 dy, {y, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dx, db, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dy, db, %3, t;\n\t"
      "add.u32 x, %1, 2;\n\tadd.u32 y, %1, 1026;\n\tadd.u32 z, %2, 2;\n\t"
      "mov.b64 dx, {x, %4};\n\tmov.b64 dy, {y, %4};\n\tmov.b64 db, {z, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dx, db, %3, t;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dy, db, %3, t;\n\t"
      "add.u32 x, %1, 4;\n\tadd.u32 y, %1, 1028;\n\tadd.u32 z, %2, 4;\n\t"
      "mov.b64 dx, {x, %4};\n\tmov.b64 dy, {y, %4};\n\tmov.b64 db, {z, %4};\n\t"
      "@w tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dx, db, %3, t;\n\t"
      "@w tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dy, db, %3, t;\n\t"
      "add.u32 x, %1, 6;\n\tadd.u32 y, %1, 1030;\n\tadd.u32 z, %2, 6;\n\t"
      "mov.b64 dx, {x, %4};\n\tmov.b64 dy, {y, %4};\n\tmov.b64 db, {z, %4};\n\t"
      "@w tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dx, db, %3, t;\n\t"
      "@w tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], dy, db, %3, t;\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(kId), "r"(desc_high(1024, true)), "r"((int)wide), "r"(done)
      : "memory");
}
// One tile's O (+)= W V: weights f16 at TMEM column w (8 columns for 16 positions), values f16 along N (16 positions in
// 2048 bytes).
__device__ __forceinline__ void mma_values(uint32_t d, uint32_t w, uint32_t v, uint32_t idesc, uint32_t acc, uint32_t done) {
  asm volatile(
      "{\n\t.reg .pred p, t;\n\t.reg .b32 a, b;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t"
      "add.u32 a, %1, 8;\n\tadd.u32 b, %2, 128;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 16;\n\tadd.u32 b, %2, 256;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 24;\n\tadd.u32 b, %2, 384;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 32;\n\tadd.u32 b, %2, 512;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 40;\n\tadd.u32 b, %2, 640;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 48;\n\tadd.u32 b, %2, 768;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "add.u32 a, %1, 56;\n\tadd.u32 b, %2, 896;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, t;\n\t"
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),
      "r"(w), "r"(v), "r"(idesc), "r"(acc), "r"(desc_high(1024, true)), "r"(done)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace

__global__ void __launch_bounds__(kThreads, 1)
    kv_prompt_kernel(const __grid_constant__ KvAttentionCall p, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, float* partials, int* counters) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* factors = reinterpret_cast<float*>(sm + kAtFactors);   // of the unit's rows
  float4* scales = reinterpret_cast<float4*>(sm + kAtScales);   // [2][4 tiles][8]: key factor, value exponent, 2^-exponent
  int* begin = reinterpret_cast<int*>(sm + kAtBegin);           // the first tile: sequence, head, unit, tile; [8] flags
  int* warp_sums = begin + 16;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kAtBars);
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  const uint32_t sm0 = smem_u32(sm);
  const uint32_t kKfull = smem_u32(bars), kKfree = kKfull + 8 * kKStages, kVfull = kKfree + 8 * kKStages;
  const uint32_t kVfree = kVfull + 8 * kVStages, kFfull = kVfree + 8 * kVStages, kFfree = kFfull + 16;  // values in f16
  const uint32_t kSfull = kFfree + 16, kWfull = kSfull + 16, kOdone = kWfull + 16, kOfree = kOdone + 16;
  const uint32_t kQfull = kOfree + 16, kQfree = kQfull + 8, kMfull = kQfree + 8, kMfree = kMfull + 16;
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(kKfull + 8 * s, 1);
      mbar_init(kKfree + 8 * s, 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(kVfull + 8 * s, 1);
      mbar_init(kVfree + 8 * s, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(kFfull + 8 * i, 4);
      mbar_init(kFfree + 8 * i, 1);
      mbar_init(kSfull + 8 * i, 1);
      mbar_init(kWfull + 8 * i, 4);
      mbar_init(kOdone + 8 * i, 1);
      mbar_init(kOfree + 8 * i, 4);
      mbar_init(kMfull + 8 * i, 1);
      mbar_init(kMfree + 8 * i, 8);
    }
    mbar_init(kQfull, 4);
    mbar_init(kQfree, 9);  // the MMAs and the softmax warps
    fence_barrier_init();
  }
  if (warp == 13) {
    tc::alloc(smem_u32(slot), 512);
    tc::relinquish();
  }
  if (warp == 12 && lane == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_wait();
  pdl_launch_dependents();
  // All tiles, and where this CTA's first one lies: a warp has a run of sequences, a lane every 32nd unit of one.
  const int each = (p.seq.batch + 15) / 16, mine0 = min(p.seq.batch, warp * each), mine1 = min(p.seq.batch, mine0 + each);
  const int zeros[4] = {0, 0, 0, 0};
  Walk scan(p, 0, 0, zeros);
  auto tiles_of_head = [&](int b) {
    scan.b = b;
    scan.sequence();
    int n = 0, at;
    for (int i = lane; i < scan.units(); i += 32) n += scan.tiles_of(i, at);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    return n;
  };
  int sum = 0;
  for (int b = mine0; b < mine1; ++b) sum += tiles_of_head(b) * p.cache.heads;
  if (lane == 0) warp_sums[warp] = sum;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = (uint32_t)__shfl_sync(0xFFFFFFFFu, (int)*slot, 0);
  int total = 0, before = 0;
  for (int w = 0; w < 16; ++w) {
    total += warp_sums[w];
    before += w < warp ? warp_sums[w] : 0;
  }
  // Each of the CTAs that take part has a tile at least: those of a unit's parts are all that the join waits for.
  const int ctas = max(1, min((int)gridDim.x, total));
  const bool has = (int)blockIdx.x < ctas;
  const int x0 = has ? (int)((int64_t)blockIdx.x * total / ctas) : 0;
  const int x1 = has ? (int)(((int64_t)blockIdx.x + 1) * total / ctas) : 0;
  if (x0 < x1 && x0 >= before && x0 < before + sum) {
    int b = mine0, n;
    while (x0 >= before + (n = tiles_of_head(b)) * p.cache.heads) {
      before += n * p.cache.heads;
      ++b;
    }
    const int h = (x0 - before) / n, units = scan.units();
    int rest = (x0 - before) % n;  // tiles of the head before the first one
    for (int i0 = 0;; i0 += 32) {
      int at;
      const int mine = i0 + lane < units ? scan.tiles_of(i0 + lane, at) : 0;
      int upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += up;
      }
      if (rest >= upto - mine && rest < upto) {
        begin[0] = b;
        begin[1] = h;
        begin[2] = i0 + lane;
        begin[3] = rest - (upto - mine);
      }
      const int all = __shfl_sync(0xFFFFFFFFu, upto, 31);
      if (rest < all || i0 + 32 >= units) break;
      rest -= all;
    }
  }
  __syncthreads();
  Walk walk(p, x0, x1, begin);
  const int log_page = p.cache.log_page, per_tile = kKvTile >> log_page;

  // Register split, launched with 128 a thread: 256 x 192 + 128 x 80 + 128 x 48 = 512 x 128.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 12) {
      // ------------------------------------------------------------ copies
      KvRing kr, vr;
      auto page_of = [&](const Walk& w) {
        const int64_t i = (int64_t)(w.start + w.t) * per_tile + lane;
        return w.valid() && lane < per_tile && i < p.seq.table_pages ? __ldg(p.seq.table + w.b * p.seq.table_stride + i) : -1;
      };
      const uint64_t policy = l2_policy_evict_last();
      int page = page_of(walk);
      bool ok = true;
      for (int it = 0; walk.valid(); ++it) {
        const int h = walk.h;
        walk.next();
        const int next_page = page_of(walk);
        // A page outside the cache: a box outside the tensor, which reads zeros.
        const int row = page >= 0 && page < p.cache.pages ? page * p.cache.heads + h : -1;
        if (it >= kKStages && !(ok = kv_warp_wait(kKfree + 8 * kr.at, kr.phase ^ 1, kSiteKvEmpty))) break;
        if (lane == 0) mbar_arrive_expect_tx(kKfull + 8 * kr.at, kKvTileBytes);
        __syncwarp();
        if (lane < per_tile)
          tma_load_3d(sm0 + kAtK + kr.at * kKvTileBytes + lane * (128u << log_page), &kmap, 0, 0, row, kKfull + 8 * kr.at, policy);
        if (it >= kVStages && !(ok = kv_warp_wait(kVfree + 8 * vr.at, vr.phase ^ 1, kSiteKvEmpty))) break;
        if (lane == 0) mbar_arrive_expect_tx(kVfull + 8 * vr.at, kKvTileBytes);
        __syncwarp();
        if (lane < per_tile)
          tma_load_3d(sm0 + kAtV + vr.at * kKvTileBytes + lane * (128u << log_page), &vmap, 0, 0, row, kVfull + 8 * vr.at, policy);
        page = next_page;
        kr.next(kKStages);
        vr.next(kVStages);
      }
      if (!ok) kv_settle();
    } else if (warp == 13) {
      // ------------------------------------------------------------ MMA
      if (walk.valid() && tm::elect_one()) {
        const uint32_t idesc_o = tc::idesc_f16_f32(kRows, p.cache.dim) | kIdescAlongN;
        const bool wide = p.cache.dim > 64;
        const uint32_t q0 = desc_low(sm0, 16), k0 = desc_low(sm0 + kAtK, 16), v0 = desc_low(sm0 + kAtVf, kKvTileBytes);
        KvRing kr, fr;
        uint32_t qphase = 0, wphase[2] = {0, 0}, ophase[2] = {1, 1};
        bool ok = true, started[2] = {false, false};
        // The scores of a tile; those of a tile of positions that a tile of rows does not see are left out.
        auto scores = [&](const Walk& w, int q) {
          int lo, hi;
          w.bounds(q, lo, hi);
          if (w.sees(lo, hi))
            mma_scores(tmem + q * 128, q0 + q * (2 * kKvTileBytes >> 4), k0 + kr.at * (kKvTileBytes >> 4), wide, kSfull + 8 * q);
        };
        auto values = [&](const Walk& w, int q) {
          int lo, hi;
          w.bounds(q, lo, hi);
          if (!w.sees(lo, hi)) return true;
          if (!kv_wait(kWfull + 8 * q, wphase[q], kSiteKvFull)) return false;
          wphase[q] ^= 1;
          if (!started[q]) {
            // The softmax has read the last unit's O.
            if (!kv_wait(kOfree + 8 * q, ophase[q], kSiteKvEmpty)) return false;
          }
          tc::fence_after_sync();
          mma_values(tmem + 256 + q * 128, tmem + q * 128, v0 + fr.at * (kVf >> 4), idesc_o, started[q], kOdone + 8 * q);
          started[q] = true;
          return true;
        };
        Walk ahead = walk;
        auto next_scores = [&](int q) {  // of the tile after, while the softmax works on the other tile of rows
          if (!ahead.valid()) return true;
          if (q == 0) {
            if (ahead.first) {
              if (!kv_wait(kQfull, qphase, kSiteKvFull)) return false;
              qphase ^= 1;
            }
            if (!kv_wait(kKfull + 8 * kr.at, kr.phase, kSiteKvFull)) return false;
            tc::fence_after_sync();
          }
          scores(ahead, q);
          if (q == 1) {
            tc::commit(kKfree + 8 * kr.at);
            if (ahead.last()) tc::commit(kQfree);
            kr.next(kKStages);
          }
          return true;
        };
        ok = next_scores(0) && next_scores(1);
        ahead.next();
        while (ok && walk.valid()) {
          if (walk.first) started[0] = started[1] = false;
          ok = kv_wait(kFfull + 8 * fr.at, fr.phase, kSiteKvFull);
          if (!ok) break;
          // The next unit's queries may still be on their way: both tiles' values come first then.
          const bool turn = ahead.valid() && ahead.first;
          ok = values(walk, 0) && (turn || next_scores(0)) && values(walk, 1) && (!turn || next_scores(0)) && next_scores(1);
          if (!ok) break;
          tc::commit(kFfree + 8 * fr.at);
          fr.next(2);
          if (walk.last()) {
            for (int q = 0; q < 2; ++q)
              if (started[q]) ophase[q] ^= 1;
          }
          walk.next();
          ahead.next();
        }
        if (!ok) kv_settle();
      }
    } else if (warp == 14) {
      // ------------------------------------------------------------ scales: four tiles at a time, 16 positions a lane
      KvRing ring;
      for (int step = 0; walk.valid(); ++step) {
        int64_t at = -1;
        int h = 0;
        for (int i = 0; i < 4 && walk.valid(); ++i) {
          if (i == lane >> 3) {
            const int64_t k = (walk.j0() + 16 * (lane & 7)) >> log_page;
            at = k < p.seq.table_pages ? walk.b * p.seq.table_stride + k : -1;
            h = walk.h;
          }
          walk.next();
        }
        const int page = at >= 0 ? __ldg(p.seq.table + at) : -1;
        float4 v = make_float4(0.f, -INFINITY, 0.f, 0.f);  // positions without a page: x is minus infinity
        if (page >= 0 && page < p.cache.pages) {
          const int64_t row = (int64_t)page * p.cache.heads + h;
          const uint32_t kc = max((uint32_t)__ldg(p.cache.scales[0] + row), kKvMinCode);
          const uint32_t vc = max((uint32_t)__ldg(p.cache.scales[1] + row), kKvMinCode);
          v = make_float4(kc == 255u ? NAN : e8m0_to_float(kc), vc == 255u ? NAN : (float)((int)vc - 127),
                          vc == 255u ? 1.f : e8m0_to_float(254u - vc), 0.f);
        }
        if (step >= 2 && !kv_warp_wait(kMfree + 8 * ring.at, ring.phase ^ 1, kSiteKvEmpty)) break;
        scales[ring.at * 32 + lane] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(kMfull + 8 * ring.at);
        ring.next(2);
      }
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // -------------------------------------------------------------- queries and values
    const int i = threadIdx.x - 256;  // position of the tile
    const bool vec = (uintptr_t)p.q % 16 == 0 && p.qs_t % 8 == 0 && p.qs_h % 8 == 0;
    KvRing vr, fr;
    int unit = 0;
    // A half warp a row, eight dimensions a lane.
    auto queries = [&](const Walk& w) {
      if (unit > 0) kv_warp_wait(kQfree, (unit & 1) ^ 1, kSiteKvEmpty);
      ++unit;
      const int d0 = 8 * (lane & 15), r0 = kUnitRows * w.u;
      const int rows = min(kUnitRows, w.rows - r0);
#pragma unroll 1
      for (int n0 = 2 * (warp - 8) + (lane >> 4); n0 < kUnitRows; n0 += 32) {
        uint4 raw[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = n0 + 8 * k;
          raw[k] = make_uint4(0, 0, 0, 0);
          if (n < rows && d0 < p.cache.dim) {
            const int t = (r0 + n) / p.group;
            const uint16_t* q = p.q + (int64_t)(w.first_token + t) * p.qs_t +
                                (int64_t)(w.h * p.group + (r0 + n) - t * p.group) * p.qs_h + d0;
            if (vec) {
              raw[k] = __ldg(reinterpret_cast<const uint4*>(q));
            } else {
              uint32_t v[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) v[c] = (uint32_t)__ldg(q + 2 * c) | (uint32_t)__ldg(q + 2 * c + 1) << 16;
              raw[k] = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = n0 + 8 * k;
          const uint32_t v[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
          uint32_t top = absmax_bf16x2(absmax_bf16x2(v[0], v[1]), absmax_bf16x2(v[2], v[3]));
#pragma unroll
          for (int o = 8; o; o >>= 1) top = absmax_bf16x2(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
          const uint32_t code = mxfp8_scale_code(__uint_as_float(max(top & 0x7FFFu, (top >> 16) & 0x7FFFu) << 16));
          const float inv = code == 255u ? 0.f : e8m0_to_float(254u - code);
          uint32_t h[2], l[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float e[4] = {__uint_as_float(v[2 * c] << 16) * inv, __uint_as_float(v[2 * c] & 0xFFFF0000u) * inv,
                                __uint_as_float(v[2 * c + 1] << 16) * inv, __uint_as_float(v[2 * c + 1] & 0xFFFF0000u) * inv};
            split_e4m3x4(e, h[c], l[c]);
            if (code == 255u) h[c] = l[c] = 0u;
          }
          uint8_t* to = sm + (n >> 7) * 2 * kKvTileBytes + (n & 127) * 128 + (((lane & 15) >> 1 ^ (n & 7)) << 4) + (lane & 1) * 8;
          *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
          *reinterpret_cast<uint2*>(to + kKvTileBytes) = make_uint2(l[0], l[1]);
          if (d0 == 0) factors[n] = code == 255u ? NAN : p.scale * 1.4426950408889634f * e8m0_to_float(code);
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(kQfull);
    };
    if (walk.valid()) queries(walk);
    for (int it = 0; walk.valid(); ++it) {
      // A position that no row sees: its value may be anything, and zero times NaN is NaN.
      int lo, hi, lo1, hi1;
      walk.bounds(0, lo, hi);
      walk.bounds(1, lo1, hi1);
      const int64_t j = walk.j0() + i;
      const bool none = j > max(hi, hi1) || (p.window && j <= (int64_t)lo - p.window);
      kv_warp_wait(kVfull + 8 * vr.at, vr.phase, kSiteKvFull);
      if (it >= 2) kv_warp_wait(kFfree + 8 * fr.at, fr.phase ^ 1, kSiteKvEmpty);
      const uint8_t* from = sm + kAtV + vr.at * kKvTileBytes + i * 128;
      uint8_t* to = sm + kAtVf + fr.at * kVf + i * 128;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 v = *reinterpret_cast<const uint4*>(from + ((c ^ (i & 7)) << 4));
        if (none) v = make_uint4(0, 0, 0, 0);
        uint8_t* half = to + (c >> 2) * kKvTileBytes;
        const int c0 = 2 * (c & 3);
        *reinterpret_cast<uint4*>(half + ((c0 ^ (i & 7)) << 4)) =
            make_uint4(f16x2_of_e4m3x2(v.x & 0xFFFFu), f16x2_of_e4m3x2(v.x >> 16), f16x2_of_e4m3x2(v.y & 0xFFFFu), f16x2_of_e4m3x2(v.y >> 16));
        *reinterpret_cast<uint4*>(half + (((c0 + 1) ^ (i & 7)) << 4)) =
            make_uint4(f16x2_of_e4m3x2(v.z & 0xFFFFu), f16x2_of_e4m3x2(v.z >> 16), f16x2_of_e4m3x2(v.w & 0xFFFFu), f16x2_of_e4m3x2(v.w >> 16));
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(kVfree + 8 * vr.at);
        mbar_arrive(kFfull + 8 * fr.at);
      }
      vr.next(kVStages);
      fr.next(2);
      const bool more = walk.last();
      walk.next();
      if (more && walk.valid()) queries(walk);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // -------------------------------------------------------------- softmax
    const int q = warp >> 2, r = threadIdx.x & 127;
    const uint32_t ts = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + q * 128, to_ = ts + 256;
    KvRing mr;
    int in_batch = 0;
    uint32_t sphase = 0, ophase = 1;  // ophase: of the last MMAs on the values
    uint32_t qphase = 0;
    float m = kNone, l = 0.f, cq = 0.f;
    int lo = 0, hi = -1, place = -1;
    bool started = false;
    while (walk.valid()) {
      if (walk.first) {
        kv_warp_wait(kQfull, qphase, kSiteKvFull);
        qphase ^= 1;
        cq = factors[kRows * q + r];
        __syncwarp();
        if (lane == 0) mbar_arrive(kQfree);
        walk.bounds(q, lo, hi);
        const int row = kUnitRows * walk.u + kRows * q + r;
        place = row < walk.rows ? walk.place(row) : -1;
        m = kNone;
        l = 0.f;
        started = false;
      }
      if (in_batch == 0) kv_warp_wait(kMfull + 8 * mr.at, mr.phase, kSiteKvFull);
      const float4* sc = scales + mr.at * 32 + in_batch * 8;
      if (walk.sees(lo, hi)) {
        kv_warp_wait(kSfull + 8 * q, sphase, kSiteKvFull);
        sphase ^= 1;
        tc::fence_after_sync();
        uint32_t raw[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) kv_ld<32>(ts + 32 * c, raw[c]);
        kv_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) kv_tie(raw[c]);
        const int64_t j0 = walk.j0();
        const bool edge = j0 + kKvTile - 1 > lo || (p.window && j0 <= (int64_t)hi - p.window);
        float top = -INFINITY;
        if (!edge) {
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float4 v = sc[g];
            auto s = [&](int k) { return __uint_as_float(raw[g >> 1][16 * (g & 1) + k]); };
            float a = max3(s(0), s(1), s(2)), b = max3(s(3), s(4), s(5));
            a = max3(a, s(6), s(7)), b = max3(b, s(8), s(9));
            a = max3(a, s(10), s(11)), b = max3(b, s(12), s(13));
            a = max3(a, s(14), s(15));
            top = fmaxf(top, fmaf(fmaxf(a, b), cq * v.x, v.y));
          }
        } else {
          // x in place of the score, minus infinity where the row does not see.
          const int high = (int)min((int64_t)kKvTile, place - j0);  // last position of the tile that the row sees
          const int low = p.window ? (int)max((int64_t)-1, min((int64_t)kKvTile, place - (int64_t)p.window - j0)) : -1;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const float4 v = sc[g];
            const float c = cq * v.x;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int at = 16 * g + k;
              const float x = at <= high && at > low ? fmaf(__uint_as_float(raw[g >> 1][16 * (g & 1) + k]), c, v.y) : -INFINITY;
              raw[g >> 1][16 * (g & 1) + k] = __float_as_uint(x);
              top = fmaxf(top, x);
            }
          }
        }
        if (__any_sync(0xFFFFFFFFu, top > m + kHeadroom)) {
          const float to = top > m + kHeadroom ? top : m, f = ex2(m - to);
          m = to;
          l *= f;
          if (started) {
            kv_warp_wait(kOdone + 8 * q, ophase, kSiteKvFull);
            tc::fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < p.cache.dim; c += 16) {
              uint32_t o[16];
              kv_ld<16>(to_ + c, o);
              kv_wait_ld();
              kv_tie(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tc::st_cols<16>(to_ + c, o);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float4 v = sc[2 * c + g];
            const float k = edge ? 1.f : cq * v.x, add = edge ? -m : v.y - m;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float a = add, b = add;
              fma2(a, b, __uint_as_float(raw[c][16 * g + 2 * i]), __uint_as_float(raw[c][16 * g + 2 * i + 1]), k, k);
              a = ex2(a);
              b = ex2(b);
              s0 += a;
              s1 += b;
              w[8 * g + i] = f16x2_of(a, b);
            }
            l = fmaf(s0 + s1, v.z, l);
          }
          tc::st_cols<16>(ts + 16 * c, w);
        }
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(kWfull + 8 * q);
        started = true;
        ophase ^= 1;
      }
      if (++in_batch == 4) {
        in_batch = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(kMfree + 8 * mr.at);
        mr.next(2);
      }

      if (walk.last() && kUnitRows * walk.u + kRows * q < walk.rows) {
        // The unit's end, or this CTA's part of it.
        if (started) {
          kv_warp_wait(kOdone + 8 * q, ophase, kSiteKvFull);
          tc::fence_after_sync();
        }
        const int unit0 = walk.x - walk.t, unit1 = unit0 + walk.tiles - 1;  // the unit's tiles
        const int row = kUnitRows * walk.u + kRows * q + r, t = row / p.group;
        const bool valid = row < walk.rows;
        const int64_t token = walk.first_token + t, head = walk.h * p.group + row - t * p.group;
        uint16_t* out = p.out + token * p.os_t + head * p.os_h;
        const bool vec = (uintptr_t)p.out % 16 == 0 && p.os_t % 8 == 0 && p.os_h % 8 == 0;
        auto store = [&](int d, const float (&v)[16]) {  // 16 dimensions of the thread's row
          uint32_t u[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
            u[k] = *reinterpret_cast<const uint32_t*>(&b);
          }
          if (!valid) return;
          if (vec) {
            reinterpret_cast<uint4*>(out + d)[0] = make_uint4(u[0], u[1], u[2], u[3]);
            reinterpret_cast<uint4*>(out + d)[1] = make_uint4(u[4], u[5], u[6], u[7]);
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) out[d + k] = (uint16_t)(u[k >> 1] >> (16 * (k & 1)));
          }
        };
        auto store_lse = [&](float top, float all) {
          if (valid && p.lse)
            p.lse[token * p.ls_t + head * p.ls_h] = all == 0.f ? -INFINITY : (top + log2f(all)) * 0.6931471805599453f;
        };
        const bool whole = unit0 >= x0 && unit1 < x1;
        const int cta0 = whole ? 0 : kv_owner(unit0, total, ctas), cta1 = whole ? 0 : kv_owner(unit1, total, ctas);
        auto part = [&](int cta) { return partials + ((int64_t)(cta * 2 + (cta == cta0)) * 2 + q) * kPart; };
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int d = 0; d < p.cache.dim; d += 16) {
          uint32_t o[16];
          float v[16];
          if (started) {
            kv_ld<16>(to_ + d, o);
            kv_wait_ld();
            kv_tie(o);
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = started ? __uint_as_float(o[k]) : 0.f;
          if (whole) {
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = l == 0.f ? 0.f : v[k] * inv;
            store(d, v);
          } else {
            float4* at = reinterpret_cast<float4*>(part(blockIdx.x)) + (d >> 2) * kRows + r;
#pragma unroll
            for (int k = 0; k < 4; ++k) __stcg(at + k * kRows, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
          }
        }
        tc::fence_before_sync();
        if (started) {
          __syncwarp();
          if (lane == 0) mbar_arrive(kOfree + 8 * q);
        }
        if (whole) {
          store_lse(m, l);
        } else {
          // Published. The last to arrive joins all parts, in the order of the positions.
          __stcg(part(blockIdx.x) + kRows * 128 + r, m);
          __stcg(part(blockIdx.x) + kRows * 129 + r, l);
          kv_bar_sync(1 + q, 128);  // orders the warps' stores before the counting thread's release
          if (r == 0) {
            begin[8 + q] = atomic_add_acq_rel_gpu(counters + 2 * cta0 + q, 1) == cta1 - cta0;
            if (begin[8 + q]) counters[2 * cta0 + q] = 0;  // all parts are in: zero again for the next launch
          }
          kv_bar_sync(1 + q, 128);
          if (begin[8 + q]) {
            float top = kNone, all = 0.f;
#pragma unroll 4
            for (int c = cta0; c <= cta1; ++c) top = fmaxf(top, __ldcg(part(c) + kRows * 128 + r));
#pragma unroll 4
            for (int c = cta0; c <= cta1; ++c)
              all = fmaf(ex2(__ldcg(part(c) + kRows * 128 + r) - top), __ldcg(part(c) + kRows * 129 + r), all);
            const float inv_all = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
            for (int d = 0; d < p.cache.dim; d += 16) {
              float v[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k] = 0.f;
#pragma unroll 2
              for (int c = cta0; c <= cta1; ++c) {
                const float f = ex2(__ldcg(part(c) + kRows * 128 + r) - top);
                const float4* at = reinterpret_cast<const float4*>(part(c)) + (d >> 2) * kRows + r;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float4 a = __ldcg(at + k * kRows);
                  v[4 * k] = fmaf(f, a.x, v[4 * k]);
                  v[4 * k + 1] = fmaf(f, a.y, v[4 * k + 1]);
                  v[4 * k + 2] = fmaf(f, a.z, v[4 * k + 2]);
                  v[4 * k + 3] = fmaf(f, a.w, v[4 * k + 3]);
                }
              }
#pragma unroll
              for (int k = 0; k < 16; ++k) v[k] = all == 0.f ? 0.f : v[k] * inv_all;
              store(d, v);
            }
            store_lse(top, all);
          }
          kv_bar_sync(1 + q, 128);  // before the flag is used again
        }
      }
      walk.next();
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 13) {
    tc::fence_after_sync();
    tc::dealloc(tmem, 512);
  }
}

size_t kv_prompt_partial_bytes(int sms) { return (size_t)sms * 4 * kPart * sizeof(float); }

cudaError_t launch_kv_prompt(const KvAttentionCall& p, const CUtensorMap& k, const CUtensorMap& v, int sms, float* partials,
                             int* counters, cudaStream_t stream) {
  const void* kernel = (const void*)kv_prompt_kernel;
  const cudaError_t e = ensure_smem_attribute(kernel, kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(sms), dim3(kThreads), kSmem, stream, p, k, v, partials, counters);
}

cudaError_t kv_prompt_status_symbols(void** status, void** limit) {
  const cudaError_t e = cudaGetSymbolAddress(status, g_device_status);
  return e != cudaSuccess ? e : cudaGetSymbolAddress(limit, g_wait_limit_ns);
}

}  // namespace mambo
