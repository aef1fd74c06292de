// Attention of many query rows over the paged FP8 cache: prompts and chunks of
// prompts, and any sequence whose rows (tokens times the query heads of a key
// head) are more than the decode kernel takes.
//
// A unit is 256 rows of one key head (row r of a sequence: token r / group,
// query head r % group) as two MMA tiles of 128, which share the keys and
// values that pass by. For each 64 positions and tile:
//   S [128 x 64] = Q K^T        8-bit MMAs, the queries in two exact terms (kv_tc.cuh)
//   O [128 x D] += W V          f16 MMAs, the weights W from TMEM (over S, which they replace)
// TMEM holds two S of 64 positions for each tile of rows (and O), so that one is
// filled while the softmax works on the other. With one S of 128 positions every
// tile waited for its MMAs in turn: 732 us for a prompt of 8192 tokens instead of
// 596, although scores of 64 positions read the queries from shared memory twice
// as often.
// Two 8-bit terms cost what one 16-bit product does and need no conversion of
// the keys. The values are converted to f16 (exactly) by a warpgroup of their
// own: weights in f16 have 11 bits, where two more terms would have cost the
// softmax, the busiest part, more instructions than the conversion is.
//
// A softmax thread has a row: no reductions over lanes. As in the decode kernel
// x = score * log2(e) + exponent of the position's value scale, w = 2^(x - m),
// l += w * 2^-exponent, and m moves (O is rescaled) only when weights pass 2^7
// to 2^11, which shows in their sums: the common tile has no pass for its
// maximum. What paces the kernel is the softmax: two of its warps share a
// scheduler and take some 3600 clocks for both tiles and 128 positions, of which
// the special function unit is busy 1800 (an eighth of the 2^x are polynomials:
// none, a quarter and a half took 602, 596 and 629 us where an eighth took 588)
// and the tensor core 2050 (2700 with what scores of 64 positions read from
// shared memory). 32 query heads over 8 key heads of 128, 8192 tokens of a
// prompt: 528 us, 1041 TFLOP/s, 0.63 of the measured rate of 16-bit products
// (584 us where calls follow larger ones, at the power limit).
//
// Work: all units' tiles in a row, one equal range per SM (units have unequal
// lengths under the causal mask, and there may be few of them). A unit that
// several CTAs share is joined by the last to arrive, in the order of the
// positions.
//
// Warps 0-3 and 4-7 softmax of either tile, and its queries; 8-11 values; 12 copies and the units to come, which it
// describes to the others; 13 and 14 the MMAs of either tile; 15 the pages' scales.
//
// Compiled as a whole program of its own (no relocatable device code): the compiler takes setmaxnreg into account only
// then. Without it the softmax's 128 registers were too few, and registers spilled to local memory come back from the L2,
// as the shared memory leaves next to no L1: that alone made a tile's softmax twice as long. So it has its own device
// status.
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
constexpr float kNone = -3e38f;       // m of a row that has seen nothing
constexpr float kMostSum = 2048.f;    // of 16 weights, before m is moved: f16 holds 2^16
constexpr float kMostPoly = 100.f;    // of the exponents that the polynomial takes: a larger one would not show in its sum
// What a unit costs besides its tiles, in tiles: where the ranges of the CTAs are cut, units count as this much longer.
// Its queries, first scores, masked halves and results. Prompt of 8192 tokens and a mixed step:
// 3 557 and 110 us, 4 533 and 105, 5 529 and 114, 6 529 and 109 to 114 (the mixed step with its 31 us of the decode kernel).
constexpr int kUnitCost = 6;

// Shared memory: queries [2 tiles][hi, lo][128][128], keys, values as they come and in f16 [2 halves of D][128][128 bytes].
constexpr uint32_t kQ = 4 * kKvTileBytes, kVf = 2 * kKvTileBytes;
constexpr uint32_t kAtK = kQ, kAtV = kAtK + kKStages * kKvTileBytes, kAtVf = kAtV + kVStages * kKvTileBytes;
// Of each softmax warp 2 KB: rows' factors, and results on their way out.
constexpr uint32_t kAtStage = kAtVf + 2 * kVf, kAtScales = kAtStage + 8 * 2048, kAtUnits = kAtScales + 2 * 32 * 16;
constexpr int kUnitStages = 4;
constexpr uint32_t kAtBegin = kAtUnits + (kUnitStages + 1) * 96, kAtBars = kAtBegin + 128;
constexpr int kNumBars = 2 * kKStages + 2 * kVStages + 4 + 14 + 4 + 4 + 2 * kUnitStages;
constexpr uint32_t kSmem = 1024 + kAtBars + kNumBars * 8 + 16;
constexpr int kPart = kRows * 130;    // floats of a tile's part: O [32][128][4], m, l

// A CTA's part of a unit, as one warp works it out and the others read it.
struct alignas(16) Unit {
  int tile, n;        // tiles [tile, tile + n) of the sequence's positions; n == 0: there is no further unit
  int b, h;           // sequence, key head
  int row0, rows;     // the unit's first row, all rows of the sequence
  int token, place0;  // the sequence's first token and its position
  int lo[2], hi[2];   // positions of the first and last rows of either tile of rows
  int from[2], to[2]; // tiles that any of them sees: [from, to)
  int x, tiles;       // the unit's tiles in the work: [x, x + tiles); this part is all of it where n == tiles
  __device__ __forceinline__ bool has(int q) const { return row0 + kRows * q < rows; }
};
static_assert(sizeof(Unit) <= 96, "shared memory");

// The units of a call: sequence b, key head h, unit u of `units` of that head.
struct Plan {
  const KvAttentionCall& p;
  int b, h, u, units, token, place0, rows;
  __device__ __forceinline__ void sequence() {
    const KvSpan s = kv_span(p.seq, b);
    token = s.first;
    rows = (int64_t)s.count * p.group > p.few ? s.count * p.group : 0;
    place0 = kv_length(p.seq, b, p.cache.page) - s.count;
    units = (rows + kUnitRows - 1) / kUnitRows;
  }
  __device__ __forceinline__ int place(int row) const { return place0 + min(row, rows - 1) / p.group; }
  // Tiles of positions of unit i, at least one (of masked ones), and the first of them.
  __device__ __forceinline__ int tiles_of(int i, int& first) const {
    const int64_t low = p.window ? place(kUnitRows * i) + 1 - (int64_t)p.window : 0;
    first = low > 0 ? (int)(low / kKvTile) : 0;
    const int high = place(kUnitRows * i + kUnitRows - 1);
    return max((high >= 0 ? high / kKvTile + 1 : 0) - first, 1);
  }
  // Its share of the work: the tiles come last.
  __device__ __forceinline__ int cost_of(int i) const {
    int first;
    return tiles_of(i, first) + kUnitCost;
  }
  __device__ __forceinline__ void next() {
    if (++u < units) return;
    u = 0;
    if (++h < p.cache.heads) return;
    h = 0;
    do {
      ++b;
      sequence();
    } while (rows == 0);  // called only where there is one
  }
};

// Half a tile's S = Q K^T, 64 positions: head size up to 64 or 128, two terms of A.
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b, bool wide, uint32_t done) {
  constexpr uint32_t kId = tc::idesc_e4m3_f32(kRows, kKvTile / 2);
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
// Half a tile's O (+)= W V, 64 positions: weights f16 at TMEM column w (8 columns for 16 positions), values f16 along N (16 positions in
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
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t}" ::"r"(d),
      "r"(w), "r"(v), "r"(idesc), "r"(acc), "r"(desc_high(1024, true)), "r"(done)
      : "memory");
}

// Packed FP32 pairs in 64-bit registers.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float low_of(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high_of(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
// 2^x of a pair in the FMA pipe, which has room where the special function unit has none. x = n + f with n the nearest
// integer (read off the low bits of x + 1.5 * 2^23), f in [-1/2, 1/2]; 2^f is the minimax polynomial of degree 4 (by
// Remez' exchange, relative error 2.6e-6); n is added to its exponent, which holds for x up to 127: `top` tells the caller.
// Below -126 x counts as that.
__device__ __forceinline__ uint64_t ex2_poly(uint64_t x, float& top) {
  float a, b;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(low_of(x)), "f"(-126.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(high_of(x)), "f"(-126.f));
  asm("max.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(a), "f"(b));
  x = pack2(a, b);
  const uint64_t n = add_2(x, pack2(12582912.f, 12582912.f));
  const uint64_t f = add_2(x, fma_2(n, pack2(-1.f, -1.f), pack2(12582912.f, 12582912.f)));
  uint64_t y = fma_2(pack2(0.009570102f, 0.009570102f), f, pack2(0.05591786f, 0.05591786f));
  y = fma_2(y, f, pack2(0.24024744f, 0.24024744f));
  y = fma_2(y, f, pack2(0.6931218f, 0.6931218f));
  y = fma_2(y, f, pack2(0.9999993f, 0.9999993f));
  return pack2(__uint_as_float((uint32_t)y + ((uint32_t)n << 23)), __uint_as_float((uint32_t)(y >> 32) + ((uint32_t)(n >> 32) << 23)));
}

}  // namespace

__global__ void __launch_bounds__(kThreads, 1)
    kv_prompt_kernel(const __grid_constant__ KvAttentionCall p, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, float* partials, int* counters) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float4* scales = reinterpret_cast<float4*>(sm + kAtScales);   // [2][4 tiles][8]: key factor, value exponent, 2^-exponent
  Unit* units = reinterpret_cast<Unit*>(sm + kAtUnits);         // [kUnitStages], and an empty one
  int* begin = reinterpret_cast<int*>(sm + kAtBegin);           // where the share begins: sequence, head, unit, place in its work; [8] flags
  int* warp_sums = begin + 16;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + kAtBars);
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  const uint32_t sm0 = smem_u32(sm);
  const uint32_t kKfull = smem_u32(bars), kKfree = kKfull + 8 * kKStages, kVfull = kKfree + 8 * kKStages;
  const uint32_t kVfree = kVfull + 8 * kVStages, kFfull = kVfree + 8 * kVStages, kFfree = kFfull + 16;  // values in f16
  const uint32_t kSfull = kFfree + 16, kWfull = kSfull + 32, kOdone = kWfull + 32, kOfree = kOdone + 32;
  const uint32_t kQfull = kOfree + 16, kQfree = kQfull + 16, kMfull = kQfree + 16, kMfree = kMfull + 16;
  const uint32_t kUfull = kMfree + 16, kUfree = kUfull + 8 * kUnitStages;
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(kKfull + 8 * s, 1);
      mbar_init(kKfree + 8 * s, 2);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(kVfull + 8 * s, 1);
      mbar_init(kVfree + 8 * s, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(kFfull + 8 * i, 4);
      mbar_init(kFfree + 8 * i, 2);
      mbar_init(kSfull + 16 * i, 1);  // of either tile of rows: two halves
      mbar_init(kSfull + 16 * i + 8, 1);
      mbar_init(kWfull + 16 * i, 4);
      mbar_init(kWfull + 16 * i + 8, 4);
      mbar_init(kOdone + 16 * i, 1);
      mbar_init(kOdone + 16 * i + 8, 1);
      mbar_init(kOfree + 8 * i, 4);
      mbar_init(kMfull + 8 * i, 1);
      mbar_init(kMfree + 8 * i, 8);
    }
    for (int i = 0; i < kUnitStages; ++i) {
      mbar_init(kUfull + 8 * i, 1);
      mbar_init(kUfree + 8 * i, 15);  // MMAs, scales, 4 warps of values, 8 of the softmax
    }
    units[kUnitStages] = Unit{};
    for (int i = 0; i < 2; ++i) {
      mbar_init(kQfull + 8 * i, 4);
      mbar_init(kQfree + 8 * i, 1);
    }
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
  // Also behind the decode kernel of the same call, with which it shares nothing but the arguments: those are what kernels before
  // that one have just written (cache, scales, lengths, queries), and only this wait makes their writes visible here.
  pdl_wait();
  pdl_launch_dependents();
  // The whole work, and where this CTA's share begins: a warp has a run of sequences, a lane every 32nd unit of one.
  const int each = (p.seq.batch + 15) / 16, mine0 = min(p.seq.batch, warp * each), mine1 = min(p.seq.batch, mine0 + each);
  Plan plan{p, 0, 0, 0, 0, 0, 0, 0};
  auto cost_of_head = [&](int b) {
    plan.b = b;
    plan.sequence();
    int n = 0;
    for (int i = lane; i < plan.units; i += 32) n += plan.cost_of(i);
#pragma unroll
    for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    return n;
  };
  int sum = 0;
  for (int b = mine0; b < mine1; ++b) sum += cost_of_head(b) * p.cache.heads;
  if (lane == 0) warp_sums[warp] = sum;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = (uint32_t)__shfl_sync(0xFFFFFFFFu, (int)*slot, 0);
  int total = 0, before = 0;
  #pragma unroll 1
  for (int w = 0; w < 16; ++w) {
    total += warp_sums[w];
    before += w < warp ? warp_sums[w] : 0;
  }
  // Each share is a tile at least, so that of the CTAs between a unit's first and last tile each has one: those are all
  // that the join waits for.
  const int ctas = max(1, min((int)gridDim.x, total));
  const bool has = (int)blockIdx.x < ctas;
  const int x0 = has ? (int)((int64_t)blockIdx.x * total / ctas) : 0;
  const int x1 = has ? (int)(((int64_t)blockIdx.x + 1) * total / ctas) : 0;
  if (x0 < x1 && x0 >= before && x0 < before + sum) {
    int b = mine0, n;
    while (x0 >= before + (n = cost_of_head(b)) * p.cache.heads) {
      before += n * p.cache.heads;
      ++b;
    }
    const int h = (x0 - before) / n;
    int rest = (x0 - before) % n;  // what comes before in the head
    for (int i0 = 0;; i0 += 32) {
      const int mine = i0 + lane < plan.units ? plan.cost_of(i0 + lane) : 0;
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
      if (rest < all || i0 + 32 >= plan.units) break;
      rest -= all;
    }
  }
  __syncthreads();
  // The next unit of this CTA, told by its ring's barrier; a role gives it back once it is through with it.
  auto unit_of = [&](const KvRing& ring) -> const Unit& {
    return units[kv_wait(kUfull + 8 * ring.at, ring.phase, kSiteKvFull) ? ring.at : kUnitStages];
  };
  const int log_page = p.cache.log_page, per_tile = kKvTile >> log_page;

  // Register split, launched with 128 a thread: 256 x 176 + 256 x 80 = 512 x 128.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 12) {
      // ------------------------------------------------------------ copies, and the units
      KvRing kr, vr, ur;
      const uint64_t policy = l2_policy_evict_last();
      bool ok = true;
      plan.b = begin[0];
      plan.h = begin[1];
      plan.u = begin[2];
      if (x0 < x1) plan.sequence();
      int x = x0, at = begin[3];  // place in the work, and in the unit's
      int count = 0;
      // The next unit of this CTA's share (one with n == 0 behind the last), told to the others.
      auto unit_ahead = [&]() {
        Unit u{};
        if (x < x1) {
          u.tiles = plan.tiles_of(plan.u, u.tile);
          const int t = max(at - kUnitCost, 0), left = x1 - x - max(kUnitCost - at, 0);
          u.x = x - at + kUnitCost;
          u.n = max(min(u.tiles - t, left), 0);  // of the last unit only the work besides its tiles may fall to this CTA
          x = u.x + u.tiles;
          at = 0;
          u.tile += t;
          u.b = plan.b;
          u.h = plan.h;
          u.row0 = kUnitRows * plan.u;
          u.rows = plan.rows;
          u.token = plan.token;
          u.place0 = plan.place0;
          for (int q = 0; q < 2; ++q) {
            if (!u.has(q)) continue;
            u.lo[q] = plan.place(u.row0 + kRows * q);
            u.hi[q] = plan.place(u.row0 + kRows * q + kRows - 1);
            const int64_t low = p.window ? u.lo[q] + 1 - (int64_t)p.window : 0;
            u.from[q] = low > 0 ? (int)(low / kKvTile) : 0;
            u.to[q] = u.hi[q] >= 0 ? u.hi[q] / kKvTile + 1 : 0;
          }
          if (x < x1) plan.next();
        }
        if (count >= kUnitStages && !(ok = kv_warp_wait(kUfree + 8 * ur.at, ur.phase ^ 1, kSiteKvEmpty))) u.n = 0;
        if (lane == 0) {
          units[ur.at] = u;
          mbar_arrive(kUfull + 8 * ur.at);
        }
        // The unit's queries on their way to the L2; those of the first are fetched at once.
        if (count > 0 && u.n > 0) {
#pragma unroll 1
          for (int i = lane; i < kUnitRows && u.row0 + i < u.rows; i += 32) {
            const int row = u.row0 + i, tok = row / p.group;
            bulk_prefetch_l2(p.q + (int64_t)(u.token + tok) * p.qs_t + (int64_t)(u.h * p.group + row - tok * p.group) * p.qs_h, p.cache.dim * 2);
          }
        }
        ur.next(kUnitStages);
        ++count;
        return u;
      };
      Unit ahead = unit_ahead();
      for (int it = 0; ok && ahead.n > 0;) {
        const Unit u = ahead;
        const int n = u.n, h = u.h;
        const int64_t i0 = (int64_t)u.tile * per_tile + lane;
        const int* row_pages = p.seq.table + u.b * p.seq.table_stride + i0;
        auto page_of = [&](int t) {
          return t < n && lane < per_tile && i0 + t * per_tile < p.seq.table_pages ? __ldg(row_pages + t * per_tile) : -1;
        };
        int page = page_of(0);
        for (int t = 0; t < n; ++t, ++it) {
          const int next_page = page_of(t + 1);
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
          if (t == 0) ahead = unit_ahead();  // the next unit, behind the first loads of this one
          if (!ok) break;
        }
      }
      if (!ok) kv_settle();
    } else if (warp < 15) {
      // ------------------------------------------------------------ MMA: a thread for each tile of rows. A tile's weights
      // lie over its scores, and its next scores over them: in the order in which they are issued.
      if (tm::elect_one()) {
        const int q = warp - 13;
        const uint32_t idesc_o = tc::idesc_f16_f32(kRows, p.cache.dim) | kIdescAlongN;
        const bool wide = p.cache.dim > 64;
        const uint32_t ds = tmem + q * 128, dout = ds + 256, a = desc_low(sm0 + q * 2 * kKvTileBytes, 16);
        const uint32_t k0 = desc_low(sm0 + kAtK, 16), v0 = desc_low(sm0 + kAtVf, kKvTileBytes);
        const uint32_t sfull = kSfull + 16 * q, wfull = kWfull + 16 * q, odone = kOdone + 16 * q, ofree = kOfree + 8 * q;
        const uint32_t qfull = kQfull + 8 * q, qfree = kQfree + 8 * q;
        KvRing kr, fr, ur;
        uint32_t qphase = 0, wphase = 0, ophase = 1;
        // The tile whose scores come next, one ahead of the tile whose values do: the unit's tiles left, and those that
        // these rows see.
        int tile = 0, left = 0, from = 0, to = 0;
        bool begins = true;  // at a unit's first tile
        auto enter = [&]() {
          const Unit& u = unit_of(ur);
          tile = u.tile;
          left = u.n;
          from = u.from[q];
          to = u.to[q];
          if (left > 0) mbar_arrive(kUfree + 8 * ur.at);
          ur.next(kUnitStages);
          begins = true;
        };
        bool ok = true;
        bool seen = false;  // whether these rows see the tile
        auto scores = [&](int half) {
          if (seen) {
            tc::fence_after_sync();
            mma_scores(ds + 64 * half, a, k0 + kr.at * (kKvTileBytes >> 4) + half * (kKvTileBytes >> 5), wide, sfull + 8 * half);
          }
          if (half == 0) return;
          tc::commit(kKfree + 8 * kr.at);
          kr.next(kKStages);
          ++tile;
          if (--left == 0) {
            tc::commit(qfree);
            enter();
          }
        };
        auto both = [&]() {  // a unit's first tile
          ok = kv_wait(qfull, qphase, kSiteKvFull) && kv_wait(kKfull + 8 * kr.at, kr.phase, kSiteKvFull);
          qphase ^= 1;
          begins = false;
          seen = tile >= from && tile < to;
          if (!ok) return;
          scores(0);
          scores(1);
        };
        enter();
        bool started = false, ends = left == 1, some = left > 0;
        if (some) both();
        while (ok && some) {
          // Half a tile's values, and over its weights the scores of the next tile's half: the softmax works on the other
          // half meanwhile. A next unit's queries may still be on their way; then its scores come at the end.
          const bool last = ends, go = seen;
          some = left > 0;
          ends = left == 1;
          const bool next = some && !begins;
          ok = kv_wait(kFfull + 8 * fr.at, fr.phase, kSiteKvFull);
          if (ok && next) ok = kv_wait(kKfull + 8 * kr.at, kr.phase, kSiteKvFull);
          // The softmax has read the last unit's O.
          if (ok && go && !started) {
            ok = kv_wait(ofree, ophase, kSiteKvEmpty);
            ophase ^= 1;
          }
          if (next) seen = tile >= from && tile < to;
          const uint32_t values = v0 + fr.at * (kVf >> 4);
          if (go) {
            ok = ok && kv_wait(wfull, wphase, kSiteKvFull);
            if (!ok) break;
            tc::fence_after_sync();
            mma_values(dout, ds, values, idesc_o, started, odone);
          }
          if (!ok) break;
          if (next) scores(0);
          if (go) {
            if (!(ok = kv_wait(wfull + 8, wphase, kSiteKvFull))) break;
            wphase ^= 1;
            tc::fence_after_sync();
            mma_values(dout, ds + 64, values + 512, idesc_o, 1, odone + 8);
            started = true;
          }
          tc::commit(kFfree + 8 * fr.at);
          fr.next(2);
          if (last) started = false;
          if (next) scores(1);
          if (some && !next) both();
        }
        if (!ok) kv_settle();
      }
    } else {
      // ------------------------------------------------------------ scales: four tiles at a time, 16 positions a lane
      KvRing ring, ur;
      int step = 0, fill = 0;  // tiles in the current batch
      int64_t at = -1;         // of this lane's tile: place in the table; and its head
      int head = 0;
      auto publish = [&]() {
        const int page = at >= 0 ? __ldg(p.seq.table + at) : -1;
        float4 v = make_float4(0.f, -INFINITY, 0.f, 0.f);  // positions without a page: x is minus infinity
        if (page >= 0 && page < p.cache.pages) {
          const int64_t row = (int64_t)page * p.cache.heads + head;
          const uint32_t kc = max((uint32_t)__ldg(p.cache.scales[0] + row), kKvMinCode);
          const uint32_t vc = max((uint32_t)__ldg(p.cache.scales[1] + row), kKvMinCode);
          v = make_float4(kc == 255u ? NAN : e8m0_to_float(kc), vc == 255u ? NAN : (float)((int)vc - 127),
                          vc == 255u ? 1.f : e8m0_to_float(254u - vc), 0.f);
        }
        if (step >= 2) kv_warp_wait(kMfree + 8 * ring.at, ring.phase ^ 1, kSiteKvEmpty);
        ++step;
        scales[ring.at * 32 + lane] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(kMfull + 8 * ring.at);
        ring.next(2);
        fill = 0;
        at = -1;
      };
      for (;;) {
        const Unit& unit = unit_of(ur);
        const int n = unit.n, tile = unit.tile, b = unit.b, h = unit.h;
        if (n <= 0) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(kUfree + 8 * ur.at);
        ur.next(kUnitStages);
        for (int t = 0; t < n;) {
          const int take = min(4 - fill, n - t), mine = (lane >> 3) - fill;  // tiles t .. t + take - 1 join the batch
          if (mine >= 0 && mine < take) {
            const int64_t k = ((int64_t)(tile + t + mine) * kKvTile + 16 * (lane & 7)) >> log_page;
            at = k < p.seq.table_pages ? b * p.seq.table_stride + k : -1;
            head = h;
          }
          t += take;
          fill += take;
          if (fill == 4) publish();
        }
      }
      if (fill) publish();
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // -------------------------------------------------------------- values
    const int i = threadIdx.x - 256;  // position of the tile
    KvRing vr, fr, ur;
    int it = 0;
    for (;;) {
      const Unit& unit = unit_of(ur);
      const int n = unit.n;
      if (n <= 0) break;
      // A position that no row sees: its value may be anything, and zero times NaN is NaN.
      const int64_t above = unit.has(1) ? unit.hi[1] : unit.hi[0], below = p.window ? (int64_t)unit.lo[0] - p.window : -1;
      int64_t j = (int64_t)unit.tile * kKvTile + i;
      __syncwarp();
      if (lane == 0) mbar_arrive(kUfree + 8 * ur.at);
      ur.next(kUnitStages);
      for (int tile = 0; tile < n; ++tile, ++it, j += kKvTile) {
        const bool none = j > above || j <= below;
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
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // -------------------------------------------------------------- softmax
    const int q = warp >> 2, r = threadIdx.x & 127;
    const uint32_t ts = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + q * 128, to_ = ts + 256;
    uint8_t* stage = sm + kAtStage + warp * 2048;
    KvRing mr, ur;
    int in_batch = 0;
    uint32_t sphase = 0;              // of the tile: its scores, and the MMAs on its values
    uint32_t qphase = 1;              // a fresh barrier's previous phase counts as over
    // Of the unit's queries this warp's 32 rows, split into two terms, to shared memory: a half warp a row, eight dimensions
    // a lane. The rows come as they are to where their terms go (a row of bf16 is as large as both), all at once and
    // asynchronously, and are split in place. The factor of this thread's row is returned; minus zero stands for a row that is
    // not finite, whose sum becomes NaN at the unit's end if it sees anything.
    const int step_t = 2 / p.group, step_h = 2 - step_t * p.group;  // two rows on: tokens and heads
    auto queries = [&](const Unit& u) {
      const int c = lane & 15, r0 = 32 * (warp & 3) + (lane >> 4);
      const int rows = 8 * c < p.cache.dim ? u.rows - u.row0 - kRows * q : 0;
      const int row = u.row0 + kRows * q + r0;
      const int t = row / p.group;
      int hh = row - t * p.group;
      // Two rows on: step_t tokens and step_h query heads, and where that passes the group another token and a group back.
      const int64_t on = step_t * p.qs_t + step_h * p.qs_h, wrap = p.qs_t - p.group * p.qs_h;
      const uint16_t* from = p.q + (int64_t)(u.token + t) * p.qs_t + (int64_t)(u.h * p.group + hh) * p.qs_h + 8 * c;
      // Chunk c of a row: eight in the first term's place, eight in the second's.
      const uint32_t tile0 = q * 2 * kKvTileBytes, mine = tile0 + (c >> 3) * kKvTileBytes;
#pragma unroll 4
      for (int r1 = r0; r1 < r0 + 32; r1 += 2) {
        const bool have = r1 < rows;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm0 + mine + r1 * 128 + (((c ^ r1) & 7) << 4)),
                     "l"(have ? from : p.q), "r"(have ? 16 : 0)
                     : "memory");
        hh += step_h;
        const bool over = hh >= p.group;
        from += over ? on + wrap : on;
        hh -= over ? p.group : 0;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      // A lane has a row: no shuffles, and one scale for it. (With 16 lanes a row this took 6000 clocks and more, and the
      // prompt of 8192 tokens 590 us for 575.) In loops, because a short call is paced by the fetch of its instructions: all
      // at once from registers took 5400 clocks there.
      const int r1 = 32 * (warp & 3) + lane;
      uint8_t* const to = sm + tile0 + r1 * 128;
      uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll 2
      for (int i = 0; i < 16; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(to + (i >> 3) * kKvTileBytes + (((i ^ r1) & 7) << 4));
        top[0] = absmax_bf16x2(top[0], x.x), top[1] = absmax_bf16x2(top[1], x.y);
        top[2] = absmax_bf16x2(top[2], x.z), top[3] = absmax_bf16x2(top[3], x.w);
      }
      top[0] = absmax_bf16x2(absmax_bf16x2(top[0], top[1]), absmax_bf16x2(top[2], top[3]));
      const uint32_t code = bf16_scale_code(max(top[0] & 0x7FFFu, (top[0] >> 16) & 0x7FFFu));
      const bool bad = code == 255u;
      const float inv = bad ? 0.f : e8m0_to_float(254u - code);
      // 16 dimensions d at a time: chunks 2d and 2d + 1 of the row as it came, of which the first terms go to chunk d and the
      // second ones to chunk 8 + d. In the order 0 to 3, 7 to 4 no chunk is written that is still to be read, but for the
      // second terms of 0 to 3, which wait in the stage.
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const int d = i < 4 ? i : 11 - i;
        uint32_t v[8], h[4], l[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c2 = 2 * d + k;
          const uint4 x = *reinterpret_cast<const uint4*>(to + (c2 >> 3) * kKvTileBytes + (((c2 ^ r1) & 7) << 4));
          v[4 * k] = x.x, v[4 * k + 1] = x.y, v[4 * k + 2] = x.z, v[4 * k + 3] = x.w;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // 8 significant bits up to 448: exact in f16 (down to 2^-17), and so is what the first term leaves.
          const uint32_t x = v[2 * k], y = v[2 * k + 1];
          const uint32_t e0 = f16x2_of(__uint_as_float(x << 16) * inv, __uint_as_float(x & 0xFFFF0000u) * inv);
          const uint32_t e1 = f16x2_of(__uint_as_float(y << 16) * inv, __uint_as_float(y & 0xFFFF0000u) * inv);
          const uint32_t h0 = e4m3x2_of_f16x2(e0), h1 = e4m3x2_of_f16x2(e1);
          h[k] = bad ? 0u : h0 | (h1 << 16);
          l[k] = bad ? 0u : e4m3x2_of_f16x2(sub_f16x2(e0, f16x2_of_e4m3x2(h0))) | (e4m3x2_of_f16x2(sub_f16x2(e1, f16x2_of_e4m3x2(h1))) << 16);
        }
        const int at = ((d ^ r1) & 7) << 4;
        *reinterpret_cast<uint4*>(to + at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(i < 4 ? stage + d * 512 + lane * 16 : to + kKvTileBytes + at) = make_uint4(l[0], l[1], l[2], l[3]);
      }
#pragma unroll
      for (int d = 0; d < 4; ++d)
        *reinterpret_cast<uint4*>(to + kKvTileBytes + (((d ^ r1) & 7) << 4)) = *reinterpret_cast<const uint4*>(stage + d * 512 + lane * 16);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(kQfull + 8 * q);
      return bad ? -0.f : p.scale * 1.4426950408889634f * e8m0_to_float(code);
    };
    // Through the units, one behind: the next one's queries are on their way before this one's results are waited for.
    float m = kNone, l = 0.f, cq = 0.f;
    int n = 0, first = 0, from = 0, end = 0, lo = 0, hi = 0, place = -1;
    bool started = false;
    for (;;) {
      for (int tile = first, left = n; left > 0; ++tile, --left) {
        if (in_batch == 0) kv_warp_wait(kMfull + 8 * mr.at, mr.phase, kSiteKvFull);
        const float4* sc = scales + mr.at * 32 + in_batch * 8;
        if (tile >= from && tile < end) {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            const uint32_t th = ts + 64 * half;
            const float4* sh = sc + 4 * half;
            kv_warp_wait(kSfull + 16 * q + 8 * half, sphase, kSiteKvFull);
            tc::fence_after_sync();
            const int64_t j0 = (int64_t)tile * kKvTile + 64 * half;
            const bool edge = j0 + 63 > lo || (p.window && j0 <= (int64_t)hi - p.window);
            bool plain = started && !edge;
            if (plain) {
              // One pass with m as it is. A weight that is too large shows in the sums; then the half is done over.
              uint32_t w[32];
              float sum = 0.f, most = 0.f, top = 0.f;
              uint32_t raw[2][32];
              kv_ld<32>(th, raw[0]);
              kv_ld<32>(th + 32, raw[1]);
              kv_wait_ld();
              kv_tie(raw[0]);
              kv_tie(raw[1]);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                  const float4 v = sh[2 * c + g];
                  const uint64_t k2 = pack2(cq * v.x, cq * v.x), add2 = pack2(v.y - m, v.y - m);
                  uint64_t sum2 = 0;
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const int at = 16 * g + 2 * i;
                    const uint64_t x = fma_2(pack2(__uint_as_float(raw[c][at]), __uint_as_float(raw[c][at + 1])), k2, add2);
                    const uint64_t e = i == 3 ? ex2_poly(x, top) : pack2(ex2(low_of(x)), ex2(high_of(x)));
                    sum2 = add_2(sum2, e);
                    w[16 * c + 8 * g + i] = f16x2_of(low_of(e), high_of(e));
                  }
                  const float part = low_of(sum2) + high_of(sum2);
                  most = fmaxf(most, part);
                  sum = fmaf(part, v.z, sum);
                }
              }
              plain = !__any_sync(0xFFFFFFFFu, most > kMostSum || top > kMostPoly);
              if (plain) {
                l += sum;
                tc::st_cols<32>(th, w);
              }
            }
            if (!plain) {
              // Masks, or m moves. The positions that the row sees, a bit each; their x, minus infinity for the others, and the
              // largest of them. (Two passes over TMEM, 16 scores at a time, took 3800 clocks where a plain half takes 1200,
              // and the prompt of 8192 tokens 575 us for 551.)
              const int64_t behind = place + 1 - j0;
              const int high = (int)max((int64_t)0, min((int64_t)64, behind));
              const int low = p.window ? (int)max((int64_t)0, min((int64_t)64, behind - p.window)) : 0;
              const uint64_t bits = (high < 64 ? (1ull << high) - 1 : ~0ull) & (low < 64 ? ~0ull << low : 0ull);
              const uint32_t seen[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
              uint32_t x[2][32];
              kv_ld<32>(th, x[0]);
              kv_ld<32>(th + 32, x[1]);
              kv_wait_ld();
              kv_tie(x[0]);
              kv_tie(x[1]);
              float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float4 v = sh[g];
                const float c = cq * v.x;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  uint32_t& at = x[g >> 1][16 * (g & 1) + k];
                  const bool in = (g < 2 ? seen[0] : seen[1]) >> (16 * (g & 1) + k) & 1;
                  at = in ? __float_as_uint(fmaf(__uint_as_float(at), c, v.y)) : 0xFF800000u;
                  t4[k & 3] = fmaxf(t4[k & 3], __uint_as_float(at));
                }
              }
              const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
              const float up = fmaxf(m, top), f = ex2(m - up);
              m = up;
              l *= f;
              if (started) {
                // The half before: this tile's first, or the last tile's second.
                kv_warp_wait(kOdone + 16 * q + 8 * (half ^ 1), sphase ^ half ^ 1, kSiteKvFull);
                tc::fence_after_sync();
                if (__any_sync(0xFFFFFFFFu, f != 1.f)) {
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
              // x first and then less m: the row's largest is 2^0 exactly, however large its score and its rounding are.
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                  uint32_t (&at)[32] = x[g >> 1];
                  const float e0 = ex2(__uint_as_float(at[16 * (g & 1) + k]) - m), e1 = ex2(__uint_as_float(at[16 * (g & 1) + k + 1]) - m);
                  sum0 += e0;
                  sum1 += e1;
                  x[0][8 * g + (k >> 1)] = f16x2_of(e0, e1);  // behind what has been read
                }
                l = fmaf(sum0 + sum1, sh[g].z, l);
              }
              tc::st_cols<32>(th, x[0]);
            }
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(kWfull + 16 * q + 8 * half);
            started = true;
          }
          sphase ^= 1;
        }
        if (++in_batch == 4) {
          in_batch = 0;
          __syncwarp();
          if (lane == 0) mbar_arrive(kMfree + 8 * mr.at);
          mr.next(2);
        }
      }

      // The next unit's queries, before this one's results are waited for.
      KvRing after = ur;
      if (n > 0) after.next(kUnitStages);
      const Unit& next = unit_of(after);
      float next_cq = 0.f;
      if (next.n > 0) {
        kv_warp_wait(kQfree + 8 * q, qphase, kSiteKvEmpty);
        qphase ^= 1;
        next_cq = queries(next);
      }
      const Unit& unit = units[ur.at];
      if (n > 0 && unit.has(q)) {
        // The unit's end, or this CTA's part of it.
        if (started) {
          kv_warp_wait(kOdone + 16 * q, sphase ^ 1, kSiteKvFull);
          kv_warp_wait(kOdone + 16 * q + 8, sphase ^ 1, kSiteKvFull);
          tc::fence_after_sync();
        }
        const int row = unit.row0 + kRows * q + r, t = row / p.group;
        const int64_t token = unit.token + t, head = unit.h * p.group + row - t * p.group;
        const int64_t out_at = row < unit.rows ? token * p.os_t + head * p.os_h : -1;
        // 32 dimensions of the warp's rows to memory, through the stage: 64 bytes of each of eight rows at a time.
        auto store = [&](int c, const float (&v)[32]) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * k + 2 * i], v[8 * k + 2 * i + 1]);
              u[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int rr = (lane >> 2) + 8 * k, d = c + 8 * (lane & 3);
            const int64_t at = __shfl_sync(0xFFFFFFFFu, out_at, rr);
            const uint4 u = *reinterpret_cast<const uint4*>(stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4));
            if (at >= 0 && d < p.cache.dim) *reinterpret_cast<uint4*>(p.out + at + d) = u;
          }
        };
        auto store_lse = [&](float top, float all) {
          if (out_at >= 0 && p.lse)
            p.lse[token * p.ls_t + head * p.ls_h] = all == 0.f ? -INFINITY : (top + log2f(all)) * 0.6931471805599453f;
        };
        const bool whole = n == unit.tiles;
        const int cta0 = whole ? 0 : kv_owner(unit.x, total, ctas);
        const int cta1 = whole ? 0 : kv_owner(unit.x + unit.tiles - 1, total, ctas);
        auto part = [&](int cta) { return partials + ((int64_t)(cta * 2 + (cta == cta0)) * 2 + q) * kPart; };
        if (l != 0.f && __float_as_uint(cq) == 0x80000000u) l = NAN;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint32_t o[32];
        if (started) kv_ld<32>(to_, o);
#pragma unroll 1
        for (int c = 0; c < p.cache.dim; c += 32) {
          float v[32];
          if (started) kv_wait_ld();
          kv_tie(o);
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = started ? __uint_as_float(o[k]) : 0.f;
          if (started && c + 32 < p.cache.dim) kv_ld<32>(to_ + c + 32, o);
          if (whole) {
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = l == 0.f ? 0.f : v[k] * inv;
            store(c, v);
          } else {
            float4* at = reinterpret_cast<float4*>(part(blockIdx.x)) + (c >> 2) * kRows + r;
#pragma unroll
            for (int k = 0; k < 8; ++k) __stcg(at + k * kRows, make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
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
            for (int k = cta0; k <= cta1; ++k) top = fmaxf(top, __ldcg(part(k) + kRows * 128 + r));
#pragma unroll 4
            for (int k = cta0; k <= cta1; ++k)
              all = fmaf(ex2(__ldcg(part(k) + kRows * 128 + r) - top), __ldcg(part(k) + kRows * 129 + r), all);
            const float inv_all = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
            for (int c = 0; c < p.cache.dim; c += 32) {
              float v[32];
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = 0.f;
#pragma unroll 1
              for (int k = cta0; k <= cta1; ++k) {
                const float f = ex2(__ldcg(part(k) + kRows * 128 + r) - top) * inv_all;
                const float4* at = reinterpret_cast<const float4*>(part(k)) + (c >> 2) * kRows + r;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float4 a = __ldcg(at + i * kRows);
                  v[4 * i] = fmaf(f, a.x, v[4 * i]);
                  v[4 * i + 1] = fmaf(f, a.y, v[4 * i + 1]);
                  v[4 * i + 2] = fmaf(f, a.z, v[4 * i + 2]);
                  v[4 * i + 3] = fmaf(f, a.w, v[4 * i + 3]);
                }
              }
              if (all == 0.f) {
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = 0.f;
              }
              store(c, v);
            }
            store_lse(top, all);
          }
        }
        if (!whole) kv_bar_sync(1 + q, 128);  // before the flag is used again
      }
      __syncwarp();
      if (n > 0 && lane == 0) mbar_arrive(kUfree + 8 * ur.at);
      ur = after;
      n = next.n;
      if (n <= 0) break;
      first = next.tile;
      from = next.from[q], end = next.to[q];
      lo = next.lo[q], hi = next.hi[q];
      const int next_row = next.row0 + kRows * q + r;
      place = next_row < next.rows ? next.place0 + next_row / p.group : -1;
      cq = next_cq;
      m = place >= 0 ? kNone : -kNone;  // rows that see nothing have weights of zero whatever the scores are
      l = 0.f;
      started = false;
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
