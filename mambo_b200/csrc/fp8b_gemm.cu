// FP8 block-scaled product on tcgen05: out[t, n] = sum over K blocks b of
//   sw[n / 128, b] * sum_{k in b} (xq[t, k] * 2^e(t, k / 32)) * wq[n, k].
//
// The weight tile is the MMA's A operand (128 rows in the TMEM lanes), the
// tokens its N dimension, so one kernel serves one token and a full tile, and
// a ragged segment wastes at most 15 columns. The tensor core applies the
// activations' power-of-two scales itself (block-scaled MMA, one scale per 32
// K); a K block's partial product then has one factor left, the f32 scale of
// the 128 x 128 weight block: the epilogue warps add D * sw to their FP32
// registers, one packed FMA per two values, while the next blocks' MMAs run
// into other D buffers.
//
// Two forms. Tiles of 128 rows x 16, 32 or 64 tokens on single CTAs stream the
// weights: 28672 x 8192 at 8 tokens 40.4-41.4 us, 0.87-0.89 of the measured
// HBM bandwidth (38 repeated on one input). Tiles of 256 rows x 192 tokens on
// CTA pairs carry prompts: 8192 x 28672 at 4096 tokens takes 910-945 us with
// its quantizer in short bursts (2.0-2.1 PFLOP/s) and 1046-1103 in long runs
// (1.7-1.8), where the power limit holds the SMs near 1.5 GHz.
// 14336 x 4096 at 2048 tokens: 120 us, the tensor pipe active
// 60 % of the time. What paces them is the way of a D buffer through the
// epilogue and back, and power.
//
// Work: the (row tile, token tile) tiles of all experts, numbered expert by
// expert, one per CTA and wave. Where the last wave would leave many CTAs idle
// for long, its tiles are cut at K blocks into equal ranges instead (stream-K),
// which come first; a tile that several CTAs share is summed in K order by
// whichever arrives last: nothing waits, and the sums do not depend on who.
//
// Warps: 0 weights producer, 1 and 3 MMA, 2 activations producer, then the
// epilogue warps, one per TMEM lane quadrant (and per half of the columns),
// and for one or two tokens four warps that quantize them.
//
// Compiled as a whole program of its own (no relocatable device code): the
// compiler takes setmaxnreg into account only then, and the pair kernel's
// epilogue holds 96 sums and 96 loaded values a thread. So it has its own
// device status.
#define MAMBO_OWN_DEVICE_STATUS
#include <type_traits>

#include "fp8b.cuh"
#include "iq3s_tm.cuh"
#include "kernels.cuh"
#include "mxfp8.cuh"
#include "tcgen05.cuh"

namespace mambo {

namespace {

constexpr int kMaxStagesB = 12;
// Whether the last wave's tiles are split along K: publishing and adding up the parts has to cost less than the CTAs that
// the wave leaves idle could do. All of it in K blocks of a CTA that streams its weights alone, 0.225 us (a pair 0.285);
// measured with and without the split over 1 to 420 tiles of 8 to 192 blocks, weights from HBM.
// Single wave. All CTAs at once take 1.65 times as long a block, for HBM, so a split saves K * (1 - 1.65 * tiles / CTAs).
// It costs some 20 blocks for tiles of 16 tokens, 30 for 32, and for 64, whose parts are added one by one, 35 and 4 a part.
// One token of 4096 x 4096 10.2 us unsplit, 10.4 split, x 14336 28.3 and 17.5, 8192 x 4096 10.3 and 13.2; 64 tokens of
// 4096 x 4096 12.9 and 21.6, x 14336 30.5 and 26.9.
// After a whole wave the parts are added up under the tiles that follow, so that a loss of 30 blocks on average is enough:
// 8 tokens of 28672 x 8192 (31) 41.9 and 40.9, x 4096 (15) 24.0 and 26.8. After two the CTAs have drifted apart and the last
// ones run faster alone: 340 tiles of 48 blocks lose 1 us, 380 lose 2.
// CTA pairs: 55 and 5 a part of what the idle pairs lose, and only where they are most of them. 192 tokens of 4096 x 8192
// (50, 5 parts) 25.4 unsplit, 32.2 split, x 14336 (87) 39.8 and 37.4, x 28672 (175) 72.9 and 45.5.
template <int NT>
__host__ __device__ inline bool fb_split_pays(int tiles, int kblocks, int ctas) {  // kblocks up to 2^17: all fits 32 bits
  const int rem = tiles < ctas ? tiles : tiles - ctas;
  if (rem <= 0 || rem >= ctas) return false;
  const int parts = ctas * 4 < rem * kblocks ? ctas / rem : kblocks / 4;  // of a tile: at least 4 blocks each
  const int idle = (ctas - rem) * kblocks;
  if (NT > 64) return 2 * tiles <= ctas && idle >= (55 + 5 * parts) * ctas;
  if (NT <= 32 && tiles > ctas) return idle >= 30 * ctas;
  return (20 * ctas - 33 * rem) * kblocks >= 20 * ctas * (NT <= 16 ? 20 : NT <= 32 ? 30 : 35 + 4 * parts);
}

// kPair: CTA pairs. A tile is 256 weight rows (a row tile per CTA) x NT tokens; each CTA loads half of the
// tokens and the pair's tensor cores read both halves. The tile's tokens are two MMAs of up to 96, each with D
// buffers and epilogue warps of its own: a buffer's way through the epilogue then has the time of three other MMAs
// (of one, as a single MMA of 192). 96 sums and 96 loaded values are what an epilogue thread can hold.
template <int NT, bool kPair, bool kQuant = false>
struct FbCfg {
  static constexpr int kHalves = kPair ? 2 : 1;
  static constexpr int kEpiWarps = 4 * kHalves;
  static constexpr int kCols = NT / kHalves;  // columns of an epilogue warp
  static constexpr int kD = kPair ? 2 : 4;    // D buffers (of each half), kCols columns each
  // Scale factors: the weights' (all 2^0), and 4 columns of the activations' per D buffer.
  static constexpr uint32_t kSfa = kHalves * kD * kCols;
  static constexpr uint32_t kSfb = kSfa + 16;
  static constexpr uint32_t kTmemUsed = kSfb + 4 * kD * kHalves;
  static constexpr uint32_t kTmem = kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
  static constexpr int kQuantWarps = kQuant ? 4 : 0;
  static constexpr int kThreads = (4 + kEpiWarps + kQuantWarps) * 32;
  // A stage: the weight record and this CTA's part of the activation record, both on 1024-byte boundaries.
  static constexpr uint32_t kStage = (kFbRecord + fb_part_bytes(NT) + 1023) / 1024 * 1024;
  static_assert(kCols % 16 == 0 && kSfa % 16 == 0 && kTmemUsed <= 512, "TMEM plan");
};

constexpr uint32_t kFbBarBytes = 512;

__host__ __device__ inline uint32_t fb_tables_bytes(int experts) {
  return ((uint32_t)(experts + 1) * 8 + 127) / 128 * 128;  // tile and row prefix
}

// This CTA's share of the tiles. Whole: one tile of each wave. kSplit: where it pays (above), an equal range of the K
// blocks of the last wave's tiles comes first (stream-K); the parts' sums are published and added up.
template <bool kSplit, int NT>
struct FbWalk;
template <int NT>
struct FbWalk<false, NT> {
  int kb_n, tiles, ncl, at;
  int tile, kb1;  // the current segment
  static constexpr int kb0 = 0, cl = 0;
  __device__ __forceinline__ FbWalk(int tiles_, int kblocks, int cl, int ncl_)
      : kb_n(kblocks), tiles(tiles_), ncl(ncl_), at(cl), tile(0), kb1(kblocks) {}
  __device__ __forceinline__ bool next() {
    tile = at;
    at += ncl;
    return tile < tiles;
  }
  __device__ __forceinline__ int owner(int) const { return 0; }  // of no split tile
};
template <int NT>
struct FbWalk<true, NT> {
  int kb_n, sk, tiles, ncl, cl, nsk;
  int u, u1, units;    // the host keeps tiles * K blocks below 2^31
  int at;              // next whole tile
  int tile, kb0, kb1;  // the current segment
  __device__ __forceinline__ FbWalk(int tiles_, int kblocks, int cl_, int ncl_) {
    kb_n = kblocks;
    tiles = tiles_;
    ncl = ncl_;
    cl = cl_;
    sk = fb_split_pays<NT>(tiles, kb_n, ncl) ? (tiles < ncl ? tiles : tiles - ncl) : 0;  // the last wave's tiles
    units = sk * kb_n;
    // Each part at least four K blocks.
    nsk = max(1, min(ncl, units / 4));
    u = cl < nsk ? (int)((int64_t)cl * units / nsk) : 0;
    u1 = cl < nsk ? (int)((int64_t)(cl + 1) * units / nsk) : 0;
    at = sk + cl;
    tile = kb0 = kb1 = 0;
  }
  __device__ __forceinline__ bool next() {
    if (u < u1) {
      tile = u / kb_n;
      kb0 = u - tile * kb_n;
      kb1 = min(kb_n, kb0 + (u1 - u));
      u += kb1 - kb0;
      return true;
    }
    if (at < tiles) {
      tile = at;
      at += ncl;
      kb0 = 0;
      kb1 = kb_n;
      return true;
    }
    return false;
  }
  // The CTA whose range holds unit x.
  __device__ __forceinline__ int owner(int x) const { return (int)((((int64_t)x + 1) * nsk - 1) / units); }
};

// The tile's expert, row tile and tokens, from the prefix tables in shared memory.
struct FbTile {
  int e, rt, row0, n;  // n tokens from row row0 of the expert's segment
  int64_t slot;
  int o;
};
struct FbCursor {
  const int* tiles;  // [experts + 1] first tile of each expert
  const int* offs;   // [experts + 1] clamped, non-decreasing
  int experts, nt, row_groups, e;
  __device__ __forceinline__ FbTile at(int tile) {
    while (e + 1 < experts && tile >= tiles[e + 1]) ++e;
    FbTile t;
    t.e = e;
    t.o = offs[e];
    const int count = offs[e + 1] - t.o;
    const int tt_n = fb_tiles(count, nt), tr = fb_tile_rows(count, tt_n);
    // Blocks of 8 row groups; inside one, token tile by token tile: the tiles that run together then read the fewest
    // weight and token rows (some 8 groups x 9 token tiles on 74 pairs, instead of 3 x all).
    const int local = tile - tiles[e], per = 8 * tt_n, block = local / per, in = local - block * per;
    const int rows = min(8, row_groups - 8 * block), tt = in / rows;
    t.rt = 8 * block + (in - tt * rows);  // row group: of the pair, in pairs
    t.row0 = tt * tr;
    t.n = count - t.row0 < tr ? count - t.row0 : tr;
    t.slot = fb_slot_start(t.o, e, nt) + tt;
    return t;
  }
};

// Bounded waits for a barrier phase, by one thread and by a whole warp (which agrees on the outcome). The main loop
// is a chain of such waits, most of them for a phase that is over already: that path is one try and a vote inline
// (47 + 20 clocks); with a retry loop around the try the same wait took 260. The clock is read only every 256 tries.
__device__ __forceinline__ bool fb_wait_slow(uint32_t bar, uint32_t parity, int site) {
  unsigned long long t0 = 0;
#pragma unroll 1
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (*(volatile int*)&g_device_status.code != 0 || now - t0 > g_wait_limit_ns) {
        record_timeout(site);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool fb_wait(uint32_t bar, uint32_t parity, int site) {
  return mbar_try_wait(bar, parity) || fb_wait_slow(bar, parity, site);
}
__device__ __forceinline__ bool fb_warp_wait(uint32_t bar, uint32_t parity, int site) {
  if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xFFFFFFFFu, fb_wait_slow(bar, parity, site));
}

__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

// Arrival on a barrier of the pair's other CTA. What it announces is not memory that this thread wrote: bulk copies
// that completed on a barrier, and TMEM loads that were waited for. So it needs no release at cluster scope, which
// holds the thread up until its stores are visible there: with it a K block took 1.5 times as long (prefill of
// 2048 x 14336 x 4096: 277 us, without 190 us).
__device__ __forceinline__ void arrive_remote(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}
// Packed FP32 pairs in 64-bit registers.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// N (16 or 32) consecutive TMEM columns of this lane, and the wait that makes them readable (it names the registers,
// so that no use is scheduled before it). The wait is for all of the thread's loads.
template <int N>
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32, "16 or 32 columns");
  if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,"
        "%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
  }
}
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
  } else {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
  }
}

// Ties registers to the wait before: no use of them moves ahead of it.
template <int N>
__device__ __forceinline__ void tie(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// After a wait gave up: time for the bulk copies in flight to land before the CTA leaves its shared memory.
__device__ __forceinline__ void settle_copies() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

// A K block by its issuing thread: the scale codes' atom to TMEM columns sfb (of a pair each CTA's to its own TMEM),
// four MMAs D[d] (+)= A x (B * 2^sfb)^T of 32 K each, block scaled (A's factors, at sfa, are 2^0), and the arrivals
// once they are done: on `done` (D may be read) and `empty` (the stage may be refilled), of a pair in both CTAs. a_lo,
// b_lo, s_lo: the low words of the operands' shared-memory descriptors; idesc: the instruction descriptor, whose
// bits 4-5 pick the scale code of the 32 K.
template <bool kPair>
__device__ __forceinline__ void issue_block(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t s_lo, uint32_t idesc,
                                            uint32_t sfa, uint32_t sfb, uint32_t done, uint32_t empty) {
  // High words: 8-row groups 1024 bytes apart, 128-byte swizzle; and 128 bytes apart without one, descriptor version 1.
  constexpr uint32_t kSwHi = (1024u >> 4) | (1u << 14) | (2u << 29), kSfHi = (128u >> 4) | (1u << 14);
  const uint32_t al = (a_lo & 0x3FFFu) | (1u << 16), bl = (b_lo & 0x3FFFu) | (1u << 16);
  const uint32_t sl = (s_lo & 0x3FFFu) | ((128u >> 4) << 16);
  if constexpr (kPair) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 a, b, id;\n\t.reg .b64 da, db, ds;\n\t"
        "mov.b64 ds, {%3, %9};\n\t"
        "tcgen05.cp.cta_group::2.32x128b.warpx4 [%6], ds;\n\t"
        "setp.ne.b32 p, 0, 0;\n\t"
        "mov.b64 da, {%1, %10};\n\tmov.b64 db, {%2, %10};\n\tmov.b32 id, %4;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "setp.eq.b32 p, 0, 0;\n\tadd.u32 a, %1, 2;\n\tadd.u32 b, %2, 2;\n\tadd.u32 id, %4, 16;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "add.u32 a, %1, 4;\n\tadd.u32 b, %2, 4;\n\tadd.u32 id, %4, 32;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "add.u32 a, %1, 6;\n\tadd.u32 b, %2, 6;\n\tadd.u32 id, %4, 48;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%7], %11;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%8], %11;\n\t}"
        ::"r"(d), "r"(al), "r"(bl), "r"(sl), "r"(idesc), "r"(sfa), "r"(sfb), "r"(done), "r"(empty), "r"(kSfHi),
        "r"(kSwHi), "h"((uint16_t)0x3)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 a, b, id;\n\t.reg .b64 da, db, ds;\n\t"
        "mov.b64 ds, {%3, %9};\n\t"
        "tcgen05.cp.cta_group::1.32x128b.warpx4 [%6], ds;\n\t"
        "setp.ne.b32 p, 0, 0;\n\t"
        "mov.b64 da, {%1, %10};\n\tmov.b64 db, {%2, %10};\n\tmov.b32 id, %4;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "setp.eq.b32 p, 0, 0;\n\tadd.u32 a, %1, 2;\n\tadd.u32 b, %2, 2;\n\tadd.u32 id, %4, 16;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "add.u32 a, %1, 4;\n\tadd.u32 b, %2, 4;\n\tadd.u32 id, %4, 32;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "add.u32 a, %1, 6;\n\tadd.u32 b, %2, 6;\n\tadd.u32 id, %4, 48;\n\t"
        "mov.b64 da, {a, %10};\n\tmov.b64 db, {b, %10};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, id, [%5], [%6], p;\n\t"
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t"
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%8];\n\t}"
        ::"r"(d), "r"(al), "r"(bl), "r"(sl), "r"(idesc), "r"(sfa), "r"(sfb), "r"(done), "r"(empty), "r"(kSfHi),
        "r"(kSwHi)
        : "memory");
  }
}

}  // namespace

template <int NT, bool kPair, bool kHidden, bool kSplit, bool kQuant>
__global__ void __launch_bounds__(FbCfg<NT, kPair, kQuant>::kThreads, 1) fb_gemm_kernel(const __grid_constant__ FbGemmParams p) {
  using C = FbCfg<NT, kPair, kQuant>;
  static_assert(!kQuant || (!kPair && NT == 16), "quantizing warps: tiles of 16 tokens");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* tiles0 = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int S = p.stages;
  int* tile_start = reinterpret_cast<int*>(tiles0 + (size_t)S * C::kStage);
  int* offs = tile_start + p.experts + 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(tile_start) + fb_tables_bytes(p.experts));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStagesB + 2 * 4 + 1 + 4);
  float* xchg = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + kFbBarBytes);  // kHidden: 4 KB per two warps
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t kFull = bar0, kEmpty = bar0 + 8 * kMaxStagesB;
  const uint32_t kMdone = bar0 + 16 * kMaxStagesB, kEfree = kMdone + 8 * 4, kEdone = kEfree + 8 * 4;
  const uint32_t kPairBar = kEdone + 8;  // kHidden: two epilogue warps meet, 4 of them
  static_assert(C::kD * C::kHalves <= 4, "barriers");
  // Values that the whole warp shares are broadcast from lane 0, so that the compiler keeps them, and what the MMAs
  // take as operands, in uniform registers.
  const int warp = uniform((int)(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const int KB = p.act.kblocks;
  const int rank = kPair ? (int)cluster_ctarank() : 0;
  const int row_groups = kPair ? (p.row_tiles + 1) / 2 : p.row_tiles;
  // Rank 0's copy of a barrier: it issues the pair's MMAs, rank 1 arrives there.
  auto lead = [&](uint32_t bar) { return mapa_shared(bar, 0); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      // Both producers, and in rank 0 of a pair the other CTA's landed operands.
      mbar_init(kFull + 8 * s, kPair && rank == 0 ? 3 : 2);
      mbar_init(kEmpty + 8 * s, kPair ? 2 : 1);  // a pair's two issuers
    }
    for (int d = 0; d < C::kD * C::kHalves; ++d) {  // buffer d of half h: barrier h * kD + d
      mbar_init(kMdone + 8 * d, 1);
      mbar_init(kEfree + 8 * d, kPair ? 8 : 4);
    }
    mbar_init(kEdone, C::kEpiWarps);
    for (int i = 0; i < 4; ++i) mbar_init(kPairBar + 8 * i, 2);
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tc::alloc_pair(smem_u32(tmem_slot), C::kTmem);
      tc::relinquish_pair();
    } else {
      tc::alloc(smem_u32(tmem_slot), C::kTmem);
      tc::relinquish();
    }
  }
  if (warp == 0) {
    // Row and tile prefix of the experts. Offsets are clamped to [0, rows] and
    // made non-decreasing, so that no offsets can lead out of the buffers.
    if (p.offsets) {
      pdl_wait();
      int prev = __ldg(p.offsets);
      prev = prev < 0 ? 0 : prev > p.rows ? (int)p.rows : prev;
      int tiles = 0;
      if (lane == 0) {
        tile_start[0] = 0;
        offs[0] = prev;
      }
      for (int b = 0; b < p.experts; b += 32) {
        const int e = b + lane;
        int o = e < p.experts ? __ldg(p.offsets + e + 1) : 0;
        o = o > p.rows ? (int)p.rows : o;
        o = max(o, prev);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(0xFFFFFFFFu, o, d);
          if (lane >= d) o = max(o, up);
        }
        int before = __shfl_up_sync(0xFFFFFFFFu, o, 1);
        if (lane == 0) before = prev;
        int t = fb_tiles(o - before, NT) * row_groups;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int up = __shfl_up_sync(0xFFFFFFFFu, t, d);
          if (lane >= d) t += up;
        }
        if (e < p.experts) {
          tile_start[e + 1] = tiles + t;
          offs[e + 1] = o;
        }
        tiles += __shfl_sync(0xFFFFFFFFu, t, 31);
        prev = __shfl_sync(0xFFFFFFFFu, o, 31);
      }
    } else if (lane == 0) {
      tile_start[0] = 0;
      tile_start[1] = fb_tiles((int)p.rows, NT) * row_groups;
      offs[0] = 0;
      offs[1] = (int)p.rows;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);
  // The weights' MMA scale factors: 2^0 in every lane and byte.
  if (warp >= 4 && warp < 8) {
    tc::st_x4(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + C::kSfa, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    tc::wait_st();
  }
  tc::fence_before_sync();
  __syncthreads();
  if constexpr (kPair) cluster_sync_all();  // both CTAs' barriers and TMEM are ready before any remote use
  tc::fence_after_sync();

  FbWalk<kSplit, NT> walk(uniform(tile_start[p.experts]), KB, (int)blockIdx.x / (kPair ? 2 : 1), (int)gridDim.x / (kPair ? 2 : 1));
  FbCursor cur{tile_start, offs, p.experts, NT, row_groups, 0};

  // Register split of the pair kernel, launched with 168 a thread (384 threads): 128 x 56 + 256 x 224 = 384 x 168.
  // Each instruction opens its own branch, so that the compiler knows every role's count.
  if (warp < 4) {
    if constexpr (kPair) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // -------------------------------------------------------------- weights producer
      if (lane == 0) {
        // Weights may be read ahead of the previous kernel's end where that is the quantizer, which waited for all
        // before it; a kernel that is the first of its call may follow the one that packed them.
        if (kQuant) pdl_wait();
        const uint64_t policy = l2_policy_evict_first();
        int it = 0, s = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok && walk.next()) {
          const FbTile t = cur.at(walk.tile);
          const int rt = kPair ? 2 * t.rt + rank : t.rt;
          const bool have = !kPair || rt < p.row_tiles;  // the second row tile of the last pair may not exist
          const uint8_t* rec = p.packed + (((int64_t)t.e * p.row_tiles + rt) * KB) * kFbRecord;
          for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
            if (it >= S && !fb_wait(kEmpty + 8 * s, ph ^ 1, kSiteFbEmpty)) {
              ok = false;
              break;
            }
            const uint32_t dst = smem_u32(tiles0 + (size_t)s * C::kStage);
            if (have) {
              mbar_arrive_expect_tx(kFull + 8 * s, kFbRecord);
            } else {
              mbar_arrive(kFull + 8 * s);  // whatever the stage holds: these rows are not stored
            }
            if (!have) {
            } else if (p.evict_weights) {
              bulk_load_hint(dst, rec + (int64_t)kb * kFbRecord, kFbRecord, kFull + 8 * s, policy);
            } else {
              bulk_load(dst, rec + (int64_t)kb * kFbRecord, kFbRecord, kFull + 8 * s);
            }
            if (++s == S) {
              s = 0;
              ph ^= 1;
            }
          }
        }
        if (!ok) settle_copies();
      }
      __syncwarp();
    } else if (warp == 2) {
      // -------------------------------------------------------------- activations producer
      if (!kQuant && lane == 0) {
        pdl_wait();
        int it = 0, s = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok && walk.next()) {
          const FbTile t = cur.at(walk.tile);
          const uint32_t bytes = (uint32_t)fb_part_rows(t.n, kPair) * 128u + fb_atoms_per_tile(NT) * kFbAtom;
          const uint8_t* x = p.act.x8 + t.slot * KB * fb_record_bytes(NT) + (kPair ? rank * fb_part_bytes(NT) : 0u);
          for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
            if (it >= S && !fb_wait(kEmpty + 8 * s, ph ^ 1, kSiteFbEmpty)) {
              ok = false;
              break;
            }
            const uint32_t full = kFull + 8 * s;
            mbar_arrive_expect_tx(full, bytes);
            bulk_load(smem_u32(tiles0 + (size_t)s * C::kStage) + kFbRecord, x + (int64_t)kb * fb_record_bytes(NT), bytes,
                      full);
            if (++s == S) {
              s = 0;
              ph ^= 1;
            }
          }
        }
        if (!ok) settle_copies();
      }
      __syncwarp();
    } else {
      // -------------------------------------------------------------- MMA
      // Two issuing warps, 1 and 3, each with D buffers of its own: of a pair's tile each issues one half, alone they
      // take the K blocks in turn. A K block costs its issuer some 400 clocks (two waits, the scale copy, four MMAs,
      // two commits), which alone would pace the kernel.
      const int who = warp >> 1;
      if (kPair && rank == 1 && who == 0) {
        // Rank 1 of a pair: its operands have landed, told to rank 0, which issues the MMAs of both.
        if (lane == 0) {
          int s = 0;
          uint32_t ph = 0;
          bool ok = true;
          while (ok && walk.next()) {
            for (int kb = walk.kb0; kb < walk.kb1; ++kb) {
              ok = fb_wait(kFull + 8 * s, ph, kSiteFbFull);
              if (!ok) break;
              arrive_remote(lead(kFull + 8 * s));
              if (++s == S) {
                s = 0;
                ph ^= 1;
              }
            }
          }
        }
        __syncwarp();
      }
      // One thread issues: the chain from a free D buffer to its MMAs has no votes and no elections, and what the
      // instructions take is ready before the waits.
      if ((!kPair || rank == 0) && tm::elect_one()) {
        // The loop is a chain of dependent instructions of one thread: everything that it can carry along is carried.
        constexpr int kMine = kPair ? C::kD : C::kD / 2;  // D buffers of this issuer: a half's, or every other one
        constexpr uint32_t kStep = kPair ? 1 : 2;
        const uint32_t buf0 = kPair ? who * C::kD : who;
        const uint32_t stage0 = smem_u32(tiles0) >> 4;
        int s = 0, buf = 0;
        uint32_t ph = 0, eph = 1, stage = stage0;  // eph: a fresh barrier's previous phase counts as over
        bool ok = true, turn = kPair || who == 0;
        while (ok && walk.next()) {
          const int n_tile = cur.at(walk.tile).n;
          const int nn = (n_tile + 15) / 16 * 16, n0 = kPair ? fb_split(n_tile) : nn;
          const int n = who == 0 || !kPair ? n0 : nn - n0;
          const uint32_t idesc = tc::idesc_mx_e4m3(kPair ? 256 : 128, n, 0, 0);
          // This MMA's tokens, and the scale codes after all rows that the CTA holds.
          const uint32_t b_at = (kFbRecord + (kPair && who ? n0 / 2 * 128u : 0u)) >> 4;
          const uint32_t sf_at = (kFbRecord + (uint32_t)fb_part_rows(n_tile, kPair) * 128u + (kPair ? who * kFbAtom : 0u)) >> 4;
          for (int left = walk.kb1 - walk.kb0; left > 0; --left) {
            const uint32_t full = kFull + 8 * s;
            if (kPair ? n > 0 : turn) {
              const uint32_t b = buf0 + kStep * buf, bar = 8u * b;
              uint32_t d = tmem + b * C::kCols, sfb = tmem + C::kSfb + 4u * b;
              uint32_t a_lo = stage, b_lo = stage + b_at, s_lo = stage + sf_at;
              asm volatile("" : "+r"(a_lo), "+r"(b_lo), "+r"(s_lo), "+r"(d), "+r"(sfb));  // before the waits
              ok = fb_wait(full, ph, kSiteFbFull) && fb_wait(kEfree + bar, eph, kSiteFbEmpty);
              if (!ok) break;
              tc::fence_after_sync();
              issue_block<kPair>(d, a_lo, b_lo, s_lo, idesc, tmem + C::kSfa, sfb, kMdone + bar, kEmpty + 8 * s);
              if (++buf == kMine) {
                buf = 0;
                eph ^= 1;
              }
            } else if (kPair) {
              // A tile of at most 16 tokens has no second MMA: the stage is released as if it had been read.
              ok = fb_wait(full, ph, kSiteFbFull);
              if (!ok) break;
              arrive_remote(mapa_shared(kEmpty + 8 * s, 0));
              arrive_remote(mapa_shared(kEmpty + 8 * s, 1));
            }
            if (!kPair) turn = !turn;
            stage += C::kStage >> 4;
            if (++s == S) {
              s = 0;
              ph ^= 1;
              stage = stage0;
            }
          }
        }
      }
      __syncwarp();
      if (who == 0) {
        // Free the TMEM once every epilogue warp has read its last results.
        fb_wait(kEdone, 0, kSiteFbFull);
        __syncwarp();
        tc::fence_after_sync();
        if constexpr (kPair) {
          tc::dealloc_pair(tmem, C::kTmem);
        } else {
          tc::dealloc(tmem, C::kTmem);
        }
      }
    }
  } else if (kQuant && warp >= 8) {
    // -------------------------------------------------------------- quantizing warps
    // For tiles of one or two tokens: four warps take the K blocks in turn and write each block's E4M3 bytes and scale
    // codes straight into its stage, a half warp a token, 8 values a lane. Every tile's CTA quantizes the tokens anew:
    // for one token that is less than a launch of the quantizer (repeated, weights in L2: 4096 x 4096 11.2 -> 10.6 us, 64 experts of 2048 x
    // 1408, six a token: 32.0 -> 27.9), for eight it held the weights up (28672 x 8192: 39 -> 54 us). A call of one or two
    // tokens has tiles of more rows only where a route names an expert repeatedly: those follow two at a time (the loop
    // for them costs the others 0.5 %: one token of 64 experts, weights from HBM, 28.8 -> 28.95 us).
    const FbSource& src = p.src;
    const int who = warp - 8, col = (lane & 15) * 8, r = lane >> 4;
    pdl_wait();
    int it = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const FbTile t = cur.at(walk.tile);
      const uint32_t sf_at = kFbRecord + (uint32_t)fb_part_rows(t.n, false) * 128u;
      // Where row i of the tile starts in x (the last row for one past it).
      auto row_at = [&](int i) {
        const int mine = t.o + t.row0 + min(i, t.n - 1);
        return min(src.rows ? max(__ldg(src.rows + mine), 0) / src.top : mine, src.last) * src.ldx;
      };
      auto load = [&](int64_t row, int kb, uint4& lo, uint4& hi) {
        const int64_t k0 = (int64_t)kb * 128 + col;
        lo = hi = make_uint4(0, 0, 0, 0);
        if (src.bf16) {
          const uint16_t* x = reinterpret_cast<const uint16_t*>(src.x) + row + k0;
          if (src.vec && k0 + 8 <= src.k) {
            lo = __ldg(reinterpret_cast<const uint4*>(x));
          } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (k0 + i < src.k) w[i >> 1] |= (uint32_t)__ldg(x + i) << (16 * (i & 1));
            lo = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          const uint32_t* x = reinterpret_cast<const uint32_t*>(src.x) + row + k0;
          if (src.vec && k0 + 8 <= src.k) {
            lo = __ldg(reinterpret_cast<const uint4*>(x));
            hi = __ldg(reinterpret_cast<const uint4*>(x) + 1);
          } else {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = k0 + i < src.k ? __ldg(x + i) : 0u;
            lo = make_uint4(w[0], w[1], w[2], w[3]);
            hi = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      };
      // A half warp's values to row i of the stage (a row past the tile's holds the last one again; nothing stores it).
      auto store = [&](uint8_t* st, int i, const uint4& lo, const uint4& hi) {
        uint32_t word;
        uint2 q;
        if (src.bf16) {
          q = quantize8(lo, src.group, lane, word);
        } else {
          const float v[8] = {__uint_as_float(lo.x), __uint_as_float(lo.y), __uint_as_float(lo.z), __uint_as_float(lo.w),
                              __uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w)};
          q = quantize8(v, src.group, lane, word);
        }
        *reinterpret_cast<uint2*>(st + kFbRecord + i * 128 + ((((lane & 15) >> 1) ^ (i & 7)) << 4) + (lane & 1) * 8) = q;
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(st + sf_at + i * 16) = word;
      };
      const int64_t row = row_at(r);
      int kb = walk.kb0 + ((who - it) & 3);  // this warp's first block of the segment
      uint4 lo, hi, lo2, hi2;
      if (kb < walk.kb1) load(row, kb, lo, hi);
      for (; kb < walk.kb1; kb += 4) {
        if (kb + 4 < walk.kb1) load(row, kb + 4, lo2, hi2);
        const int at = it + (kb - walk.kb0), s = at % S;
        if (at >= S && !(ok = fb_warp_wait(kEmpty + 8 * s, (uint32_t)(at / S - 1) & 1u, kSiteFbEmpty))) break;
        uint8_t* st = tiles0 + (size_t)s * C::kStage;
        store(st, r, lo, hi);
#pragma unroll 1
        for (int i = 2; i < t.n; i += 2) {
          uint4 more_lo, more_hi;
          load(row_at(i + r), kb, more_lo, more_hi);
          store(st, i + r, more_lo, more_hi);
        }
        fence_proxy_async_shared();  // the tensor core reads the stage through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive(kFull + 8 * s);
        lo = lo2;
        hi = hi2;
      }
      it += walk.kb1 - walk.kb0;
    }
    __syncwarp();
  } else {
    if constexpr (kPair) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, h = (warp - 4) >> 2;
    const int rl = 32 * q + lane;
    const uint32_t tq0 = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(h * C::kD * C::kCols);
    uint64_t acc2[C::kCols / 2];  // pairs of columns
#pragma unroll
    for (int i = 0; i < C::kCols / 2; ++i) acc2[i] = 0;
    auto acc = [&](int c) {
      return __uint_as_float((c & 1) ? (uint32_t)(acc2[c >> 1] >> 32) : (uint32_t)acc2[c >> 1]);
    };
    pdl_wait();  // the output and the workspace may belong to the previous kernel
    pdl_launch_dependents();
    const uint32_t efree0 = kPair ? lead(kEfree + 8 * h * C::kD) : 0u;  // this half's, in rank 0
    int db = 0;
    uint32_t dph = 0;
    bool ok = true;
    // kHidden: this warp and the one with the other half of its features meet (a bounded wait, as every one).
    const uint32_t meet = kPairBar + 8u * (uint32_t)(h * 2 + (q >> 1));
    uint32_t mph = 0;
    auto pair_sync = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet);
      const bool met = fb_warp_wait(meet, mph, kSiteFbFull);
      mph ^= 1;
      return met;
    };
    while (ok && walk.next()) {
      const float* sw;
      int cols;  // this warp's valid columns (may be <= 0)
      {
        const FbTile t = cur.at(walk.tile);
        const int rt = kPair ? 2 * t.rt + rank : t.rt;
        const int n = uniform(t.n), n0 = kPair ? fb_split(n) : n;
        cols = h ? n - n0 : min(n, n0);
        // A row tile past the end has no scales; its sums are not stored.
        sw = p.scales + (((int64_t)t.e * p.row_tiles + (rt < p.row_tiles ? rt : 0)) * 2 + (q & 1)) * KB;
      }
#pragma unroll
      for (int i = 0; i < C::kCols / 2; ++i) acc2[i] = 0;
      if (cols <= 0) continue;  // this half's MMAs are not issued either
      // A K block: all of the warp's columns to registers at once, the D buffer released, then the additions. The
      // buffer's way back to the MMAs is what paces the kernel, and additions between its loads lengthen it: with
      // chunks of 32 columns loaded ahead of their additions a K block of 224 tokens took 912 clocks, 505 without
      // the additions. Columns past the tile's in a chunk are added like the others (whatever they hold), never stored.
      constexpr int kCh = C::kCols < 32 ? C::kCols : 32;
      // One loop per number of column chunks, so that a ragged tile loads and adds no more than it has: branches inside
      // one loop made every tile slower (14336 x 4096 at 2048 tokens 150 -> 183 us).
      auto k_loop = [&](auto chunks) {
        constexpr int kChunks = decltype(chunks)::value;
        float sv = 0.f;
#pragma unroll 1
        for (int kb = walk.kb0; kb < walk.kb1; ++kb) {
          if (kb == walk.kb0 || (kb & 31) == 0) sv = (kb & ~31) + lane < KB ? __ldg(sw + (kb & ~31) + lane) : 0.f;
          const float w = __shfl_sync(0xFFFFFFFFu, sv, kb & 31);
          const uint64_t w2 = pack2(w, w);
          ok = fb_warp_wait(kMdone + 8 * (h * C::kD + db), dph, kSiteFbFull);
          if (!ok) return;
          tc::fence_after_sync();
          uint32_t v[kChunks][kCh];
#pragma unroll
          for (int c = 0; c < kChunks; ++c) ld_cols(tq0 + (uint32_t)db * C::kCols + c * kCh, v[c]);
          wait_ld(v[0]);
#pragma unroll
          for (int c = 1; c < kChunks; ++c) tie(v[c]);
          tc::fence_before_sync();
          // The loads' wait was the whole warp's, so one lane may speak for it; in both CTAs of a pair to rank 0.
          if (kPair) {
            if (lane == 0) arrive_remote(efree0 + 8 * db);
          } else {
            if (lane == 0) mbar_arrive(kEfree + 8 * db);
          }
          if (++db == C::kD) {
            db = 0;
            dph ^= 1;
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int i = 0; i < kCh / 2; ++i)
              acc2[c * kCh / 2 + i] =
                  fma2(pack2(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), w2, acc2[c * kCh / 2 + i]);
        }
      };
      if constexpr (C::kCols == 3 * kCh) {
        if (cols > 2 * kCh) {
          k_loop(std::integral_constant<int, 3>{});
        } else {
          k_loop(std::integral_constant<int, 2>{});
        }
      } else {
        k_loop(std::integral_constant<int, C::kCols / kCh>{});
      }
      if (!ok) break;
      if (kSplit && (walk.kb0 != 0 || walk.kb1 != KB)) {
        // A tile shared between CTAs: publish this warp's part, and sum all
        // parts in K order if it is the last to arrive.
        const int u_tile = walk.tile * KB;
        const int first = walk.owner(u_tile), last = walk.owner(u_tile + KB - 1);
        constexpr int kQuads = NT / 4;
        auto part = [&](int cta) {
          // Slot 1 holds the part that starts its tile (the CTA's last tile), slot 0 the others.
          const int64_t at = kPair ? cta * 2 + rank : cta;
          return reinterpret_cast<float4*>(p.partials) + ((at * 2 + (cta == first ? 1 : 0)) * kQuads + h * C::kCols / 4) * 128 + rl;
        };
        float4* mine = part(walk.cl);
#pragma unroll
        for (int c = 0; c < C::kCols; c += 4)
          if (C::kCols <= 32 || c < cols)
            __stcg(mine + (c / 4) * 128, make_float4(acc(c), acc(c + 1), acc(c + 2), acc(c + 3)));
        __syncwarp();  // orders the warp's stores before the counting lane's release
        int* counter = p.counters + (kPair ? first * 2 + rank : first) * 8 + (warp - 4);
        int done = 0;
        if constexpr (kHidden) {
          // The two warps finish a tile together, so one of them counts for both, once both have published.
          if (!(ok = pair_sync())) break;
          int* flag = reinterpret_cast<int*>(xchg + (h * 2 + (q >> 1)) * 1024);
          if (lane == 0 && (q & 1) == 0) {
            *flag = atomic_add_acq_rel_gpu(counter, 1) == last - first;
            if (*flag) *counter = 0;  // all parts are in: zero again for the next launch
          }
          if (!(ok = pair_sync())) break;
          done = *flag;
          if (!(ok = pair_sync())) break;  // before the flag's place is used again
          if (!done) continue;
        } else {
          if (lane == 0) done = atomic_add_acq_rel_gpu(counter, 1) == last - first;
          done = __shfl_sync(0xFFFFFFFFu, done, 0);
          if (!done) continue;
          if (lane == 0) *counter = 0;  // all parts are in: zero again for the next launch
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < C::kCols / 2; ++c) acc2[c] = 0;
        // The parts in K order. Of a small tile several parts' loads are in flight at once; a large one's columns are
        // enough, and holding more would cost its K loop registers.
        constexpr int kBatch = C::kCols <= 16 ? 8 : C::kCols <= 32 ? 4 : 1;
        for (int cta = first; cta <= last; cta += kBatch) {
          if constexpr (kBatch == 1) {
            const float4* src = part(cta);
#pragma unroll
            for (int c = 0; c < C::kCols; c += 4) {
              if (c < cols) {
                const float4 v = __ldcg(src + (c / 4) * 128);
                acc2[c / 2] = pack2(acc(c) + v.x, acc(c + 1) + v.y);
                acc2[c / 2 + 1] = pack2(acc(c + 2) + v.z, acc(c + 3) + v.w);
              }
            }
          } else {
            float4 v[kBatch][C::kCols / 4];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
              const float4* src = part(min(cta + j, last));
#pragma unroll
              for (int c = 0; c < C::kCols; c += 4) v[j][c / 4] = __ldcg(src + (c / 4) * 128);
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
              if (cta + j <= last) {
#pragma unroll
                for (int c = 0; c < C::kCols; c += 4) {
                  acc2[c / 2] = pack2(acc(c) + v[j][c / 4].x, acc(c + 1) + v[j][c / 4].y);
                  acc2[c / 2 + 1] = pack2(acc(c + 2) + v[j][c / 4].z, acc(c + 3) + v[j][c / 4].w);
                }
              }
            }
          }
        }
      }
      // Looked up again: held over the K loop, these would cost it registers.
      const FbTile t = cur.at(walk.tile);
      if constexpr (kHidden) {
        // The even warps hold gate rows, the odd ones the up rows of the same 32 features (a MXFP8 group of the next
        // product's K). Of 16 columns at a time the even warp forms h for the first eight, the odd one for the
        // others: each sends the other eight over shared memory. Then a lane is a feature and a group's maximum is
        // one warp reduction. Bound by instructions (some 25 a column), with the MMAs waiting: hence the packed
        // code arithmetic below; a first version of 60 a column took 1073 us in all where this one takes 805
        // (gate/up product of 4096 tokens, 64 experts of 2048 x 4096, eight a token).
        const FbActivations& hid = p.hidden;
        const bool odd = q & 1;
        const int n0 = fb_split(t.n), per = (h ? (t.n + 15) / 16 * 16 - n0 : n0) / 2;
        uint8_t* rec = hid.x8 + (t.slot * hid.kblocks + (kPair ? t.rt : t.rt >> 1)) * fb_record_bytes(NT);
        const int rt = kPair ? rank : t.rt & 1;  // half of the 128-feature block
        uint8_t* row0 = rec + 64 * rt + 16 * (q & 2) + lane;  // the lane's byte of an unswizzled row
        // Scale codes: lanes 0-7 store those of eight tokens, of a pair lanes 8-15 the other CTA's copy.
        uint8_t* sf = rec + fb_part_rows(t.n, kPair) * 128 + h * kFbAtom + 2 * rt + (q >> 1) + (lane & 7) * 16 +
                      (lane >= 8 ? fb_part_bytes(NT) : 0u);
        float* xch = xchg + (h * 2 + (q >> 1)) * 1024 + lane;
#pragma unroll 1
        for (int b = 0; b < cols; b += 16) {
          float own[8], other[8];
          float* buf = xch + (b & 16) * 32;  // two buffers: one meeting per turn
#pragma unroll
          for (int k = 0; k < C::kCols; k += 16) {
            if (k == b) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                own[i] = odd ? acc(k + 8 + i) : acc(k + i);
                buf[(odd ? 256 : 0) + i * 32] = odd ? acc(k + i) : acc(k + 8 + i);
              }
            }
          }
          if (!(ok = pair_sync())) break;
#pragma unroll
          for (int i = 0; i < 8; ++i) other[i] = buf[(odd ? 0 : 256) + i * 32];
          const int c8 = b + (odd ? 8 : 0);  // this warp's eight tokens, among this half's
          uint32_t most = 0;                 // lane i (mod 8): token i's largest magnitude
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float g = odd ? other[i] : own[i], u = odd ? own[i] : other[i];
            // The fast exponential and quotient: off by some 4 + 1.2 |g| units of 2^-23 (2^-18 at |g| = 24, 2^-16 at 88,
            // past which the quotient is 0, as its value to 1e-36), where E4M3 rounds by up to 2^-4.
            own[i] = __fdividef(g, 1.0f + __expf(-g)) * u;
            const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(own[i]) & 0x7FFFFFFFu);
            if ((lane & 7) == i) most = m;
          }
          const uint32_t code = mxfp8_scale_code(__uint_as_float(most));
          const int part = kPair && c8 >= per;
          // Eight tokens are eight rows of one swizzle group of one part: row i lies 128 i on, its chunks xor i.
          uint8_t* r8 = row0 + part * fb_part_bytes(NT) + (kPair ? c8 - part * per + h * (n0 / 2) : c8) * 128;
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const uint32_t k0 = __shfl_sync(0xFFFFFFFFu, code, i), k1 = __shfl_sync(0xFFFFFFFFu, code, i + 1);
            // 2^-e, e = code - 127; the bytes of a NaN group (code 255) do not matter.
            const uint32_t two = cvt_e4m3x2_rn(own[i] * __uint_as_float((254u - k0) << 23),
                                               own[i + 1] * __uint_as_float((254u - k1) << 23));
            if (c8 + i < cols) *reinterpret_cast<uint8_t*>(((uintptr_t)r8 ^ (i << 4)) + 128 * i) = (uint8_t)two;
            if (c8 + i + 1 < cols)
              *reinterpret_cast<uint8_t*>(((uintptr_t)r8 ^ ((i + 1) << 4)) + 128 * (i + 1)) = (uint8_t)(two >> 8);
          }
          if (lane < (kPair ? 16 : 8) && c8 + (lane & 7) < cols) sf[(c8 & 31) * 16 + (c8 >> 5) * 4] = (uint8_t)code;
        }
        // The next tile's first turn may use either buffer: the other warp has read both.
        if (ok) ok = pair_sync();
        continue;
      }
      const int row = (kPair ? 2 * t.rt + rank : t.rt) * 128 + rl;
      if (row < p.n_rows) {
        const int64_t at = ((int64_t)t.o + t.row0 + (h ? fb_split(t.n) : 0)) * p.ldo + row;
        if (p.out_bf16) {
          __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
          for (int c = 0; c < C::kCols; ++c)
            if (c < cols) o[(int64_t)c * p.ldo] = __float2bfloat16_rn(acc(c));
        } else {
          float* o = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
          for (int c = 0; c < C::kCols; ++c)
            if (c < cols) o[(int64_t)c * p.ldo] = acc(c);
        }
      }
    }
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(kEdone);
    __syncwarp();
  }
  // Neither CTA of a pair leaves while the other may still use its shared memory or TMEM.
  if constexpr (kPair) cluster_sync_all();
}

// --------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------
namespace {

template <int NT, bool kPair>
uint32_t smem_of(int experts, int stages, bool hidden) {
  using C = FbCfg<NT, kPair>;
  return 1024 + (uint32_t)stages * C::kStage + fb_tables_bytes(experts) + kFbBarBytes +
         (hidden ? (uint32_t)C::kEpiWarps / 2 * 4096 : 0u);
}
template <int NT, bool kPair, bool kHidden, bool kSplit, bool kQuant = false>
cudaError_t launch_kernel(const FbGemmParams& p, int grid, cudaStream_t stream) {
  const uint32_t smem = smem_of<NT, kPair>(p.experts, p.stages, kHidden);
  const void* k = (const void*)fb_gemm_kernel<NT, kPair, kHidden, kSplit, kQuant>;
  cudaError_t e = ensure_smem_attribute(k, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl_cluster(k, dim3(grid), dim3(FbCfg<NT, kPair, kQuant>::kThreads), smem, stream, kPair ? 2 : 1, p);
}
// Single CTAs decide on the device whether to split (an expert-grouped call's tiles are counted there). A CTA pair's
// partial sums are large (98 KB a CTA), and the code for them costs its K loop registers, used or not (14336 x 4096 at 2048
// tokens: 131 us without it, 148 with), so the host decides, and a grouped call does not split. That one would gain little
// and lose more: 4 experts of 1024 x 14336 at 800 rows 49.3 us, with the split kernel 46.8; one of 8 experts of 14336 x 4096
// at 512 rows 45.3 and 62.4; 64 of 4096 x 4096 at 16384 rows 474 and 490.
template <int NT, bool kQuant = false>
cudaError_t launch_one(const FbGemmParams& p, int grid, cudaStream_t stream) {
  return p.hidden.x8 ? launch_kernel<NT, false, true, true, kQuant>(p, grid, stream)
                     : launch_kernel<NT, false, false, true, kQuant>(p, grid, stream);
}
cudaError_t launch_pair(const FbGemmParams& p, int grid, cudaStream_t stream) {
  constexpr int NT = kFbPairTokens;
  if (p.hidden.x8) return launch_kernel<NT, true, true, false>(p, grid, stream);
  const int tiles = (p.row_tiles + 1) / 2 * fb_tiles((int)p.rows, NT), pairs = grid / 2;  // the host's size check: they fit
  if (!p.offsets && fb_split_pays<NT>(tiles, p.act.kblocks, pairs))
    return launch_kernel<NT, true, false, true>(p, grid, stream);
  return launch_kernel<NT, true, false, false>(p, grid, stream);
}

}  // namespace

// The smallest tile that holds the rows, of single CTAs up to 64, then a pair's. Microseconds for N of 1024, 4096 and 14336
// (K 4096, weights from HBM): 33 to 64 rows in single tiles 12.5, 13.0, 14.7, in pair tiles 15.0, 15.2, 16.2; 77 rows in two
// single tiles 12.6, 12.9, 23.9, in a pair's 15.2, 15.3, 16.7; 192 rows in three 12.7, 13.5, 32.3, in a pair's 15.4, 15.8,
// 19.2. So from 65 rows on single tiles would be faster by a sixth as long as all fit one wave, and slower by up to 70 %
// where they do not; the rule looks at rows only and takes the form that cannot lose as much.
int fb_tile_for(int64_t expected_rows) {
  return expected_rows <= 16 ? 16 : expected_rows <= 32 ? 32 : expected_rows <= 64 ? 64 : kFbPairTokens;
}

uint32_t fb_gemm_smem(int nt, int experts, int stages, bool hidden) {
  switch (nt) {
    case 16: return smem_of<16, false>(experts, stages, hidden);
    case 32: return smem_of<32, false>(experts, stages, hidden);
    case 64: return smem_of<64, false>(experts, stages, hidden);
    default: return smem_of<kFbPairTokens, true>(experts, stages, hidden);
  }
}

int fb_gemm_stages(int nt, int experts, int smem_optin, bool hidden) {
  int s = kMaxStagesB;
  while (s > 2 && (int)fb_gemm_smem(nt, experts, s, hidden) > smem_optin) --s;
  return s;
}

cudaError_t fb_status_symbols(void** status, void** limit) {
  cudaError_t e = cudaGetSymbolAddress(status, g_device_status);
  return e == cudaSuccess ? cudaGetSymbolAddress(limit, g_wait_limit_ns) : e;
}

int fb_gemm_grid(int nt, int sms) { return nt == kFbPairTokens ? sms / 2 * 2 : sms; }
size_t fb_partial_bytes(int nt, int sms) { return (size_t)sms * 2 * 128 * nt * sizeof(float); }

cudaError_t launch_fb_gemm(const FbGemmParams& p, int grid, cudaStream_t stream) {
  switch (p.act.nt) {
    case 16: return p.src.x ? launch_one<16, true>(p, grid, stream) : launch_one<16>(p, grid, stream);
    case 32: return launch_one<32>(p, grid, stream);
    case 64: return launch_one<64>(p, grid, stream);
    default: return launch_pair(p, grid, stream);
  }
}

}  // namespace mambo
