// What the attention kernels share: bounded waits, 8-bit conversions, the
// tensor core's descriptors for operands that lie along M or N, and the cut of
// a call's work into equal ranges.
#pragma once

#include "kv.cuh"
#include "mxfp8.cuh"
#include "tcgen05.cuh"

namespace mambo {

// Positions of a tile of keys and values.
constexpr int kKvTile = 128;
constexpr uint32_t kKvTileBytes = 128u * 128u;  // rows of 128 bytes, zero behind the head size

// Waits for a barrier phase, bounded in time. A waiting warp sleeps in the try (up to 20 us, or until the phase is over):
// tries in a loop fill the pipe that also takes the other warps' shuffles and shared-memory accesses.
__device__ __forceinline__ bool kv_wait_slow(uint32_t bar, uint32_t parity, int site) {
  const unsigned long long t0 = globaltimer_ns();
#pragma unroll 1
  while (!mbar_try_wait_sleep(bar, parity, 20000u)) {
    if (*(volatile int*)&g_device_status.code != 0 || globaltimer_ns() - t0 > g_wait_limit_ns) {
      record_timeout(site);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool kv_wait(uint32_t bar, uint32_t parity, int site) {
  return mbar_try_wait(bar, parity) || kv_wait_slow(bar, parity, site);
}
__device__ __forceinline__ bool kv_warp_wait(uint32_t bar, uint32_t parity, int site) {
  if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xFFFFFFFFu, kv_wait_slow(bar, parity, site));
}
// After a wait gave up: time for the copies in flight to land before the CTA leaves its shared memory.
__device__ __forceinline__ void kv_settle() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

// Phases of a ring of n buffers: the buffer in use and the parity of its current phase.
struct KvRing {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++at == n) {
      at = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Packed conversions: f16 pairs to and from E4M3 pairs (the low half in the low byte).
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_of_f16x2(uint32_t h) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t c) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(c));
  return h;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The UE8M0 code of the power of two that brings a bf16 magnitude (its bits) to at most 448, 255 for NaN and infinity; as
// mxfp8_scale_code, but for zero, and without branches: those keep the compiler from overlapping the chains of several
// rows, and a row's chain (shuffles, code, conversions) is some 400 clocks.
__device__ __forceinline__ uint32_t bf16_scale_code(uint32_t bits) {
  const int biased = (int)(bits >> 7);
  const int code = max(biased - ((bits & 0x7Fu) <= 0x60u ? 8 : 7), 0);
  return biased == 255 ? 255u : (uint32_t)code;
}

// A row of queries as two E4M3 terms: q * 2^-e = hi + lo with e the power of two that brings its largest magnitude to at
// most 448. A bf16 has 8 significant bits: hi rounds to 4, what is left has 4, so the sum is exact (down to 2^-10, that
// is 2^-18 of the row's largest value). The products with E4M3 keys are exact then, at the tensor core's 8-bit rate.
__device__ __forceinline__ void split_e4m3x4(const float (&v)[4], uint32_t& hi, uint32_t& lo) {
  const uint32_t h0 = cvt_e4m3x2_rn(v[0], v[1]), h1 = cvt_e4m3x2_rn(v[2], v[3]);
  const uint32_t f0 = f16x2_of_e4m3x2(h0), f1 = f16x2_of_e4m3x2(h1);
  const __half2 a = *reinterpret_cast<const __half2*>(&f0), b = *reinterpret_cast<const __half2*>(&f1);
  hi = h0 | (h1 << 16);
  lo = cvt_e4m3x2_rn(v[0] - __low2float(a), v[1] - __high2float(a)) |
       (cvt_e4m3x2_rn(v[2] - __low2float(b), v[3] - __high2float(b)) << 16);
}

// Shared-memory descriptors of operands that are contiguous along M or N (8-bit: 16 elements, 16-bit: 8 elements are a
// 16-byte unit). With the 128-byte swizzle: rows of 128 bytes along M or N, one per K; `sbo` between groups of 8 K,
// `lbo` between the 128-byte columns of M or N. Without: 16-byte rows, 8 K in 128 bytes; `lbo` between groups of 8 K,
// `sbo` between 16-byte columns.
constexpr uint32_t kIdescAlongM = 1u << 15, kIdescAlongN = 1u << 16;

// Instructions whose operands sit in uniform registers issue in a few clocks each; descriptors formed one by one in a loop
// took 130 clocks an MMA. So the groups of MMAs below are one asm statement each, which steps the descriptors' low words
// (start address and leading offset) itself.
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) { return ((saddr & 0x3FFFFu) >> 4) | (lbo >> 4) << 16; }
__host__ __device__ constexpr uint32_t desc_high(uint32_t sbo, bool swizzled) { return (sbo >> 4) | 1u << 14 | (swizzled ? 2u << 29 : 0u); }

// Two 32-wide steps of E4M3 operands along K (128-byte swizzle, 32 bytes a step), for two terms of B.
__device__ __forceinline__ void mma_along_k_2x2(uint32_t d, uint32_t a, uint32_t b0, uint32_t b1, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t;\n\t.reg .b32 a1, c0, c1;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 a1, %1, 2;\n\tadd.u32 c0, %2, 2;\n\tadd.u32 c1, %3, 2;\n\t"
      "mov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, p;\n\t"
      "mov.b64 db, {%3, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, t;\n\t"
      "mov.b64 da, {a1, %6};\n\tmov.b64 db, {c0, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, t;\n\t"
      "mov.b64 db, {c1, %6};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %4, t;\n\t}" ::"r"(d),
      "r"(a), "r"(b0), "r"(b1), "r"(idesc), "r"(acc), "r"(desc_high(1024, true))
      : "memory");
}

// The CTA whose range holds tile x, of `ctas` equal ranges of `total` tiles; range c is [c * total / ctas, ...).
__device__ __forceinline__ int kv_owner(int x, int total, int ctas) { return (int)((((int64_t)x + 1) * ctas - 1) / total); }

// Loads of TMEM columns of this lane, and the wait that ties them.
template <int N>
__device__ __forceinline__ void kv_ld(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32, "16 or 32 columns");
  if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
  }
}
template <int N>
__device__ __forceinline__ void kv_tie(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void kv_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void kv_bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
// Barrier of `threads` threads that tells all of them whether any has p.
__device__ __forceinline__ bool kv_bar_any(int id, int threads, bool p) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((int)p)
      : "memory");
  return r != 0;
}

}  // namespace mambo
