// FP8 block-scaled product on tcgen05: out[t, n] = sum over K blocks b of
//   sw[n / 128, b] * sum_{k in b} (xq[t, k] * 2^e(t, k / 32)) * wq[n, k].
//
// The weight tile is the MMA's A operand (128 rows in the TMEM lanes), the
// tokens its N dimension, so one kernel serves one token and a full tile, and
// a ragged segment wastes at most 15 columns. The tensor core applies the
// activations' power-of-two scales itself (block-scaled MMA, one scale per 32
// K); a K block's partial product then has one factor left, the f32 scale of
// the 128 x 128 weight block: the epilogue warps add D * sw to their FP32
// registers, one packed FMA per two values, while the next block's MMAs run
// into another D buffer.
//
// Work: the (row tile, token tile) tiles of all experts, numbered expert by
// expert, token tiles inner. Whole waves of tiles go one per CTA; the rest
// (between one and two waves) is cut at K blocks into equal ranges, one per
// CTA (stream-K), so every CTA ends at the same time. A tile that several CTAs
// share is summed in K order by whichever arrives last: nothing waits.
//
// Warps: 0 weights producer, 1 MMA, 2 activations producer, 3 idle, then the
// epilogue warps, one per TMEM lane quadrant (and per half of the columns).
#include "fp8b.cuh"
#include "iq3s_tm.cuh"
#include "kernels.cuh"
#include "tcgen05.cuh"

namespace mambo {

namespace {

constexpr int kMaxStagesB = 12;

template <int NT>
struct FbCfg {
  static constexpr int kEpiWarps = NT > 64 ? 8 : 4;
  static constexpr int kCols = NT > 64 ? NT / 2 : NT;  // columns of an epilogue warp
  static constexpr int kD = NT > 64 ? 3 : 4;           // D buffers
  static constexpr uint32_t kDStride = NT;
  static constexpr uint32_t kSfa = kD * kDStride;      // weights' scale factors, all 2^0
  static constexpr uint32_t kSfb = kSfa + 16;          // activations' scale factors, 8 columns per D buffer
  static constexpr uint32_t kTmem = kSfb + 8 * kD <= 128 ? 128 : kSfb + 8 * kD <= 256 ? 256 : 512;
  static constexpr int kThreads = (4 + kEpiWarps) * 32;
  static constexpr int kApt = (NT + 127) / 128;
  static constexpr uint32_t kXBytes = NT * 128u;
  static constexpr uint32_t kStage = kFbRecord + kXBytes + kApt * kFbAtom;
  static_assert(kStage % 512 == 0, "stage");
  // Operand tiles start on 1024-byte boundaries: weights and tokens first, then all scale atoms.
  static constexpr uint32_t kTiles = kFbRecord + kXBytes;
  static_assert(kTiles % 1024 == 0, "swizzle atoms");
};

constexpr uint32_t kFbBarBytes = 512;

__host__ __device__ inline uint32_t fb_tables_bytes(int experts) {
  return ((uint32_t)(experts + 1) * 8 + 127) / 128 * 128;  // tile and row prefix
}

// This CTA's share of the tiles: a stream-K range over the first sk tiles,
// then one tile of each whole wave.
struct FbWalk {
  int kb_n, sk, waves, ncl, cl, nsk;
  int64_t u, u1, units;
  int wave;
  int tile, kb0, kb1;  // the current segment
  __device__ __forceinline__ FbWalk(int tiles, int kblocks, int cl_, int ncl_) {
    kb_n = kblocks;
    ncl = ncl_;
    cl = cl_;
    waves = tiles / ncl;
    if (tiles % ncl && waves > 0) --waves;
    sk = tiles - waves * ncl;
    units = (int64_t)sk * kb_n;
    nsk = (int)(units < ncl ? units : ncl);
    u = cl < nsk ? cl * units / nsk : 0;
    u1 = cl < nsk ? (cl + 1) * units / nsk : 0;
    wave = 0;
    tile = kb0 = kb1 = 0;
  }
  __device__ __forceinline__ bool next() {
    if (u < u1) {
      tile = (int)(u / kb_n);
      kb0 = (int)(u - (int64_t)tile * kb_n);
      const int64_t left = u1 - u;
      kb1 = left < kb_n - kb0 ? kb0 + (int)left : kb_n;
      u += kb1 - kb0;
      return true;
    }
    if (wave < waves) {
      tile = sk + wave * ncl + cl;
      ++wave;
      kb0 = 0;
      kb1 = kb_n;
      return true;
    }
    return false;
  }
  // The CTA whose range holds unit x.
  __device__ __forceinline__ int owner(int64_t x) const { return (int)(((x + 1) * nsk - 1) / units); }
};

// The tile's expert, row tile and tokens, from the prefix tables in shared memory.
struct FbTile {
  int e, rt, row0, n;  // n tokens from row row0 of the expert's segment
  int64_t prow, slot;
  int o;
};
struct FbCursor {
  const int* tiles;  // [experts + 1] first tile of each expert
  const int* offs;   // [experts + 1] clamped, non-decreasing
  int experts, row_tiles, nt, e;
  __device__ __forceinline__ FbTile at(int tile) {
    while (e + 1 < experts && tile >= tiles[e + 1]) ++e;
    FbTile t;
    t.e = e;
    t.o = offs[e];
    const int count = offs[e + 1] - t.o;
    const int tt_n = fb_tiles(count, nt), tr = fb_tile_rows(count, tt_n);
    const int local = tile - tiles[e];
    t.rt = local / tt_n;
    const int tt = local - t.rt * tt_n;
    t.row0 = tt * tr;
    t.n = count - t.row0 < tr ? count - t.row0 : tr;
    t.prow = fb_row_start(t.o, e) + t.row0;
    t.slot = fb_slot_start(t.o, e, nt) + tt;
    return t;
  }
};

// After a wait gave up: time for the bulk copies in flight to land before the CTA leaves its shared memory.
__device__ __forceinline__ void settle_copies() {
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

// D[tmem] (+)= A[smem] x (B[smem] * 2^sfb)^T, block scaled (A's factors are 2^0), issued by one thread.
__device__ __forceinline__ void mma_mx_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                          uint32_t tmem_sfa, uint32_t tmem_sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
          tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb));
}

}  // namespace

template <int NT>
__global__ void __launch_bounds__(FbCfg<NT>::kThreads, 1) fb_gemm_kernel(const __grid_constant__ FbGemmParams p) {
  using C = FbCfg<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* tiles0 = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int S = p.stages;
  uint8_t* atoms0 = tiles0 + (size_t)S * C::kTiles;
  int* tile_start = reinterpret_cast<int*>(atoms0 + (size_t)S * C::kApt * kFbAtom);
  int* offs = tile_start + p.experts + 1;
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(tile_start) + fb_tables_bytes(p.experts));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStagesB + 2 * 4 + 1);
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t kFull = bar0, kEmpty = bar0 + 8 * kMaxStagesB;
  const uint32_t kMdone = bar0 + 16 * kMaxStagesB, kEfree = kMdone + 8 * 4, kEdone = kEfree + 8 * 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KB = p.act.kblocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(kFull + 8 * s, 2);
      mbar_init(kEmpty + 8 * s, 1);
    }
    for (int d = 0; d < C::kD; ++d) {
      mbar_init(kMdone + 8 * d, 1);
      mbar_init(kEfree + 8 * d, C::kEpiWarps);
    }
    mbar_init(kEdone, C::kEpiWarps);
    fence_barrier_init();
  }
  if (warp == 1) {
    tc::alloc(smem_u32(tmem_slot), C::kTmem);
    tc::relinquish();
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
        int t = fb_tiles(o - before, NT) * p.row_tiles;
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
      tile_start[1] = fb_tiles((int)p.rows, NT) * p.row_tiles;
      offs[0] = 0;
      offs[1] = (int)p.rows;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // The weights' MMA scale factors: 2^0 in every lane and byte.
  if (warp >= 4 && warp < 8) {
    tc::st_x4(tmem + ((uint32_t)(32 * (warp & 3)) << 16) + C::kSfa, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu, 0x7F7F7F7Fu);
    tc::wait_st();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();

  FbWalk walk(tile_start[p.experts], KB, (int)blockIdx.x, (int)gridDim.x);
  FbCursor cur{tile_start, offs, p.experts, p.row_tiles, NT, 0};

  if (warp == 0) {
    // -------------------------------------------------------------- weights producer
    if (lane == 0) {
      const uint64_t policy = l2_policy_evict_first();
      int it = 0, s = 0;
      uint32_t ph = 0;
      bool ok = true;
      while (ok && walk.next()) {
        const FbTile t = cur.at(walk.tile);
        const uint8_t* rec = p.packed + (((int64_t)t.e * p.row_tiles + t.rt) * KB) * kFbRecord;
        for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
          if (it >= S && !mbar_wait_bounded(kEmpty + 8 * s, ph ^ 1, kSiteFbEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(kFull + 8 * s, kFbRecord);
          const uint32_t dst = smem_u32(tiles0 + (size_t)s * C::kTiles);
          if (p.evict_weights) {
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
    if (lane == 0) {
      pdl_wait();
      int it = 0, s = 0;
      uint32_t ph = 0;
      bool ok = true;
      while (ok && walk.next()) {
        const FbTile t = cur.at(walk.tile);
        const uint32_t xb = (uint32_t)((t.n + 7) / 8) * 1024u;
        const uint8_t* x = p.act.x8 + t.prow * 128;
        const uint8_t* sf = p.act.atoms + t.slot * KB * (C::kApt * kFbAtom);
        for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
          if (it >= S && !mbar_wait_bounded(kEmpty + 8 * s, ph ^ 1, kSiteFbEmpty)) {
            ok = false;
            break;
          }
          const uint32_t full = kFull + 8 * s;
          mbar_arrive_expect_tx(full, xb + C::kApt * kFbAtom);
          bulk_load(smem_u32(tiles0 + (size_t)s * C::kTiles) + kFbRecord, x + (int64_t)kb * p.act.rows_pad * 128, xb,
                    full);
          bulk_load(smem_u32(atoms0 + (size_t)s * C::kApt * kFbAtom), sf + (int64_t)kb * (C::kApt * kFbAtom),
                    C::kApt * kFbAtom, full);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) settle_copies();
    }
    __syncwarp();
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA
    int it = 0, s = 0, db = 0;
    uint32_t ph = 0, dph = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const FbTile t = cur.at(walk.tile);
      const uint32_t idesc = tc::idesc_mx_e4m3(128, (t.n + 15) / 16 * 16, 0, 0);
      for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++it) {
        ok = tm::warp_wait(kFull + 8 * s, ph, kSiteFbFull);
        if (ok && it >= C::kD) ok = tm::warp_wait(kEfree + 8 * db, dph ^ 1, kSiteFbEmpty);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t wt = smem_u32(tiles0 + (size_t)s * C::kTiles);
        const uint32_t at = smem_u32(atoms0 + (size_t)s * C::kApt * kFbAtom);
        const uint64_t adesc = tc::smem_desc_sw128(wt, 1024u), bdesc = tc::smem_desc_sw128(wt + kFbRecord, 1024u);
        const uint32_t d = tmem + (uint32_t)db * C::kDStride, sfb = tmem + C::kSfb + 8u * (uint32_t)db;
        if (tm::elect_one()) {
#pragma unroll
          for (int a = 0; a < C::kApt; ++a)
            tc::cp_32x128b_warpx4(sfb + 4u * a, tc::smem_desc(at + a * kFbAtom, 128u, 128u));
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_mx_ss(d, adesc + (uint64_t)(2 * j), bdesc + (uint64_t)(2 * j), idesc | ((uint32_t)j << 4),
                      tmem + C::kSfa, sfb, j != 0);
          tc::commit(kEmpty + 8 * s);
          tc::commit(kMdone + 8 * db);
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
        if (++db == C::kD) {
          db = 0;
          dph ^= 1;
        }
      }
    }
    // Free the TMEM once every epilogue warp has read its last results.
    mbar_wait_bounded(kEdone, 0, kSiteFbFull);
    __syncwarp();
    tc::fence_after_sync();
    tc::dealloc(tmem, C::kTmem);
  } else if (warp >= 4) {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, h = (warp - 4) >> 2;
    const int rl = 32 * q + lane;
    const int c0 = h * C::kCols;
    const uint32_t tq0 = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)c0;
    float acc[C::kCols];
    pdl_wait();  // the output and the workspace may belong to the previous kernel
    pdl_launch_dependents();
    int db = 0;
    uint32_t dph = 0;
    bool ok = true;
    while (ok && walk.next()) {
      const FbTile t = cur.at(walk.tile);
      const int cols = t.n - c0;  // this warp's valid columns (may be <= 0)
      const float* sw = p.scales + (((int64_t)t.e * p.row_tiles + t.rt) * 2 + (q & 1)) * KB;
#pragma unroll
      for (int i = 0; i < C::kCols; ++i) acc[i] = 0.f;
      float sv = 0.f;
      for (int kb = walk.kb0; kb < walk.kb1; ++kb) {
        if (kb == walk.kb0 || (kb & 31) == 0) sv = (kb & ~31) + lane < KB ? __ldg(sw + (kb & ~31) + lane) : 0.f;
        const float w = __shfl_sync(0xFFFFFFFFu, sv, kb & 31);
        ok = tm::warp_wait(kMdone + 8 * db, dph, kSiteFbFull);
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t tq = tq0 + (uint32_t)db * C::kDStride;
#pragma unroll
        for (int b = 0; b < C::kCols; b += 16) {
          if (b < cols) {
            const uint32_t off[2] = {(uint32_t)b, (uint32_t)b + 8u};
            float v[2][8];
            tc::ld_x8_multi<2>(tq, off, v);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < 8; i += 2)
                fma2(acc[b + 8 * j + i], acc[b + 8 * j + i + 1], v[j][i], v[j][i + 1], w, w);
          }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(kEfree + 8 * db);
        if (++db == C::kD) {
          db = 0;
          dph ^= 1;
        }
      }
      if (!ok) break;
      if (walk.kb0 != 0 || walk.kb1 != KB) {
        // A tile shared between CTAs: publish this warp's part, and sum all
        // parts in K order if it is the last to arrive.
        const int64_t u_tile = (int64_t)walk.tile * KB;
        const int first = walk.owner(u_tile), last = walk.owner(u_tile + KB - 1);
        constexpr int kQuads = NT / 4;
        auto part = [&](int cta) {
          // Slot 1 holds the part that starts its tile (the CTA's last tile), slot 0 the others.
          return reinterpret_cast<float4*>(p.partials) +
                 (((int64_t)cta * 2 + (cta == first ? 1 : 0)) * kQuads + c0 / 4) * 128 + rl;
        };
        float4* mine = part(walk.cl);
#pragma unroll
        for (int c = 0; c < C::kCols; c += 4)
          if (c < cols) __stcg(mine + (c / 4) * 128, make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]));
        __threadfence();
        __syncwarp();
        int* counter = p.counters + first * 8 + (warp - 4);
        int done = 0;
        if (lane == 0) done = atomic_add_acq_rel_gpu(counter, 1) == last - first;
        done = __shfl_sync(0xFFFFFFFFu, done, 0);
        if (!done) continue;
        if (lane == 0) *counter = 0;  // all parts are in: zero again for the next launch
        __threadfence();
#pragma unroll
        for (int c = 0; c < C::kCols; ++c) acc[c] = 0.f;
        for (int cta = first; cta <= last; ++cta) {
          const float4* src = part(cta);
#pragma unroll
          for (int c = 0; c < C::kCols; c += 4) {
            if (c < cols) {
              const float4 v = __ldcg(src + (c / 4) * 128);
              acc[c] += v.x;
              acc[c + 1] += v.y;
              acc[c + 2] += v.z;
              acc[c + 3] += v.w;
            }
          }
        }
      }
      const int row = t.rt * 128 + rl;
      if (row < p.n_rows) {
        const int64_t at = ((int64_t)t.o + t.row0 + c0) * p.ldo + row;
        if (p.out_bf16) {
          __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
          for (int c = 0; c < C::kCols; ++c)
            if (c < cols) o[(int64_t)c * p.ldo] = __float2bfloat16_rn(acc[c]);
        } else {
          float* o = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
          for (int c = 0; c < C::kCols; ++c)
            if (c < cols) o[(int64_t)c * p.ldo] = acc[c];
        }
      }
    }
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(kEdone);
    __syncwarp();
  }
}

// --------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------
namespace {
template <int NT>
uint32_t smem_of(int experts, int stages) {
  return 1024 + (uint32_t)stages * (FbCfg<NT>::kTiles + FbCfg<NT>::kApt * kFbAtom) + fb_tables_bytes(experts) +
         kFbBarBytes;
}
template <int NT>
cudaError_t launch_nt(const FbGemmParams& p, int grid, cudaStream_t stream) {
  const uint32_t smem = smem_of<NT>(p.experts, p.stages);
  const void* k = (const void*)fb_gemm_kernel<NT>;
  cudaError_t e = ensure_smem_attribute(k, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(k, dim3(grid), dim3(FbCfg<NT>::kThreads), smem, stream, p);
}
}  // namespace

int fb_tile_for(int64_t expected_rows) {
  return expected_rows <= 16 ? 16 : expected_rows <= 32 ? 32 : expected_rows <= 64 ? 64 : 128;
}

uint32_t fb_gemm_smem(int nt, int experts, int stages) {
  return nt == 16 ? smem_of<16>(experts, stages) : nt == 32 ? smem_of<32>(experts, stages)
         : nt == 64 ? smem_of<64>(experts, stages) : smem_of<128>(experts, stages);
}

int fb_gemm_stages(int nt, int experts, int smem_optin) {
  int s = kMaxStagesB;
  while (s > 2 && (int)fb_gemm_smem(nt, experts, s) > smem_optin) --s;
  return s;
}

int fb_gemm_grid(int, int sms) { return sms; }
size_t fb_partial_bytes(int nt, int sms) { return (size_t)sms * 2 * 128 * nt * sizeof(float); }

cudaError_t launch_fb_gemm(const FbGemmParams& p, int grid, cudaStream_t stream) {
  switch (p.act.nt) {
    case 16: return launch_nt<16>(p, grid, stream);
    case 32: return launch_nt<32>(p, grid, stream);
    case 64: return launch_nt<64>(p, grid, stream);
    default: return launch_nt<128>(p, grid, stream);
  }
}

}  // namespace mambo
