// Products of NVFP4 rows and weights on tcgen05 (kind::mxf4nvf4, E4M3 scales per 16):
//   out[m][n] = fx[m] * fw[n] * sum_k (sum_p cx[p][m][k] sx[p][m][k / 16]) cw[n][k] sw[n][k / 16]
//
// Weight rows are the MMA's M, activation rows its N: a single token is a column block of 16 that
// the tensor cores fill, and the pieces of a row are further MMAs into the same sums that share the
// weight tile in shared memory.  Products of codes and scales are exact, sums f32.
//
// Scales go from shared to tensor memory by tcgen05.cp (32 lanes x 16 bytes, repeated in the four
// lane quarters), which is why they are kept in blocks of 128 rows x 64 columns: a block is the 512
// bytes of one such copy, and a stage's four blocks one contiguous copy from global memory.  A ring
// stage is 256 columns: 128 bytes of codes a row.
#include <string>

#include "g4_nvfp4.cuh"
#include "g4_paged_split.cuh"

namespace g4 {

// ---------------------------------------------------------------------------- PTX
__device__ __forceinline__ uint64_t nv_scale_desc(uint32_t addr) {  // 8-row groups of 128 bytes, no swizzle
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) |
         (static_cast<uint64_t>(1u) << 46);
}
template <int kCtas>
__device__ __forceinline__ void nv_cp_scales(uint32_t taddr, uint64_t desc) {
  if (kCtas == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int kCtas>
__device__ __forceinline__ void nv_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t acc) {
  if (kCtas == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
        : "memory");
}
__device__ __forceinline__ void nv_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void nv_tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void nv_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void nv_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  pa_ld_wait();
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Whether it holds for all of the 256 threads of the output warps, which meet here.
__device__ __forceinline__ bool nv_agree(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}

// A sum (2^-20 to 2^45, or 0) times the factors of its row and its weight row.  The factors' product comes first: where
// both are within 2^-60 to 2^60 it is a normal number, and the result leaves f32's range only if it has to.  Other
// factors (rows next to an end of bf16's range) may have a product beyond f32 that the sum brings back, and so may
// the sum and either of them: 64 bits.
__device__ __forceinline__ bool nv_plain(float f) { return !(fabsf(f) > 0x1p60f) && !(fabsf(f) < 0x1p-60f && f != 0.f); }
__device__ __noinline__ float nv_wide(float v, float fx, float fw) {
  return static_cast<float>(static_cast<double>(v) * fx * fw);
}

// ---------------------------------------------------------------------------- single CTAs
// A tile is 128 weight rows x `cols` activation rows; a cluster of `splits` CTAs shares its K range, and
// each CTA then adds up 128 / splits of the tile's rows, whose parts the others stored into its
// shared memory (in the cluster's order: no result hangs on timing).
//
// What bounds it: few rows are a read of the weights, 2.7 us of the 17.7 MB of 8192 x 3840, and the chain around it:
// launch, a CTA's first stage, its 4 to 15 stages, the exchange in the cluster and the end, 4 us more.  One token
// takes 6.7 us, 32 rows of 3840 x 8192 7.5 us.  Scales by tcgen05.st instead of the copy took longer, and so did a
// warp of their own for the copies, or copying a stage ahead.
constexpr int kNvTileThreads = 320;  // warp 0 copies, 1 MMA and tensor memory, 2-9 output
constexpr int kNvMaxStages = 8;

struct NvTileArgs {
  NvMatmulArgs a;
  int cols, splits, stages, stage_bytes, k_stages, kblocks, tmem_cols, row_tiles;
  size_t x_scale_piece;
};
struct NvTileBars {
  uint64_t full[kNvMaxStages], empty[kNvMaxStages], done;
  uint32_t tmem, abort;
  float fx[128], fw[128];
};

template <int P>
__global__ void __launch_bounds__(kNvTileThreads, 1)
    nv_tile_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const __grid_constant__ NvTileArgs t, Scratch* scr, uint64_t budget) {
  extern __shared__ uint8_t nv_raw[];
  __shared__ NvTileBars sm;
  const NvMatmulArgs& a = t.a;
  const uint32_t base = (smem_u32(nv_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % t.splits, tile = blockIdx.x / t.splits;
  const int n0 = tile % t.row_tiles * 128, m0 = tile / t.row_tiles * t.cols;
  const int ks0 = t.k_stages * rank / t.splits, ks1 = t.k_stages * (rank + 1) / t.splits;
  if (tid == 0) {
    for (int i = 0; i < t.stages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.done, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                 "r"(static_cast<uint32_t>(t.tmem_cols)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  if (t.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (this CTA runs)
  const uint32_t tbase = sm.tmem;
  volatile uint32_t* abort = &sm.abort;
  const uint32_t x_bytes = t.cols * 128;
  const uint32_t x_at = 16384, sw_at = x_at + P * x_bytes, sx_at = sw_at + 2048;

  if (warp == 0) {
    if (lane == 0) {
      const uint8_t* sw = a.w_scales + static_cast<size_t>(n0 >> 7) * t.kblocks * 512;
      const uint8_t* sx = a.x_scales + static_cast<size_t>(m0 >> 7) * t.kblocks * 512;
      auto weights = [&](int ks, int st) {
        const uint32_t to = base + st * t.stage_bytes, sf = min(4, t.kblocks - 4 * ks) * 512;
        mbar_arrive_expect_tx(&sm.full[st], 16384 + P * x_bytes + (1 + P) * sf);
        nv_tma_3d(to, &wmap, ks * 128, n0, 0, &sm.full[st]);
        nv_bulk(to + sw_at, sw + static_cast<size_t>(ks) * 2048, sf, &sm.full[st]);
      };
      auto rows = [&](int ks, int st) {
        const uint32_t to = base + st * t.stage_bytes, sf = min(4, t.kblocks - 4 * ks) * 512;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          nv_tma_3d(to + x_at + p * x_bytes, &xmap, ks * 128, m0, p, &sm.full[st]);
          nv_bulk(to + sx_at + p * 2048, sx + p * t.x_scale_piece + static_cast<size_t>(ks) * 2048, sf, &sm.full[st]);
        }
      };
      const int ahead = min(t.stages, ks1 - ks0);
      if (a.early)
        for (int i = 0; i < ahead; ++i) weights(ks0 + i, i);
      pdl_wait();
      pdl_launch_dependents();
      PaRing at(0, t.stages);
      for (int ks = ks0; ks < ks1; ++ks, at.next()) {
        if (ks - ks0 >= ahead && !pa_wait(&sm.empty[at.stage], at.parity ^ 1, abort, budget)) break;
        if (!a.early || ks - ks0 >= ahead) weights(ks, at.stage);
        rows(ks, at.stage);
      }
    }
  } else if (warp == 1) {
    pdl_wait();  // (the budget of a wait is for this kernel's copies, not for what the kernel before has left to do)
    constexpr uint32_t kStep = 4 * (1 + P);
    const uint32_t idesc = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(t.cols >> 3) << 17) | (8u << 24);
    const uint32_t sfa = tbase + t.cols;
    const bool leader = pa_elect();
    const uint64_t wd0 = pa_desc(base, 16, 1024), xd0 = pa_desc(base + x_at, 16, 1024);
    const uint64_t swd0 = nv_scale_desc(base + sw_at), sxd0 = nv_scale_desc(base + sx_at);
    const uint32_t stage16 = t.stage_bytes / 16, piece16 = x_bytes / 16;
    const uint32_t shift = (m0 & 127) >> 5;
    PaRing at(0, t.stages);
    for (int ks = ks0; ks < ks1; ++ks) {
      if (!pa_wait_warp(&sm.full[at.stage], at.parity, abort, budget)) break;
      pa_fence_after();
      const uint64_t off = at.stage * stage16;
      const int steps = t.kblocks - 4 * ks;
      if (leader) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s < steps) {
            nv_cp_scales<1>(sfa + s * kStep, swd0 + off + 32 * s);
#pragma unroll
            for (int p = 0; p < P; ++p) nv_cp_scales<1>(sfa + s * kStep + 4 + 4 * p, sxd0 + off + 128 * p + 32 * s);
          }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s < steps) {
#pragma unroll
            for (int p = 0; p < P; ++p)
              nv_mma<1>(tbase, wd0 + off + 2 * s, xd0 + off + p * piece16 + 2 * s, idesc, sfa + s * kStep,
                        sfa + s * kStep + 4 + 4 * p + shift, (s | p) ? 1u : static_cast<uint32_t>(ks - ks0));
          }
        }
        nv_commit(&sm.empty[at.stage]);
        if (ks == ks1 - 1) nv_commit(&sm.done);
      }
      __syncwarp();
      at.next();
    }
    // (every MMA is done before tensor memory is given back)
    pa_wait_warp(&sm.done, 0, abort, budget);
  }
  __syncwarp();
  // output: two warps a lane quarter, every other 16 columns each
  const int q = warp & 3, e = tid - 64, r = 32 * q + lane;
  const int valid = min(t.cols, a.m - m0);
  const uint32_t from = tbase + (static_cast<uint32_t>(32 * q) << 16);
  bool got = true, plain = true;
  if (warp >= 2) {
    pdl_wait();
    if (e < valid) {
      sm.fx[e] = a.x_factor[m0 + e];
      plain = nv_plain(sm.fx[e]);
    } else if (e >= 128) {
      sm.fw[e - 128] = n0 + e - 128 < a.n ? a.w_factor[a.n_factors > 1 ? n0 + e - 128 : 0] : 0.f;
      plain = nv_plain(sm.fw[e - 128]);
    }
    plain = nv_agree(plain);
    got = pa_wait_warp(&sm.done, 0, abort, budget);
    pa_fence_after();
  }
  float part[16];
  auto store = [&](int c, int row, float v) {  // (rows past the weight are nobody's)
    if (row >= a.n) return;
    const size_t to = static_cast<size_t>(m0 + c) * a.out_stride + row;
    if (a.out_f32)
      static_cast<float*>(a.out)[to] = v;
    else
      static_cast<uint16_t*>(a.out)[to] = f32_to_bf16(v);
  };
  if (t.splits == 1) {
    if (warp >= 2 && got) {
      const float fw = sm.fw[r];
      for (int c0 = 16 * (e >> 7); c0 < valid; c0 += 32) {
        nv_ld16(from + c0, part);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < valid) store(c0 + j, n0 + r, plain ? part[j] * (sm.fx[c0 + j] * fw) : nv_wide(part[j], sm.fx[c0 + j], fw));
      }
    }
  } else {
    // row r of the tile is added up by CTA r / per; its parts lie there as [cta][column quad][row][4]
    const int shift = __ffs(128 / t.splits) - 1, per = 1 << shift, quads = (valid + 3) / 4;
    const uint32_t red = base + t.stages * t.stage_bytes;
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // (they all run)
    if (warp >= 2 && got) {
      const uint32_t to = pa_map_to(red + (static_cast<uint32_t>((rank * quads << shift) + (r & (per - 1))) << 4), r >> shift);
      for (int c0 = 16 * (e >> 7); c0 < valid; c0 += 32) {
        nv_ld16(from + c0, part);
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          if (c0 + j < valid)
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (((c0 + j) / 4 << shift) << 4)),
                         "f"(part[j]), "f"(part[j + 1]), "f"(part[j + 2]), "f"(part[j + 3])
                         : "memory");
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp >= 2 && got) {
      const int all = quads << shift;
      for (int x = e; x < all; x += 256) {
        const int own = rank * per + (x & (per - 1)), c = (x >> shift) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < t.splits; ++s) {
          const uint4 v = lds128(red + (static_cast<uint32_t>(s * all + x) << 4));
          sum.x += __uint_as_float(v.x), sum.y += __uint_as_float(v.y);
          sum.z += __uint_as_float(v.z), sum.w += __uint_as_float(v.w);
        }
        const float f = sm.fw[own];
        float out[4] = {sum.x, sum.y, sum.z, sum.w};
        if (plain) {
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] *= sm.fx[c + j] * f;
        } else {
          for (int j = 0; j < 4; ++j) out[j] = nv_wide(out[j], sm.fx[c + j], f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < valid) store(c + j, n0 + own, out[j]);
      }
    }
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  if (sm.abort != 0) {
    // Gave up somewhere, whichever warp it was: say so.  Copies that no product will take and products issued before may
    // be under way (the copying lane may have had no wait of its own left): let them land (bounded) before memory is
    // given back.
    if (tid == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
    const uint64_t end = global_ns() + 1000000;
    while (global_ns() < end) __nanosleep(1000);
  }
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase),
                 "r"(static_cast<uint32_t>(t.tmem_cols)));
}

// ---------------------------------------------------------------------------- CTA pairs
// Tiles of 256 weight rows x `cols` activation rows for many rows: each CTA of a pair holds 128 of the
// weight rows and half of the activation rows of a stage (cta_group::2), all of their scales, and
// gets the sums of its 128 weight rows.  Pairs take tiles in turn.
//
// Tensor memory: two sums of `cols` columns and one stage's scales do not fit side by side at 256, so the
// sums overlap (columns acc_step to cols): the next tile's products start once these have been read.
//
// What bounds it: 4096 rows of 8192 x 3840 take 52.6 us in one piece (4.9 PFLOP/s, 75 % of four times the measured
// bf16 rate) and 88.6 us in two (5.8 PFLOP/s, 89 %).  In one piece it is the way from L2 to the SMs: a stage's 39 KB
// for 128 x 256 x 256 products of an SM are 54 bytes a clock at the full rate, and copies alone ran at 58.  A
// second piece uses each weight tile twice.  Other orders of the tiles, and weights fetched while the
// activations are quantised (509 rows 22.0 us instead of 20.2), did not help.
constexpr int kNvPairThreads = 320;  // warp 0 copies, 1 MMA (leader) and tensor memory, 2-9 output

struct NvPairArgs {
  NvMatmulArgs a;
  int cols, stages, stage_bytes, k_stages, kblocks, row_tiles, tiles;
  int acc_step, first_chunks;  // column of the second sums; chunks of 32 columns per warp in the overlap
};
struct NvPairBars {
  uint64_t full[kNvMaxStages], empty[kNvMaxStages], d_full[2], d_free[2];
  uint32_t tmem, abort;
  __align__(16) float fx[2][256];
};
constexpr int kNvOutBytes = 32 * 128 * 2;  // a chunk on its way out; two for each group of output warps
__device__ __forceinline__ void nv_pair_tma(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

template <int P, int kBlocks, bool kF32>
__global__ void __launch_bounds__(kNvPairThreads, 1)
    nv_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                   const __grid_constant__ CUtensorMap wsmap, const __grid_constant__ CUtensorMap xsmap,
                   const __grid_constant__ CUtensorMap omap, const __grid_constant__ NvPairArgs t, Scratch* scr, uint64_t budget) {
  extern __shared__ uint8_t nv_raw[];
  __shared__ NvPairBars sm;
  const NvMatmulArgs& a = t.a;
  const uint32_t base = (smem_u32(nv_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int half = t.cols / 2;
  if (tid == 0) {
    for (int i = 0; i < t.stages; ++i) {
      mbar_init(&sm.full[i], 2);
      mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.d_full[i], 1);
      mbar_init(&sm.d_free[i], 16);
    }
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // both CTAs' barriers and tensor memory are ready
  const uint32_t tbase = sm.tmem;
  volatile uint32_t* abort = &sm.abort;
  const uint32_t x_at = 16384, sw_at = x_at + P * half * 128, sx_at = sw_at + 2048;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t full0 = pa_map_to(smem_u32(&sm.full[0]), 0);
      const uint32_t bytes = 16384 + P * half * 128 + 2048 + P * kBlocks * 2048;
      bool ok = true;
      PaRing at(0, t.stages);
      auto free = [&]() {  // the stage's last products are done
        return at.passed < static_cast<uint32_t>(t.stages) || pa_wait(&sm.empty[at.stage], at.parity ^ 1, abort, budget);
      };
      pdl_wait();
      pdl_launch_dependents();
      for (int tile = pair; tile < t.tiles && ok; tile += pairs) {
        const int n0 = tile % t.row_tiles * 256 + 128 * cta, m0 = tile / t.row_tiles * t.cols;
        for (int ks = 0; ks < t.k_stages && (ok = free()); ++ks) {
          const uint32_t to = base + at.stage * t.stage_bytes, bar = full0 + 8 * at.stage;
          pa_expect_cluster(bar, bytes);
          nv_pair_tma(to, &wmap, ks * 128, n0, 0, bar);
#pragma unroll
          for (int p = 0; p < P; ++p) nv_pair_tma(to + x_at + p * half * 128, &xmap, ks * 128, m0 + half * cta, p, bar);
          nv_pair_tma(to + sw_at, &wsmap, ks * 256, n0 >> 7, 0, bar);
#pragma unroll
          for (int p = 0; p < P; ++p) nv_pair_tma(to + sx_at + p * kBlocks * 2048, &xsmap, ks * 256, m0 >> 7, p, bar);
          at.next();
        }
      }
      // Every copy has landed (the leader's products took it) once its stage is free again; both
      // CTAs stay until then.
      for (int i = 0; i < t.stages && ok; ++i, at.next()) ok = free();
    }
  } else if (warp == 1) {
    if (cta == 0) {
      pdl_wait();  // (as in the kernel above: no budget runs before it)
      const uint32_t idesc = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(t.cols >> 3) << 17) | (16u << 24);
      constexpr uint32_t kStep = 4 + 4 * kBlocks * P;  // scale columns of 64 columns' products
      const uint32_t sfa = tbase + 512 - 4 * kStep;
      const bool leader = pa_elect();
      const uint64_t wd0 = pa_desc(base, 16, 1024), xd0 = pa_desc(base + x_at, 16, 1024);
      const uint64_t swd0 = nv_scale_desc(base + sw_at), sxd0 = nv_scale_desc(base + sx_at);
      const uint32_t stage16 = t.stage_bytes / 16, piece16 = half * 8;
      bool ok = true;
      PaRing at(0, t.stages);
      uint32_t ti = 0;
      for (int tile = pair; tile < t.tiles && ok; tile += pairs, ++ti) {
        if (ti >= 1) ok = pa_wait_warp(&sm.d_free[(ti - 1) & 1], ((ti - 1) >> 1) & 1, abort, budget);
        pa_fence_after();
        const uint32_t d = tbase + (ti & 1) * t.acc_step;
        const uint32_t shift = ((tile / t.row_tiles * t.cols) & 127) >> 5;
        for (int ks = 0; ks < t.k_stages && ok; ++ks) {
          ok = pa_wait_warp(&sm.full[at.stage], at.parity, abort, budget);
          if (!ok) break;
          pa_fence_after();
          const uint64_t off = at.stage * stage16;
          const int steps = t.kblocks - 4 * ks;
          if (leader) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              if (s < steps) {
                const uint32_t sf = sfa + s * kStep;
                nv_cp_scales<2>(sf, swd0 + off + 32 * s);
#pragma unroll
                for (int b = 0; b < P * kBlocks; ++b) nv_cp_scales<2>(sf + 4 + 4 * b, sxd0 + off + 128 * b + 32 * s);
#pragma unroll
                for (int p = 0; p < P; ++p)
                  nv_mma<2>(d, wd0 + off + 2 * s, xd0 + off + p * piece16 + 2 * s, idesc, sf, sf + 4 + 4 * p * kBlocks + shift,
                            (s | p) ? 1u : static_cast<uint32_t>(ks));
              }
            }
            pa_commit(&sm.empty[at.stage]);
            if (ks == t.k_stages - 1) pa_commit(&sm.d_full[ti & 1]);
          }
          __syncwarp();
          at.next();
        }
      }
      // (the other CTA's last arrivals: nothing of it may be under way when this one ends)
      if (ok && ti > 0) ok = pa_wait_warp(&sm.d_free[(ti - 1) & 1], ((ti - 1) >> 1) & 1, abort, budget);
    }
  } else {
    // -------------------------------------------------------------- output
    pdl_wait();
    const int e = tid - 64, q = warp & 3, group = e >> 7, chunks = t.cols / 32;
    const uint32_t lanes = static_cast<uint32_t>(32 * q) << 16;
    const uint32_t free0 = pa_map_to(smem_u32(&sm.d_free[0]), 0);
    const uint32_t stage = base + t.stages * t.stage_bytes + group * 2 * kNvOutBytes;
    const bool sender = (e & 127) == 0;
    bool ok = true;
    uint32_t ti = 0, sent = 0;
    for (int tile = pair; tile < t.tiles; tile += pairs, ++ti) {
      const int n0 = tile % t.row_tiles * 256 + 128 * cta, m0 = tile / t.row_tiles * t.cols;
      const int n = n0 + 32 * q + lane;
      const float fw = n < a.n ? a.w_factor[a.n_factors > 1 ? n : 0] : 0.f;
      float* fx = sm.fx[ti & 1];
      if (e < t.cols) fx[e] = m0 + e < a.m ? a.x_factor[m0 + e] : 0.f;
      const bool plain = nv_agree(nv_plain(fw) && (e >= t.cols || nv_plain(fx[e])));
      if (t.first_chunks == 0) {  // (this tile's sums lie beside the previous tile's, which have been read)
        pa_fence_before();
        __syncwarp();
        if (lane == 0) pa_arrive_relaxed(free0 + 8 * (ti & 1));
      }
      ok = nv_agree(pa_wait_warp(&sm.d_full[ti & 1], (ti >> 1) & 1, abort, budget));
      if (!ok) break;
      pa_fence_after();
      const uint32_t d = tbase + (ti & 1) * t.acc_step + lanes;
      for (int j = group; j < chunks; j += 2) {
        // the overlap first: the top of the first sums, the bottom of the second
        const int c0 = 32 * ((ti & 1) ? j : chunks - 1 - j);
        float v[32];
        pa_ld32(d + c0, v);
        pa_ld_wait();
        if (j >> 1 == t.first_chunks - 1) {
          pa_fence_before();
          __syncwarp();
          if (lane == 0) pa_arrive_relaxed(free0 + 8 * (ti & 1));
        }
        const int valid = a.m - (m0 + c0);  // rows of the chunk that there are
        if (valid <= 0 || n0 >= a.n) continue;
        if (plain) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(fx + c0 + c);
            v[c] *= f.x * fw, v[c + 1] *= f.y * fw, v[c + 2] *= f.z * fw, v[c + 3] *= f.w * fw;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = nv_wide(v[c], fx[c0 + c], fw);
        }
        if (kF32 || (a.n % 8 != 0 && n0 + 128 > a.n)) {
          // (a copy out of shared memory writes whole 16 bytes, past an end that is not on such a border)
          if (n < a.n) {
            const size_t to = static_cast<size_t>(m0 + c0) * a.out_stride + n;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (c >= valid) continue;
              if (kF32)
                static_cast<float*>(a.out)[to + c * a.out_stride] = v[c];
              else
                static_cast<uint16_t*>(a.out)[to + c * a.out_stride] = f32_to_bf16(v[c]);
            }
          }
        } else {
          // [32 activation rows][128 weight rows] leave as one copy: 256 bytes a row, clipped to what there is
          const uint32_t buf = stage + (sent & 1) * kNvOutBytes;
          if (sent >= 2) {
            if (sender) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            named_bar_sync(2 + group, 128);
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const uint32_t two = pack_bf16x2(v[c], v[c + 1]);
            const uint32_t to = buf + c * 256 + 2 * (32 * q + lane);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(static_cast<uint16_t>(two)) : "memory");
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + 256), "h"(static_cast<uint16_t>(two >> 16)) : "memory");
          }
          fence_proxy_async();
          named_bar_sync(2 + group, 128);
          if (sender) {
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                             reinterpret_cast<uint64_t>(&omap)),
                         "r"(n0), "r"(m0 + c0), "r"(buf)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          ++sent;
        }
      }
    }
    if (sender) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // (shared memory is still there for them)
    __syncwarp();
  }
  __syncthreads();
  if (sm.abort != 0) {  // gave up somewhere: say so, and let the copies in flight land (bounded)
    if (tid == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
    const uint64_t end = global_ns() + 1000000;
    while (global_ns() < end) __nanosleep(1000);
  }
  pa_fence_before();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  pa_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(512u));
}

// ---------------------------------------------------------------------------- host side
// CTAs of clusters ask for all of an SM's shared memory, so that an SM has one of them at a time: tensor memory is
// not among what a cluster is given before it starts, and a CTA that waits for columns while its cluster waits
// for it, beside another cluster's in the same position, would wait for good.
constexpr size_t kNvSmem = 229376;
// Codes [planes][rows][cols bytes] (row stride cols), box of box_rows x 128 bytes, 128-byte swizzle;
// what lies past the rows and the columns reads as zeros.
static bool nv_code_map(CUtensorMap* m, const void* p, int cols, int rows, int planes, size_t plane, int box_rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(planes > 1 ? plane : cols)};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_rows), 1}, each[3] = {1, 1, 1};
  const EncodeFn fn = tensor_map_encoder();
  return fn != nullptr && fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(p), dims, strides, box, each,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scale blocks [planes][row blocks][column blocks of 512 bytes], box of box_rows row blocks x 4 column blocks.
static bool nv_scale_map(CUtensorMap* m, const void* p, int kblocks, int rows, int planes, int box_rows) {
  const cuuint64_t row = static_cast<cuuint64_t>(kblocks) * 512, blocks = (static_cast<cuuint64_t>(rows) + 127) / 128;
  const cuuint64_t dims[3] = {row / 8, blocks, static_cast<cuuint64_t>(planes)}, strides[2] = {row, row * blocks};
  const cuuint32_t box[3] = {256, static_cast<cuuint32_t>(box_rows), 1}, each[3] = {1, 1, 1};
  const EncodeFn fn = tensor_map_encoder();
  return fn != nullptr && fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT64, 3, const_cast<void*>(p), dims, strides, box, each,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The bf16 output [rows][cols], box of 32 rows x 128 columns.
static bool nv_out_map(CUtensorMap* m, const void* p, int cols, int rows, long long stride) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {128, 32}, each[2] = {1, 1};
  const EncodeFn fn = tensor_map_encoder();
  return fn != nullptr && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, each,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kF32>
static const void* pair_kernel(int pieces, int blocks) {
  if (blocks == 1)
    return pieces == 1   ? (const void*)nv_pair_kernel<1, 1, kF32>
           : pieces == 2 ? (const void*)nv_pair_kernel<2, 1, kF32>
                         : (const void*)nv_pair_kernel<3, 1, kF32>;
  return pieces == 1   ? (const void*)nv_pair_kernel<1, 2, kF32>
         : pieces == 2 ? (const void*)nv_pair_kernel<2, 2, kF32>
                       : (const void*)nv_pair_kernel<3, 2, kF32>;
}

static g4_status launch_pairs(g4_ctx* ctx, const NvMatmulArgs& a, int cols) {
  NvPairArgs t = {};
  t.a = a;
  t.cols = cols;
  const int blocks = cols > 128 ? 2 : 1;  // of scales, across a tile's activation rows
  t.kblocks = (a.k + 63) / 64;
  t.k_stages = (t.kblocks + 3) / 4;
  t.row_tiles = (a.n + 255) / 256;
  t.tiles = t.row_tiles * ((a.m + cols - 1) / cols);
  const int room = 512 - 4 * (4 + 4 * blocks * a.pieces);  // beside a stage's scales
  t.acc_step = 2 * cols <= room ? cols : room - cols;
  t.first_chunks = (cols - t.acc_step + 63) / 64;
  t.stage_bytes = 16384 + a.pieces * (cols / 2) * 128 + 2048 + a.pieces * blocks * 2048;
  const int out_bytes = a.out_f32 ? 0 : 4 * kNvOutBytes;
  t.stages = (static_cast<int>(kNvSmem) - 1024 - out_bytes) / t.stage_bytes;
  if (t.stages > kNvMaxStages) t.stages = kNvMaxStages;
  const size_t smem = kNvSmem;
  CUtensorMap wmap, xmap, wsmap, xsmap, omap;
  if (!nv_code_map(&wmap, a.w_codes, a.k / 2, a.n, 1, 0, 128) ||
      !nv_code_map(&xmap, a.x_codes, a.k / 2, a.m, a.pieces, static_cast<size_t>(a.max_rows) * (a.k / 2), cols / 2) ||
      !nv_scale_map(&wsmap, a.w_scales, t.kblocks, a.n, 1, 1) ||
      !nv_scale_map(&xsmap, a.x_scales, t.kblocks, a.max_rows, a.pieces, blocks) ||
      (!a.out_f32 && !nv_out_map(&omap, a.out, a.n, a.m, a.out_stride)))
    return fail(ctx, G4_ERR_CUDA, "cuTensorMapEncodeTiled failed (nvfp4 matmul)");
  const void* fn = a.out_f32 ? pair_kernel<true>(a.pieces, blocks) : pair_kernel<false>(a.pieces, blocks);
  const g4_status st = allow_max_dynamic_smem(ctx, fn, smem, "nvfp4 matmul");
  if (st != G4_OK) return st;
  Scratch* scr = ctx->buf.scratch;
  uint64_t budget = ctx->wait_budget_ns;
  void* args[] = {&wmap, &xmap, &wsmap, &xsmap, a.out_f32 ? &wmap : &omap, &t, &scr, &budget};
  const int pairs = t.tiles < ctx->sm_count / 2 ? t.tiles : ctx->sm_count / 2;
  return launch_kernel(ctx, fn, dim3(2 * pairs), dim3(kNvPairThreads), smem, args, false, "nvfp4 matmul", 2);
}

static g4_status launch_tiles(g4_ctx* ctx, const NvMatmulArgs& a, int cols, int splits) {
  NvTileArgs t = {};
  t.a = a;
  t.cols = cols;
  t.splits = splits;
  t.kblocks = (a.k + 63) / 64;
  t.k_stages = (t.kblocks + 3) / 4;
  t.x_scale_piece = nv_scale_bytes(a.max_rows, a.k);
  t.row_tiles = (a.n + 127) / 128;
  const int col_tiles = (a.m + t.cols - 1) / t.cols;
  t.tmem_cols = 32;
  while (t.tmem_cols < t.cols + 16 * (1 + a.pieces)) t.tmem_cols *= 2;
  t.stage_bytes = 16384 + a.pieces * t.cols * 128 + (1 + a.pieces) * 2048;
  const int red = t.splits > 1 ? 128 * t.cols * 4 : 0;
  const int room = static_cast<int>(kNvSmem) - 1024 - red;
  t.stages = room / t.stage_bytes < kNvMaxStages ? room / t.stage_bytes : kNvMaxStages;
  const int most = (t.k_stages + t.splits - 1) / t.splits;
  if (t.stages > most) t.stages = most;
  const size_t smem = t.splits > 1 ? kNvSmem : 1024 + static_cast<size_t>(t.stages) * t.stage_bytes;
  CUtensorMap wmap, xmap;
  if (!nv_code_map(&wmap, a.w_codes, a.k / 2, a.n, 1, 0, 128) ||
      !nv_code_map(&xmap, a.x_codes, a.k / 2, a.m, a.pieces, static_cast<size_t>(a.max_rows) * (a.k / 2), t.cols))
    return fail(ctx, G4_ERR_CUDA, "cuTensorMapEncodeTiled failed (nvfp4 matmul)");
  const void* fn = a.pieces == 1   ? (const void*)nv_tile_kernel<1>
                   : a.pieces == 2 ? (const void*)nv_tile_kernel<2>
                                   : (const void*)nv_tile_kernel<3>;
  const g4_status st = allow_max_dynamic_smem(ctx, fn, smem, "nvfp4 matmul");
  if (st != G4_OK) return st;
  Scratch* scr = ctx->buf.scratch;
  uint64_t budget = ctx->wait_budget_ns;
  void* args[] = {&wmap, &xmap, &t, &scr, &budget};
  return launch_kernel(ctx, fn, dim3(static_cast<unsigned>(t.row_tiles) * col_tiles * t.splits), dim3(kNvTileThreads), smem,
                       args, false, "nvfp4 matmul", t.splits);
}

// Which kernel, how wide a tile, how many CTAs to a K range: the least of what each would take, by a model of
// start + rounds x (K stages x a stage + a tile's end), in microseconds, fitted to sweeps of 1 to 4096
// activation rows over the decoder's projections and their tensor-parallel shares (1 to 3 pieces; it names
// the fastest or one within 6 % of it).  What it weighs, two pieces:
//   one token, 8192 x 3840       single CTAs 6.7, pairs 9.2    (more of them, K split: all SMs at work)
//   32 rows, 3840 x 4096         single CTAs 5.7, pairs 10.1
//   64 rows, 30720 x 3840        single CTAs 22.4, pairs of 64 columns 17.0
//   256 rows, 8192 x 3840        single CTAs 14.6, pairs of 128 columns 11.1, of 256 columns 15.8
//   509 rows, 8704 x 3840        pairs of 128 columns 17.6, of 256 columns 16.7
//   4096 rows, 8192 x 3840       pairs of 128 columns 103, of 256 columns 89
// Tiles start at multiples of 64 activation rows, or there is one: the MMA wants its scales at an even
// column of tensor memory.
g4_status launch_nvfp4_matmul(g4_ctx* ctx, const NvMatmulArgs& a) {
  const int stages = (a.k + 255) / 256, P = a.pieces;
  auto ceil = [](long long x, long long y) { return (x + y - 1) / y; };
  float best = 1e30f;
  int best_cols = 0, best_splits = 0;  // 0 splits: pairs
  auto offer = [&](float us, int cols, int splits) {
    if (us < best) best = us, best_cols = cols, best_splits = splits;
  };
  for (int cols = a.m <= 16 ? 16 : a.m <= 32 ? 32 : 64; cols <= 128; cols *= 2) {
    const long long tiles = ceil(a.n, 128) * ceil(a.m, cols);
    int splits = 1;
    while (splits < 8 && 2 * splits <= stages && 2 * splits * tiles <= ctx->sm_count) splits *= 2;
    const float stage = cols <= 64 ? 0.3f + 0.075f * P : 0.2f + 0.27f * P, end = 0.5f + 0.03f * (a.m < cols ? a.m : cols);
    offer(2.6f + ceil(tiles * splits, ctx->sm_count) * (ceil(stages, splits) * stage + end), cols, splits);
    if (a.m <= 32) break;
  }
  for (int cols = 64; cols <= 256; cols *= 2) {
    const float rounds = static_cast<float>(ceil(ceil(a.n, 256) * ceil(a.m, cols), ctx->sm_count / 2));
    if (cols == 64)
      offer(2.9f + rounds * (stages * (0.25f + 0.07f * P) + 0.55f), cols, 0);
    else if (cols == 128)
      offer(3.1f + rounds * (stages * (0.21f + 0.11f * P) + 0.8f), cols, 0);
    else
      offer(5.1f + rounds * (stages * (P == 1 ? 0.4f : P == 2 ? 0.62f : 1.1f) + 1.f), cols, 0);
  }
  return best_splits == 0 ? launch_pairs(ctx, a, best_cols) : launch_tiles(ctx, a, best_cols, best_splits);
}

}  // namespace g4
