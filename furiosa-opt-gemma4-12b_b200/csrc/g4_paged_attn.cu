// Attention of a chunk of new tokens over the pages of their sequences, on tcgen05.
//   o = sum_j softmax_j(scale q.k_j) v_j over the visible rows j of the token's sequence
//
// Rows.  The query heads that share a KV head are rows of one matrix: row r of (sequence,
// KV head) is token r / G, head r % G of the group (G = query heads per KV head).  A CTA
// pair (cluster of 2, cta_group::2) works on a tile of 256 rows, 128 per CTA, over 128 cache
// rows at a time: one item is (sequence, row tile, KV head), one unit of it a 128-row key tile.
//   S[256][128] = Q K^T      each CTA stages its 128 Q rows and 64 of the 128 K rows
//   O[256][256] += P V       each CTA stages 128 of the 256 V columns; P is read from tensor memory
// so every K/V byte is fetched once per 256 rows (per SM pair), without multicast.  Tensor
// memory holds O (256 columns) and two S tiles (128 each; P overwrites its S), all 512
// columns: S of the next key tile runs while the softmax of this one does.  A head of 512 has
// twice the O columns, so its two halves of V are two pairs' work: both compute S (1.5x the
// products) and they run side by side, so the second fetch of K hits the L2.
//
// Softmax in f32 with the running maximum and sum, two threads per row (64 of the tile's 128
// columns each; the maxima meet in shared memory): the time from S to P is what the tensor
// cores wait for when a head is 256 wide.  O is rescaled only
// when a row's maximum rises by more than 2^8 (the maximum that P is relative to may lag:
// P <= 256 then, exact in range for f32 sums and for P's rounding to bf16).  P is rounded to
// bf16 once, V's type, as kind::f16 wants it; its error is 2^-8 per weight, the size of the
// output's own rounding.  What the rounding left over could go in as a second bf16, as
// g4_paged_few.cu does it, but here the products and the softmax are the bound: half as many
// products again took 97 us instead of 71 (sliding prompt of 4096 tokens) and 385 instead of 279
// (full).
//
// Work split.  All units of the call, in order, are cut into as many equal ranges as there
// are pairs (or half as many pairs of pairs for heads of 512), from the device-resident
// lengths: a long cache with few rows is split along its keys, a batch of any raggedness is
// balanced.  An item that crosses a range's end leaves partial sums (f32) that a second
// kernel joins in range order.
//
// Roles of a CTA's 16 warps: 0-7 softmax, 8 K copies, 9 MMA (leader CTA) and tensor memory,
// 10 V copies, 11 Q copies and the V tiles at a sequence's ends (TMA cannot stop at its last row;
// rows past it may hold NaN, and 0 * NaN is NaN, so they are zeroed there), 12-15 output: O of
// one item leaves while the scores and the softmax of the next are under way.
#include <cmath>
#include <string>

#include "g4_paged_split.cuh"

namespace g4 {

constexpr int kPaThreads = 512;
constexpr float kPaLog2e = 1.4426950408889634f;  // the softmax's exponentials are powers of two
constexpr int kPaRows = 256;      // rows per item (both CTAs)
constexpr int kPaStage = 32768;   // bytes per ring stage: 64 K rows x 256 dims, or 128 V rows x 128 dims
constexpr uint32_t kPaColS = 256; // tensor memory: O [0, 256), S/P tiles at 256 and 384
constexpr int kPaItemCost = 2;     // an item's start and end, in units, for the work split
// kind::f16, D f32, A and B bf16, M = 256; S: N = 128, both K-major; O: N = 256, B (V) MN-major
constexpr uint32_t kPaIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (16u << 17) | (16u << 24);
constexpr uint32_t kPaIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (32u << 17) | (16u << 24);
constexpr int kPaPartFloats = 128 * 256 + 2 * 128;  // a partial: O as [64 column quads][128 rows][4], then (m, l) [128][2]

template <int D>
struct __align__(1024) PaSmem {
  // K and V each have a ring of their own: every ring has one filler, which meets the phases of
  // its barriers one by one (a parity tells two neighbouring phases apart, not three)
  static constexpr int kK = D == 256 ? 3 : 2, kV = D == 256 ? 2 : 1, kStages = kK + kV;
  uint8_t q[D / 64][128 * 128];  // 64-dim blocks [128 rows][64], 128-byte swizzle
  uint8_t ring[kStages][kPaStage];  // K stages, then V stages
  uint64_t full[kStages], empty[kStages], s_full[2], p_full, pv_done, q_full, q_empty, edge_full, edge_done;
  uint64_t o_full, o_free, ml_full, ml_free;
  float m[128], l[2][128];  // an item's reference maxima and column halves' sums, for the output warps
  float top[2][128];        // the rows' maxima over each half of a tile's columns
  uint32_t tmem;
  uint32_t abort;
  PaRange range;
};

// ---------------------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t pa_map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void pa_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Relaxed: what they announce is ordered by the copies themselves (expect) or by the tensor
// memory fences around them (P).  A release at cluster scope costs about 1000 cycles here.
__device__ __forceinline__ void pa_expect_cluster(uint32_t addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(addr), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void pa_arrive_relaxed(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
// Arrives on the barrier at this address in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void pa_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void pa_tma(uint32_t dst, uint64_t map, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}
// The eight softmax warps agree on whether all of their waits held.
__device__ __forceinline__ bool pa_agree(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}
// The 16-byte chunks w[4 j .. 4 j + 3] (j < 4) of the four lanes of a quad, transposed: lane q
// gets chunk q of the quad's lane j in place j.
__device__ __forceinline__ void pa_quad_transpose(uint32_t (&w)[16], int lane) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & bit) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t give = up ? w[4 * j + i] : w[4 * (j | bit) + i];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, bit);
        if (up)
          w[4 * j + i] = got;
        else
          w[4 * (j | bit) + i] = got;
      }
    }
  }
}
template <int D>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPaThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                      const __grid_constant__ CUtensorMap qmap, const __grid_constant__ PaArgs a,
                      const __grid_constant__ PagedBatch b, Scratch* scr, uint64_t budget) {
  using Smem = PaSmem<D>;
  constexpr int kK = Smem::kK, kV = Smem::kV, kStages = Smem::kStages, kHalves = D / 256, kChunks = D / 256;  // a K tile is kChunks stages
  // (all of an SM's shared memory: there is no room to align it by hand)
  static_assert(sizeof(Smem) <= 232448, "an SM's shared memory");
  extern __shared__ __align__(1024) uint8_t pa_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(pa_raw);
  if ((smem_u32(pa_raw) & 1023u) != 0) {  // the swizzle counts on it
    if (threadIdx.x == 0) {
      atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
      a.tail[(blockIdx.x >> 1) / kHalves] = PaTail{-1, 0, 0, 0};
    }
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x & 1;  // rank in the pair
  const int half = (blockIdx.x >> 1) % kHalves, range = (blockIdx.x >> 1) / kHalves;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 2);
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.s_full[0], 1);
    mbar_init(&sm.s_full[1], 1);
    mbar_init(&sm.p_full, 16);
    mbar_init(&sm.pv_done, 1);
    mbar_init(&sm.q_full, a.q_tma ? 2 : 16);
    mbar_init(&sm.q_empty, 1);
    mbar_init(&sm.edge_full, 1);
    mbar_init(&sm.edge_done, 1);
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.o_free, 8);
    mbar_init(&sm.ml_full, 8);
    mbar_init(&sm.ml_free, 4);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  pdl_wait();
  pdl_launch_dependents();
  PaCount* w = reinterpret_cast<PaCount*>(&sm.ring[0][0]);  // (the ring is not in use yet)
  static_assert(G4_PAGED_MAX_SEQS * sizeof(PaCount) <= kStages * kPaStage, "unit counts fit the ring");
  pa_count(b, a, w, scr, blockIdx.x == 0);
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  if (warp == 0) {
    const PaRange found = pa_range(b, a, w, range, lane, scr);
    if (lane == 0) sm.range = found;
    fence_proxy_async();  // the ring's next writers are TMA copies
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // both CTAs' barriers and memory are ready
  const uint32_t tbase = sm.tmem;
  const int u_first = sm.range.first;
  const int u_end = range < sm.range.count ? pa_share(range + 1, sm.range.units, sm.range.count) : u_first;
  volatile uint32_t* abort = &sm.abort;
  PaWalk it(b, a, sm.range, u_end - u_first);

  // registers a thread: 128 at launch (512 x 128 in all), 8 of the output's for each softmax warp
  // group: 128 x (2 x 136 + 128 + 112) = 65536.  (Sliding 4096-token prompt: 69.4 us; 76.2 us
  // with 128 everywhere, 74.4 us with 152, 80 and 128.)
  if (warp < 8)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
  else if (warp >= 12)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
  if (warp < 8) {
    // -------------------------------------------------------------- softmax
    const int side = warp >> 2, r = tid & 127;  // half of the columns; row of the CTA's 128
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t p_full = pa_map_to(smem_u32(&sm.p_full), 0);
    // scores are scaled within the exponent's FMA; a scale that is not positive goes first
    const bool scale_first = !(a.scale > 0.f);
    const float factor_s = scale_first ? 1.f : a.scale;
    uint32_t g = 0, items = 0;  // units and items of the range
    // good: this warp's waits held; ok: every softmax warp's did, as of the last tile they met at
    // (they leave together: the others would wait at the barrier for a warp that left alone)
    bool good = true, ok = true;
    while (ok && it.next()) {
      const int rr = it.tile * kPaRows + cta * 128 + r;
      const int i = a.by_group.div(rr);
      const bool valid = i < it.s.n;
      const bool any_row = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps step
      const int pos = it.s.kv - it.s.n + i;
      const int hi = valid ? pos + 1 : 0, lo = valid ? pa_low(pos, a.window) : 0;
      if (!a.q_tma) {
        // rows of any group size: a thread copies one 16-byte column of every kStep-th row (the
        // previous item's scores are done: all these warps have read them and met since)
        constexpr int kRowChunks = D / 8, kStep = 256 / kRowChunks;
        const int ch = tid % kRowChunks;
        const uint32_t qb = smem_u32(&sm.q[0][0]) + (ch >> 3) * 16384;
        const uint16_t* q = a.q + it.head * a.group * a.q_hs + it.s.t0 * a.q_ts + 8 * ch;
#pragma unroll 4
        for (int row = tid / kRowChunks; row < 128; row += kStep) {
          const int x = it.tile * kPaRows + cta * 128 + row, qi = a.by_group.div(x);
          const bool in = qi < it.s.n;
          cp_async16(qb + pa_swizzle(row, ch), in ? q + qi * a.q_ts + (x - qi * a.group) * a.q_hs : a.q, in ? 16u : 0u);
        }
        cp_async_wait_all();
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        if (lane == 0) pa_arrive_cluster(pa_map_to(smem_u32(&sm.q_full), 0));
      }
      float m = -CUDART_INF_F, l = 0.f;
      for (int u = it.begin; u < it.end; ++u, ++g) {
        const uint32_t st = tbase + kPaColS + (g & 1) * 128 + lanes;
        good = good && pa_wait_warp(&sm.s_full[g & 1], (g >> 1) & 1, abort, budget);
        float s[2][32];
        float mine = -CUDART_INF_F;
        if (any_row) {
          pa_fence_after();
          pa_ld32(st + 64 * side, s[0]);
          pa_ld32(st + 64 * side + 32, s[1]);
          pa_ld_wait();
          if (scale_first) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < 32; ++j) s[c][j] *= a.scale;
          }
          const int base = (it.kt0 + u) * kPaKeys;
          if (__any_sync(0xffffffffu, valid && (hi < base + kPaKeys || lo > base))) {
            const int from = lo - base - 64 * side, to = hi - base - 64 * side;  // visible: columns [from, to)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int f = min(max(from - 32 * c, 0), 32), t = min(max(to - 32 * c, 0), 32);
              const uint32_t see = static_cast<uint32_t>(((1ull << t) - 1ull) & ~((1ull << f) - 1ull));
#pragma unroll
              for (int j = 0; j < 32; ++j) s[c][j] = (see >> j) & 1u ? s[c][j] : -CUDART_INF_F;
            }
          }
          float mx[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float* x = &s[c >> 1][16 * (c & 1)];
            mx[c] = pa_max3(x[0], x[1], x[2]);
#pragma unroll
            for (int j = 3; j < 15; j += 2) mx[c] = pa_max3(mx[c], x[j], x[j + 1]);
            mx[c] = fmaxf(mx[c], x[15]);
          }
          mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * factor_s;
        }
        named_bar_sync(3, 256);  // the previous tile's maxima have been read
        sm.top[side][r] = mine;
        ok = pa_agree(good);
        if (!ok) break;
        float factor = 1.f;
        if (any_row) {
          const float top = fmaxf(sm.top[0][r], sm.top[1][r]);
          // the reference maximum: the first one seen, moved only when it lags too far
          if (m == -CUDART_INF_F) {
            m = top;
          } else if (top > m + kPaLag) {
            factor = pa_exp2(m - top);
            l *= factor;
            m = top;
          }
          const float ref = m == -CUDART_INF_F ? 0.f : -m;
          const uint64_t f2 = pa_pair(factor_s, factor_s), r2 = pa_pair(ref, ref);
          uint64_t sum[4] = {0, 0, 0, 0};
          uint32_t p[32];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float e0, e1, f0, f1;
            pa_unpair(pa_fma2(pa_pair(s[0][j], s[0][j + 1]), f2, r2), e0, e1);
            pa_unpair(pa_fma2(pa_pair(s[1][j], s[1][j + 1]), f2, r2), f0, f1);
            e0 = pa_exp2(e0);
            e1 = pa_exp2(e1);
            f0 = pa_exp2(f0);
            f1 = pa_exp2(f1);
            sum[(j >> 1) & 1] = pa_add2(sum[(j >> 1) & 1], pa_pair(e0, e1));
            sum[2 + ((j >> 1) & 1)] = pa_add2(sum[2 + ((j >> 1) & 1)], pa_pair(f0, f1));
            p[j / 2] = pa_bf16x2(e0, e1);
            p[16 + j / 2] = pa_bf16x2(f0, f1);
          }
          pa_st32(st + 32 * side, p);  // (both sides' scores have been read: the warps have met)
          float a0, a1;
          pa_unpair(pa_add2(pa_add2(sum[0], sum[1]), pa_add2(sum[2], sum[3])), a0, a1);
          l += a0 + a1;
        }
        // the previous P V is done: O may be rescaled, and this unit's may follow
        if (g != 0) {
          good = good && pa_wait_warp(&sm.pv_done, (g - 1) & 1, abort, budget);
          if (good && u != it.begin && __any_sync(0xffffffffu, factor != 1.f)) {
            pa_fence_after();
#pragma unroll 1
            for (int c = 128 * side; c < 128 * side + 128; c += 32) {
              float o[32];
              uint32_t x[32];
              pa_ld32(tbase + lanes + c, o);
              pa_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(o[j] * factor);
              pa_st32(tbase + lanes + c, x);
            }
          }
        }
        pa_st_wait();
        pa_fence_before();
        __syncwarp();
        if (lane == 0 && good) pa_arrive_relaxed(p_full);
      }
      if (!ok) break;
      if (items > 0) good = good && pa_wait_warp(&sm.ml_free, (items - 1) & 1, abort, budget);
      ++items;
      if (side == 0) sm.m[r] = m;
      sm.l[side][r] = l;
      __syncwarp();
      if (lane == 0 && good) mbar_arrive(&sm.ml_full);
    }
    if (ok && good && g > 0) good = pa_wait_warp(&sm.pv_done, (g - 1) & 1, abort, budget);
    if (!(ok && good) && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  } else if (warp >= 12) {
    // -------------------------------------------------------------- output
    const int r = tid - 384;  // row of the CTA's 128
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp - 12)) << 16;
    const uint32_t o_free = pa_map_to(smem_u32(&sm.o_free), 0);
    uint32_t items = 0;
    PaTail tail = {-1, 0, 0, 0};
    bool ok = true;
    while (ok && it.next()) {
      const int rr = it.tile * kPaRows + cta * 128 + r;
      const int i = a.by_group.div(rr), hg = rr - i * a.group;
      const bool valid = i < it.s.n;
      ok = pa_wait_warp(&sm.ml_full, items & 1, abort, budget) && pa_wait_warp(&sm.o_full, items & 1, abort, budget);
      if (!ok) break;
      ++items;
      const float2 ml = make_float2(sm.m[r], sm.l[0][r] + sm.l[1][r]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.ml_free);
      const bool whole = it.begin == 0 && it.end == it.nk;
      if (it.begin == 0 && it.end < it.nk) {
        // the item's last unit is at position u_end - it.end + it.nk - 1 of the call
        const int last = u_end - it.end + it.nk - 1;
        const long long e = ((last + 1ll) * sm.range.count - 1) / sm.range.units;
        tail = {it.seq, it.tile, it.head, static_cast<int>(e) - range + 1};
      }
      pa_fence_after();
      if (!__any_sync(0xffffffffu, valid)) {
        // no row of this warp's
      } else if (whole) {
        // four lanes write 64 bytes of one row at a time: one row per lane would be 32 lines per store
        const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;  // (a NaN sum is not zero: it goes out)
        uint16_t* row[4];
        bool live[4];
        const unsigned long long mine = reinterpret_cast<unsigned long long>(
            a.out + (it.s.t0 + i) * a.o_ts + (it.head * a.group + hg) * a.o_hs + 256 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          row[j] = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, mine, (lane & 28) + j)) + 8 * (lane & 3);
          live[j] = __shfl_sync(0xffffffffu, static_cast<int>(valid), (lane & 28) + j) != 0;
        }
#pragma unroll 1
        for (int c = 0; c < 256; c += 64) {
          float o[2][32];
          pa_ld32(tbase + lanes + c, o[0]);
          pa_ld32(tbase + lanes + c + 32, o[1]);
          pa_ld_wait();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = pa_bf16x2(o[h][2 * j] * inv, o[h][2 * j + 1] * inv);
            pa_quad_transpose(x, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (live[j])
                *reinterpret_cast<uint4*>(row[j] + c + 32 * h) =
                    make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
          }
        }
      } else {
        float* part = a.part + (((static_cast<size_t>(range) * kHalves + half) * 2 + cta) * 2 + (it.begin == 0 ? 1 : 0)) *
                                   kPaPartFloats;
#pragma unroll 1
        for (int c = 0; c < 256; c += 64) {
          float o[2][32];
          pa_ld32(tbase + lanes + c, o[0]);
          pa_ld32(tbase + lanes + c + 32, o[1]);
          pa_ld_wait();
          if (valid) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<float4*>(part + ((c + 32 * h + j) / 4 * 128 + r) * 4) =
                    make_float4(o[h][j], o[h][j + 1], o[h][j + 2], o[h][j + 3]);
          }
        }
        *reinterpret_cast<float2*>(part + 128 * 256 + 2 * r) = ml;
      }
      pa_fence_before();
      __syncwarp();
      if (lane == 0) pa_arrive_relaxed(o_free);
    }
    if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
    if (r == 0 && cta == 0 && half == 0) a.tail[range] = ok ? tail : PaTail{-1, 0, 0, 0};
  } else if (warp == 8 || warp == 10) {
    // -------------------------------------------------------------- K copies (8), V copies (10)
    // A K stage is 4 blocks of 64 dims x 64 rows, a V stage 2 halves of 64 rows x 2 blocks.  Where
    // a page holds 64 rows in one piece, a box is all of a K stage or of a half; else a box is
    // 2^log_box rows of one block.  A lane copies one box.  The lanes meet at every wait: those that
    // have no box hold no stage back, and a parity tells only two neighbouring phases apart, so that
    // a lane which lags or runs ahead by one more would wait for the wrong one.
    const bool is_k = warp == 8;
    PaRing at(is_k ? 0 : kK, is_k ? kK : kV);
    uint32_t edges = 0;  // V tiles that warp 11 finishes
    const uint64_t map = reinterpret_cast<uint64_t>(is_k ? &kmap : &vmap);
    const int box = 1 << a.log_box, rows = is_k ? 64 : kPaKeys;
    const int blocks = a.log_box == 6 ? 1 : (is_k ? 4 : 2);  // boxes side by side
    const int slab = lane & (blocks - 1), in_stage = lane / blocks * box;
    const uint32_t rows_bytes = (is_k ? 512u : 256u) * box;  // of a box of rows over all blocks
    const uint32_t full0 = pa_map_to(smem_u32(&sm.full[0]), 0), edge_full = smem_u32(&sm.edge_full);
    const uint32_t dst0 = smem_u32(&sm.ring[0][0]) + slab * 8192u +
                          (is_k ? in_stage * 128u : (in_stage >> 6) * 16384u + (in_stage & 63) * 128u);
    bool ok = true, bad_page = false;
    // the stage's `rows` rows from row0 on: this lane's box (row -1: not copied), its page, not
    // looked at before the box is copied, and the bytes of all boxes
    struct Box {
      int page, row;
      uint32_t bytes;
    };
    auto box_of = [&](int row0) {
      const int low = it.low(), row = row0 + in_stage;
      Box x = {0, -1, 0};
      const int from = max(low - row0, 0) >> a.log_box, to = (min(it.s.kv - row0, rows) + box - 1) >> a.log_box;
      x.bytes = max(to - from, 0) * rows_bytes;
      if (in_stage < rows && row < it.s.kv && row + box > low) {
        const int j = a.by_page.div(row);
        x.page = b.tables[it.seq * b.table_stride + j];
        x.row = row - j * b.page_rows;
      }
      return x;
    };
    auto free_stage = [&]() {  // waits until the stage at `at` may be filled
      if (ok && at.passed >= static_cast<uint32_t>(at.n))
        ok = pa_wait_warp(&sm.empty[at.stage], at.parity ^ 1u, abort, budget);
      return ok;
    };
    auto fill = [&](Box& x, int dim_block, uint32_t bar) {
      if (x.row >= 0) {
        if (x.page < 0 || x.page >= b.n_pages) {
          bad_page = true;
          x.page = b.n_pages;  // out of the map's bounds: zeros
        }
        pa_tma(dst0 + at.stage * static_cast<uint32_t>(kPaStage), map, x.row, dim_block + slab, it.head, x.page, bar);
      }
      at.next();
    };
    const int v_block = 4 * half + 2 * cta;
    while (ok && it.next()) {
      auto first_row = [&](int u) { return (it.kt0 + u) * kPaKeys + (is_k ? 64 * cta : 0); };
      Box next = box_of(first_row(it.begin));
      for (int u = it.begin; u < it.end && ok; ++u) {
        Box now = next;  // the next tile's table entries are fetched while this one's stages become free
        if (u + 1 < it.end) next = box_of(first_row(u + 1));
        if (is_k) {
#pragma unroll
          for (int ch = 0; ch < kChunks; ++ch)
            if (free_stage()) {
              const uint32_t bar = full0 + 8u * at.stage;
              if (lane == 0) pa_expect_cluster(bar, now.bytes);
              fill(now, 4 * ch, bar);
            }
        } else if (!it.edge(it.kt0 + u)) {
          if (free_stage()) {
            const uint32_t bar = full0 + 8u * at.stage;
            if (lane == 0) pa_expect_cluster(bar, now.bytes);
            fill(now, v_block, bar);
          }
        } else {
          // the stage reports to warp 11, which zeroes rows of it (with no box to wait for, at
          // once: so only when it is free) and reports to the leader
          if (edges > 0) ok = pa_wait_warp(&sm.edge_done, (edges - 1) & 1, abort, budget);
          ++edges;
          if (free_stage()) {
            if (lane == 0) mbar_arrive_expect_tx(&sm.edge_full, now.bytes);
            fill(now, v_block, edge_full);
          }
        }
      }
    }
    // every stage is free again: no barrier of this CTA has an arrival outstanding when it exits
    for (uint32_t n = at.n, x = at.passed > n ? at.passed - n : 0; x < at.passed && ok; ++x)
      ok = pa_wait_warp(&sm.empty[at.first + x % n], (x / n) & 1, abort, budget);
    if (bad_page) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    if (!ok) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  } else if (warp == 9) {
    // -------------------------------------------------------------- MMA: the leader CTA's
    // The warp stays converged around the elected lane, so that descriptors live in uniform
    // registers: N = 128 MMAs issued by a lone thread took 100-150 cycles instead of 64.
    if (cta == 0) {
      PaRing k_at(0, kK), v_at(kK, kV);
      uint32_t g = 0, items = 0;
      bool ok = true;
      const bool leader = pa_elect();
      const uint64_t q_desc = pa_desc(smem_u32(&sm.q[0][0]), 16, 1024);
      const uint64_t k_desc = pa_desc(smem_u32(&sm.ring[0][0]), 16, 1024);
      const uint64_t v_desc = pa_desc(smem_u32(&sm.ring[0][0]), 8192, 1024);
      auto scores = [&](uint32_t unit) {
        const uint32_t d = tbase + kPaColS + (unit & 1) * 128;
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          ok = pa_wait_warp(&sm.full[k_at.stage], k_at.parity, abort, budget);
          if (!ok) return;
          pa_fence_after();
          const uint64_t kd = k_desc + k_at.stage * static_cast<uint32_t>(kPaStage / 16);
          if (leader) {
#pragma unroll
            for (int k = 0; k < 16; ++k)
              pa_mma_ss(d, q_desc + ((4 * ch + (k >> 2)) * 16384 + 32 * (k & 3)) / 16,
                        kd + ((k >> 2) * 8192 + 32 * (k & 3)) / 16, kPaIdescS, (ch | k) ? 1u : 0u);
            pa_commit(&sm.empty[k_at.stage]);
            if (ch == kChunks - 1) pa_commit(&sm.s_full[unit & 1]);
          }
          __syncwarp();
          k_at.next();
        }
      };
      while (ok && it.next()) {
        ok = __all_sync(0xffffffffu, pa_wait<true>(&sm.q_full, items & 1, abort, budget));
        ++items;
        for (int u = it.begin - 1; u < it.end && ok; ++u) {
          if (u + 1 < it.end) {
            scores(g + (u + 1 - it.begin));
            if (!ok) break;
            if (a.q_tma && u + 2 == it.end && leader) pa_commit(&sm.q_empty);
            __syncwarp();
          }
          if (u < it.begin) continue;
          const uint32_t unit = g + (u - it.begin);
          const uint32_t p = tbase + kPaColS + (unit & 1) * 128;
          ok = pa_wait_warp(&sm.p_full, unit & 1, abort, budget);
          if (ok && u == it.begin && items > 1) ok = pa_wait_warp(&sm.o_free, (items - 2) & 1, abort, budget);
          const bool edge = it.edge(it.kt0 + u);
          if (ok)
            ok = edge ? __all_sync(0xffffffffu, pa_wait<true>(&sm.full[v_at.stage], v_at.parity, abort, budget))
                      : pa_wait_warp(&sm.full[v_at.stage], v_at.parity, abort, budget);
          if (!ok) break;
          pa_fence_after();
          const uint64_t vd = v_desc + v_at.stage * static_cast<uint32_t>(kPaStage / 16);
          const uint32_t more = u > it.begin ? 1u : 0u;
          if (leader) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              pa_mma_ts(tbase, p + 8 * k, vd + ((k >> 2) * 16384 + 2048 * (k & 3)) / 16, kPaIdescO, k ? 1u : more);
            pa_commit(&sm.empty[v_at.stage]);
            pa_commit(&sm.pv_done);
            if (u + 1 == it.end) pa_commit(&sm.o_full);
          }
          __syncwarp();
          v_at.next();
        }
        g += it.end - it.begin;
      }
      if (ok && items > 0) ok = pa_wait_warp(&sm.o_free, (items - 1) & 1, abort, budget);
      if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
    }
  } else {
    // -------------------------------------------------------------- Q copies; V tiles at the ends
    PaRing at(kK, kV);
    uint32_t items = 0, edges = 0;
    bool ok = true;
    const uint64_t map = reinterpret_cast<uint64_t>(&qmap);
    const uint32_t q_full = pa_map_to(smem_u32(&sm.q_full), 0), full0 = pa_map_to(smem_u32(&sm.full[0]), 0);
    while (ok && it.next()) {
      // (the softmax warps copy Q behind their own waits, and nothing would then keep this one within
      // a phase of q_empty)
      if (a.q_tma && items > 0) ok = pa_wait_warp(&sm.q_empty, (items - 1) & 1, abort, budget);
      ++items;
      if (!ok) break;
      if (a.q_tma && lane == 0) {
        pa_expect_cluster(q_full, 128 * D * 2);
        const int token = it.s.t0 + a.by_group.div(it.tile * kPaRows + cta * 128);
#pragma unroll
        for (int blk = 0; blk < D / 64; blk += 4)
          pa_tma(smem_u32(&sm.q[blk][0]), map, 0, token, blk, it.head, q_full);
      }
      __syncwarp();
      for (int u = it.begin; u < it.end && ok; ++u) {
        const int stage = at.stage;
        at.next();
        if (!it.edge(it.kt0 + u)) continue;
        ok = pa_wait_warp(&sm.edge_full, edges & 1, abort, budget);
        ++edges;
        if (!ok) break;
        // rows outside [low, kv) of the tile's 128: this CTA's 128 columns are 16 chunks a row
        const int row0 = (it.kt0 + u) * kPaKeys;
        const int front = min(max(it.low() - row0, 0), kPaKeys), back = min(max(it.s.kv - row0, 0), kPaKeys);
        const int n = front + kPaKeys - back;
        for (int x = lane; x < 16 * n; x += 32) {
          const int k = x >> 4, ch = x & 15, r = k < front ? k : back + k - front;
          *reinterpret_cast<uint4*>(&sm.ring[stage][(r >> 6) * 16384 + (ch >> 3) * 8192 + pa_swizzle(r & 63, ch)]) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          pa_arrive_cluster(full0 + 8u * stage);
          mbar_arrive(&sm.edge_done);
        }
      }
    }
    if (ok && a.q_tma && items > 0) ok = pa_wait_warp(&sm.q_empty, (items - 1) & 1, abort, budget);
    if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  }
  __syncthreads();
  if (sm.abort != 0) {  // gave up somewhere: let the copies in flight land (bounded)
    const uint64_t end = global_ns() + 1000000;
    while (global_ns() < end) __nanosleep(1000);
  }
  // Both CTAs are done with both tensor memories.  Every arrival from the other CTA has been
  // waited for, so nothing but this order is asked of the barrier: a release would wait for
  // the output stores in flight.
  pa_fence_before();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  pa_fence_after();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(512u));
}

// Joins the parts of the items that cross range ends: with M the largest of the parts' reference
// maxima, o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in range order.  A block has 32 rows
// (lanes: the parts hold a column quad's rows side by side) and 64 columns of one half; each of
// its 8 warps takes 8 columns, and the results leave through shared memory, 128 bytes a row.
constexpr int kPaJoinThreads = 256, kPaJoinRows = 32;
template <int D>
__global__ void __launch_bounds__(kPaJoinThreads) paged_join_kernel(const __grid_constant__ PaArgs a,
                                                                    const __grid_constant__ PagedBatch b) {
  constexpr int kHalves = D / 256;
  __shared__ uint4 tile[kPaJoinRows][9];  // (9: the rows of a 16-byte column fall into different banks)
  pdl_wait();
  pdl_launch_dependents();
  const PaTail t = a.tail[blockIdx.x];
  if (t.seq < 0) return;
  bool bad;
  const PagedSeq s = paged_seq(b, t.seq, &bad);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int half = blockIdx.z % kHalves, col0 = blockIdx.z / kHalves * 64;
  const int row0 = blockIdx.y * kPaJoinRows, cta = row0 >> 7, row = (row0 & 127) + lane;
  if (a.by_group.div(t.tile * kPaRows + row0) >= s.n) return;  // (of all rows)
  // the first part is its range's second slot, the others their first
  const float* first = a.part + (((static_cast<size_t>(blockIdx.x) * kHalves + half) * 2 + cta) * 2 + 1) * kPaPartFloats;
  const size_t step = static_cast<size_t>(kHalves) * 4 * kPaPartFloats;
  constexpr int kBatch = 4;
  float top = -CUDART_INF_F, l = 0.f, o[2][4] = {};
  for (int k0 = 0; k0 < t.parts; k0 += kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch][2];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      ml[k] = make_float2(-CUDART_INF_F, 0.f);
      v[k][0] = v[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k < t.parts) {
        const float* p = k0 + k == 0 ? first : first - kPaPartFloats + (k0 + k) * step;
        ml[k] = *reinterpret_cast<const float2*>(p + 128 * 256 + 2 * row);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          v[k][h] = *reinterpret_cast<const float4*>(p + ((col0 / 4 + 2 * warp + h) * 128 + row) * 4);
      }
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) now = fmaxf(now, ml[k].x);
    const float ref = now == -CUDART_INF_F ? 0.f : now, w0 = pa_exp2(top - ref);
    top = now;
    l *= w0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[h][j] *= w0;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w = pa_exp2(ml[k].x - ref);
      l = fmaf(w, ml[k].y, l);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[h][0] = fmaf(w, v[k][h].x, o[h][0]);
        o[h][1] = fmaf(w, v[k][h].y, o[h][1]);
        o[h][2] = fmaf(w, v[k][h].z, o[h][2]);
        o[h][3] = fmaf(w, v[k][h].w, o[h][3]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  tile[lane][warp] = make_uint4(pa_bf16x2(o[0][0] * inv, o[0][1] * inv), pa_bf16x2(o[0][2] * inv, o[0][3] * inv),
                                pa_bf16x2(o[1][0] * inv, o[1][1] * inv), pa_bf16x2(o[1][2] * inv, o[1][3] * inv));
  __syncthreads();
  const int r = threadIdx.x / 8, c = threadIdx.x % 8;
  const int rr = t.tile * kPaRows + row0 + r;
  const int i = a.by_group.div(rr), hg = rr - i * a.group;
  if (i >= s.n) return;
  *reinterpret_cast<uint4*>(a.out + (s.t0 + i) * a.o_ts + (t.head * a.group + hg) * a.o_hs + 256 * half + col0 + 8 * c) =
      tile[r][c];
}

// ---------------------------------------------------------------------------- host
g4_status paged_scratch(g4_ctx* ctx, PaArgs& a) {
  if (ctx->paged.part == nullptr) {
    // a pair's four partials outweigh what two CTAs of the other kernel leave
    const size_t part = static_cast<size_t>(ctx->sm_count / 2) * 4 * kPaPartFloats * sizeof(float);
    g4_status st = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice");
    if (st == G4_OK && ctx->paged.tail == nullptr)
      st = check_cuda(ctx, cudaMalloc(&ctx->paged.tail, ctx->sm_count * sizeof(PaTail)), "cudaMalloc paged tails");
    if (st == G4_OK) st = check_cuda(ctx, cudaMalloc(&ctx->paged.part, part), "cudaMalloc paged partials");
    if (st != G4_OK) return st;
  }
  a.part = ctx->paged.part;
  a.tail = static_cast<PaTail*>(ctx->paged.tail);
  return G4_OK;
}

template <int D>
static g4_status launch_attention(g4_ctx* ctx, PaArgs a, PagedBatch b, const g4_paged_cache* c) {
  const void* fn = (const void*)paged_attn_kernel<D>;
  const size_t smem = sizeof(PaSmem<D>);
  g4_status st = allow_max_dynamic_smem(ctx, fn, smem, "paged attention");
  if (st != G4_OK) return st;
  int& pairs = ctx->paged.pairs[D == 256 ? 0 : 1];
  if (pairs == 0) {  // CTA pairs the device runs at once: a range too many would run alone at the end
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctx->sm_count / 2 * 2);
    cfg.blockDim = dim3(kPaThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    st = check_cuda(ctx, cudaOccupancyMaxActiveClusters(&n, fn, &cfg), "paged attention: active clusters");
    if (st != G4_OK) return st;
    n = n < ctx->sm_count / 2 ? n : ctx->sm_count / 2;
    if (n < 2) return fail(ctx, G4_ERR_UNSUPPORTED, "paged attention: CTA pairs do not fit this device");
    pairs = n;
  }
  a.tile_rows = kPaRows;
  a.item_cost = kPaItemCost;
  long long items, keys;
  paged_bounds(b, a, items, keys);
  if (items * (keys + kPaItemCost) >= (1ll << 30))
    return fail(ctx, G4_ERR_TOO_LARGE, "paged attention: more than 2^30 tiles in one call");
  a.ranges = pairs / (D / 256);
  if (items * keys < a.ranges) a.ranges = static_cast<int>(items * keys);  // no more than there can be units
  const int low = b.page_rows & -b.page_rows;  // the largest power of two that divides a page's rows
  a.log_box = 0;
  while ((1 << a.log_box) < low && a.log_box < 6) ++a.log_box;
  // pages: rows, 64-dim blocks, heads, pages; a box is 2^log_box rows of one block, or 64 rows of
  // a K stage's four or a V stage's two
  CUtensorMap km, vm, qm;
  const int dims[4] = {c->page_rows, D / 64, c->n_kv_heads, c->n_pages};
  const int whole = a.log_box == 6;
  const int kbox[4] = {1 << a.log_box, whole ? 4 : 1, 1, 1}, vbox[4] = {1 << a.log_box, whole ? 2 : 1, 1, 1};
  if (!tile_map(&km, c->k, dims, {c->k_row_stride, 64, c->k_head_stride, c->k_page_stride}, kbox) ||
      !tile_map(&vm, c->v, dims, {c->v_row_stride, 64, c->v_head_stride, c->v_page_stride}, vbox))
    return fail(ctx, G4_ERR_UNSUPPORTED, "paged attention: the cache's layout has no TMA descriptor");
  // Q: heads of a group, tokens, blocks, KV heads; a box is a CTA's 128 rows of four blocks
  const int qdims[4] = {a.group, b.n_tokens, D / 64, a.n_kv};
  const int64_t qstr[4] = {a.q_hs, a.q_ts, 64, a.q_hs * a.group};
  a.q_tma = 0;
  if (128 % a.group == 0 && (a.q_hs > 0 || a.group * a.n_kv == 1) && (a.q_ts > 0 || b.n_tokens == 1)) {
    const int qbox[4] = {a.group, 128 / a.group, 4, 1};
    a.q_tma = tile_map(&qm, a.q, qdims, qstr, qbox) ? 1 : 0;
  }
  if (!a.q_tma) qm = km;  // (not used)
  Scratch* scr = ctx->buf.scratch;
  uint64_t budget = ctx->wait_budget_ns;
  void* args[] = {(void*)&km, (void*)&vm, (void*)&qm, (void*)&a, (void*)&b, (void*)&scr, (void*)&budget};
  st = launch_kernel(ctx, fn, dim3(a.ranges * (D / 256) * 2), dim3(kPaThreads), smem, args, false, "paged attention");
  if (st != G4_OK) return st;
  void* jargs[] = {(void*)&a, (void*)&b};
  const long long rows = static_cast<long long>(b.n_tokens) * a.group;
  const int row_blocks = static_cast<int>(((rows < kPaRows ? rows : kPaRows) + kPaJoinRows - 1) / kPaJoinRows);
  return launch_kernel(ctx, (const void*)paged_join_kernel<D>, dim3(a.ranges, row_blocks, 4 * (D / 256)),
                       dim3(kPaJoinThreads), 0, jargs, false, "paged attention join");
}

}  // namespace g4

using namespace g4;

extern "C" {

g4_status g4_paged_attention(g4_ctx* ctx, const g4_bf16* q, int64_t q_token_stride, int64_t q_head_stride,
                             int n_heads, const g4_paged_cache* cache, const g4_paged_batch* batch, float scale,
                             int window, g4_bf16* out, int64_t out_token_stride, int64_t out_head_stride) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_paged_cache(ctx, cache);
  if (st == G4_OK) st = check_paged_batch(ctx, batch);
  if (st != G4_OK) return st;
  if (n_heads < 1 || n_heads > 4096 || n_heads % cache->n_kv_heads != 0)
    return fail(ctx, G4_ERR_BAD_ARG, "n_heads must be a multiple of n_kv_heads, at most 4096");
  if (window < 0) return fail(ctx, G4_ERR_BAD_ARG, "negative window");
  if (!std::isfinite(scale * kPaLog2e)) return fail(ctx, G4_ERR_BAD_ARG, "scale is not finite, or too large for f32");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return G4_OK;
  if (static_cast<long long>(batch->n_tokens) * (n_heads / cache->n_kv_heads) > (1 << 30))
    return fail(ctx, G4_ERR_BAD_ARG, "too many tokens times query heads per KV head for one call");
  if ((st = check_rows(ctx, q, q_token_stride, q_head_stride, "q")) != G4_OK) return st;
  if ((st = check_out_rows(ctx, out, out_token_stride, out_head_stride, batch->n_tokens, n_heads, cache->head_dim,
                           "out")) != G4_OK)
    return st;
  PaArgs a = {};
  a.q = q;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.out = out;
  a.o_ts = out_token_stride;
  a.o_hs = out_head_stride;
  a.group = n_heads / cache->n_kv_heads;
  a.n_kv = cache->n_kv_heads;
  a.by_group = divisor(a.group);
  a.by_page = divisor(cache->page_rows);
  a.window = window;
  a.scale = scale * kPaLog2e;
  const PagedBatch b = paged_batch(batch, cache);
  if ((st = paged_scratch(ctx, a)) != G4_OK) return st;
  // Decode steps go to the kernel for few rows: at most 16 rows in all, or as many tokens as
  // sequences, which is taken for one token each (the lengths themselves are on the device; other
  // lengths are right there too, 16 rows at a time).  A step with an idle sequence or a padded token
  // is not seen as one and comes here.  32 single tokens of full layers over up to 8192 rows:
  // 56 us there, 80 us here.  With a chunk among them one launch of this kernel beats
  // one of each (31 tokens beside 509 new ones, sliding: 78 us against 89).
  const bool few = static_cast<long long>(b.n_tokens) * a.group <= kPaFewRows ||
                   (a.group <= kPaFewRows && b.n_tokens == b.n_seqs);
  if (few) return launch_paged_few(ctx, a, b, cache);
  return cache->head_dim == DS ? launch_attention<DS>(ctx, a, b, cache) : launch_attention<DF>(ctx, a, b, cache);
}

}  // extern "C"
