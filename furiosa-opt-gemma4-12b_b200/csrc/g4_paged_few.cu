// Attention of sequences with few rows (new tokens x query heads per KV head: a decode step) over
// their pages, on tcgen05 with the roles of the operands exchanged: the cache rows are the 128 rows
// of the MMA, the query rows its columns (N = 16 for S, 32 for O).
//   S^T[128 keys][16] = K Q^T           O^T[128 dims][32] += V^T P^T   (per 128 dims of the head)
// so a tile of 128 cache rows costs 32 (head of 256) or 64 (512) small MMAs instead of the
// 256-row products of g4_paged_attn.cu, and every K/V byte is fetched once.  Bound by HBM: 192 KB
// of K and V per SM are in flight, in stages of 128 rows x 128 dims (32 KB).
//
// A thread has one key of the tile: maxima over the keys go through shuffles (16 columns at a
// time: 16 exchanges instead of 80) and shared memory, P into the shared tile the second product
// reads, sums stay with the thread until the item ends.  Both operands of a kind::f16 MMA have one
// type, V's bf16, so P goes in as two bf16: its rounding in rows 0-15 of the tile, what that left
// over in rows 16-31, N = 32 columns of O that are added at the end.  A weight is off by 2^-16 of
// itself at most; the tensor cores have the time (32 single tokens of full layers over up to 8192
// rows 56.4 us, 55.6 with P rounded once; one sliding token 10.9 us, 10.7).
// Up to four rows (one token of two heads) take a quarter of that work.  The scores of the next
// tile are computed before the values of this one, so that K keeps arriving meanwhile.
//
// Work split, partial sums and the join are as there, with one CTA per range.  Warps: 0-3
// softmax, Q and output, 4 copies, 5 MMA and tensor memory, 6 zeroes V rows past a sequence's ends.
#include <string>

#include "g4_paged_split.cuh"

namespace g4 {

constexpr int kFewThreads = 224;
constexpr int kFewStage = 32768, kFewStages = 6;
constexpr uint32_t kFewCols = 256;  // tensor memory: S [0, 16) and [16, 32), O block j [32 + 32 j, 64 + 32 j)
constexpr uint32_t kFewColO = 32;   // (of P's rounded part in 16 columns, of its remainder in 16)
constexpr uint32_t kFewIdescS = (1u << 4) | (1u << 7) | (1u << 10) | (2u << 17) | (8u << 24);
constexpr uint32_t kFewIdescO =  // N = 32; A (V) dims-contiguous
    (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (4u << 17) | (8u << 24);
constexpr int kFewPBlock = 32 * 128;  // bytes of P over 64 keys

template <int D>
struct __align__(1024) FewSmem {
  uint8_t ring[kFewStages][kFewStage];  // 2 blocks of 64 dims x [128 rows][64], 128-byte swizzle
  uint8_t q[D / 64][16 * 128];
  uint8_t p[2][kFewPBlock];             // P: blocks of 64 keys x [16 rows, their remainders][64]
  float4 top[2][4][4];                  // the warps' maxima of a tile's 16 columns (two tiles' worth)
  float4 sum[4][4];
  uint64_t full[kFewStages], empty[kFewStages], raw[kFewStages];  // raw: copied, rows not zeroed yet
  uint64_t s_full[2], p_full, pv_done, q_full;
  uint32_t tmem, abort;
  PaRange range;
};
constexpr int few_part_floats(int d) { return 16 * d + 32; }  // O [16][D], then (m, l) [16][2]

__device__ __forceinline__ void few_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void few_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void few_tma(uint32_t dst, uint64_t map, int row, int block, int head, int page,
                                        uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(0), "r"(row), "r"(block), "r"(head), "r"(page), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void few_ld16(uint32_t taddr, float (&v)[16]) {
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
__device__ __forceinline__ void few_st16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"f"(v[0]),
      "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "r"(taddr)
      : "memory");
}
// The four softmax warps agree on whether all of their waits held.
__device__ __forceinline__ bool few_agree(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return r != 0;
}
// Maxima or sums of N (4 or 16) columns over the warp's 32 lanes: while a lane carries more than
// one column, each exchange halves them; lane l ends up with column l / (32 / N).
template <bool kMax, int N>
__device__ __forceinline__ float few_reduce(const float (&v)[16], int lane) {
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = v[i];
#pragma unroll
  for (int n = N / 2, bit = 16; n >= 1; n >>= 1, bit >>= 1) {
    const bool up = (lane & bit) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
      const float got = __shfl_xor_sync(0xffffffffu, give, bit);
      x[i] = kMax ? fmaxf(keep, got) : keep + got;
    }
  }
#pragma unroll
  for (int bit = 16 / N; bit >= 1; bit >>= 1) {
    const float got = __shfl_xor_sync(0xffffffffu, x[0], bit);
    x[0] = kMax ? fmaxf(x[0], got) : x[0] + got;
  }
  return x[0];
}
// The softmax of one tile, for one key (thread) and N columns: P into the shared tile, m and l
// updated.  False when a wait gave up.
template <int D, int N>
__device__ __forceinline__ bool few_tile(FewSmem<D>& sm, const PaArgs& a, const PaWalk& it, int u, uint32_t g, bool good,
                                         uint32_t tbase, float factor_s, bool scale_first, float (&m)[16],
                                         float (&l)[16], uint64_t budget) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t lanes = static_cast<uint32_t>(32 * warp) << 16;
  float s[16];
  pa_fence_after();
  few_ld16(tbase + 16 * (g & 1) + lanes, s);
  if (scale_first) {
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] *= a.scale;
  }
  // the tile's keys are [key0, key0 + 128); the item's tokens are at positions [first, last]
  const int key0 = (it.kt0 + u) * kPaKeys, base = it.s.kv - it.s.n, r0 = it.tile * 16;
  const int first = base + a.by_group.div(r0), last = base + min(it.s.n - 1, a.by_group.div(r0 + 15));
  if (key0 + kPaKeys - 1 > first || (a.window > 0 && last - key0 >= a.window)) {
    const int key = key0 + tid;
#pragma unroll
    for (int c = 0; c < N; ++c) {  // (columns past the rows: whatever they hold stays theirs)
      const int pos = base + a.by_group.div(r0 + c);
      if (key > pos || (a.window > 0 && pos - key >= a.window)) s[c] = -CUDART_INF_F;
    }
  }
  const float mine = few_reduce<true, N>(s, lane) * factor_s;
  if (lane % (32 / N) == 0) reinterpret_cast<float*>(&sm.top[g & 1][warp][0])[lane / (32 / N)] = mine;
  good = good && (g == 0 || pa_wait_warp(&sm.pv_done, (g - 1) & 1, &sm.abort, budget));
  if (!few_agree(good)) return false;
  bool moved = false;
  float f[16];
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    const float4 t0 = sm.top[g & 1][0][q], t1 = sm.top[g & 1][1][q], t2 = sm.top[g & 1][2][q], t3 = sm.top[g & 1][3][q];
    const float top[4] = {fmaxf(fmaxf(t0.x, t1.x), fmaxf(t2.x, t3.x)), fmaxf(fmaxf(t0.y, t1.y), fmaxf(t2.y, t3.y)),
                          fmaxf(fmaxf(t0.z, t1.z), fmaxf(t2.z, t3.z)), fmaxf(fmaxf(t0.w, t1.w), fmaxf(t2.w, t3.w))};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 4 * q + j;
      f[c] = 1.f;
      if (m[c] == -CUDART_INF_F) {
        m[c] = top[j];
      } else if (top[j] > m[c] + kPaLag) {
        f[c] = pa_exp2(m[c] - top[j]);
        l[c] *= f[c];
        m[c] = top[j];
        moved = true;  // (the same in every thread)
      }
    }
  }
  if (moved && u != it.begin) {
    pa_fence_after();  // O is read behind the products that pv_done stood for
#pragma unroll
    for (int c = N; c < 16; ++c) f[c] = 1.f;
#pragma unroll 1
    for (int x = 0; x < D / 128 * 2; ++x) {  // a block's 16 columns, or those of their remainders
      float o[16];
      few_ld16(tbase + lanes + kFewColO + 16 * x, o);
#pragma unroll
      for (int c = 0; c < 16; ++c) o[c] *= f[c];
      few_st16(tbase + lanes + kFewColO + 16 * x, o);
    }
    pa_st_wait();
  }
  uint8_t* p = &sm.p[tid >> 6][0];
  const int ch = (tid & 63) >> 3, eb = (tid & 7) * 2;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const float e = pa_exp2(fmaf(s[c], factor_s, m[c] == -CUDART_INF_F ? 0.f : -m[c]));
    l[c] += e;
    const uint16_t hi = f32_to_bf16(e);
    uint16_t* at = reinterpret_cast<uint16_t*>(p + pa_swizzle(c, ch) + eb);
    at[0] = hi;
    at[16 * 64] = f32_to_bf16(e - bf16_to_f32(hi));  // (16 rows on: the same place in the swizzle)
  }
  return true;
}

template <int D>
__global__ void __launch_bounds__(kFewThreads, 1)
    paged_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                     const __grid_constant__ PaArgs a, const __grid_constant__ PagedBatch b, Scratch* scr,
                     uint64_t budget) {
  using Smem = FewSmem<D>;
  constexpr int kBlocks = D / 128;  // stages of a K tile and of a V tile
  extern __shared__ uint8_t few_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(few_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, range = blockIdx.x;
  if (tid == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
      mbar_init(&sm.raw[i], 1);
    }
    mbar_init(&sm.s_full[0], 1);
    mbar_init(&sm.s_full[1], 1);
    mbar_init(&sm.p_full, 4);
    mbar_init(&sm.pv_done, 1);
    mbar_init(&sm.q_full, 4);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                 "r"(kFewCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  pdl_wait();
  pdl_launch_dependents();
  PaCount* w = reinterpret_cast<PaCount*>(&sm.ring[0][0]);  // (the ring is not in use yet)
  static_assert(G4_PAGED_MAX_SEQS * sizeof(PaCount) <= kFewStages * kFewStage, "unit counts fit the ring");
  pa_count(b, a, w, scr, blockIdx.x == 0);
  __syncthreads();
  if (warp == 0) {
    const PaRange found = pa_range(b, a, w, range, lane, scr);
    if (lane == 0) sm.range = found;
    fence_proxy_async();  // the ring's next writers are TMA copies
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  const uint32_t tbase = sm.tmem;
  const int u_first = sm.range.first;
  const int u_end = range < sm.range.count ? pa_share(range + 1, sm.range.units, sm.range.count) : u_first;
  volatile uint32_t* abort = &sm.abort;
  PaWalk it(b, a, sm.range, u_end - u_first);

  if (warp < 4) {
    // -------------------------------------------------------------- Q, softmax, output
    const uint32_t lanes = static_cast<uint32_t>(32 * warp) << 16;
    const bool scale_first = !(a.scale > 0.f);
    const float factor_s = scale_first ? 1.f : a.scale;
    uint32_t g = 0;  // unit of the range
    PaTail tail = {-1, 0, 0, 0};
    bool ok = true;
    while (ok && it.next()) {
      const int rows = it.s.n * a.group - it.tile * 16;  // valid rows (columns here), from 0
      // Q: the previous item's products are done, their last tile has been read
      for (int x = tid; x < 16 * (D / 8); x += 128) {
        const int row = x / (D / 8), ch = x % (D / 8);
        const int rr = it.tile * 16 + row, i = a.by_group.div(rr);
        const bool in = row < rows;
        const uint16_t* src = in ? a.q + (it.s.t0 + i) * a.q_ts + (it.head * a.group + rr - i * a.group) * a.q_hs + 8 * ch
                                 : a.q;
        cp_async16(smem_u32(&sm.q[ch >> 3][pa_swizzle(row, ch)]), src, in ? 16u : 0u);
      }
      cp_async_wait_all();
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
      float m[16], l[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) m[c] = -CUDART_INF_F, l[c] = 0.f;
      for (int u = it.begin; u < it.end; ++u, ++g) {
        const bool good = pa_wait_warp(&sm.s_full[g & 1], (g >> 1) & 1, abort, budget);
        ok = rows <= 4 ? few_tile<D, 4>(sm, a, it, u, g, good, tbase, factor_s, scale_first, m, l, budget)
                       : few_tile<D, 16>(sm, a, it, u, g, good, tbase, factor_s, scale_first, m, l, budget);
        if (!ok) break;
        fence_proxy_async();
        pa_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full);
      }
      if (!ok) break;
      bool good = pa_wait_warp(&sm.pv_done, (g - 1) & 1, abort, budget);
      const float part_sum = few_reduce<false, 16>(l, lane);
      if ((lane & 1) == 0) reinterpret_cast<float*>(&sm.sum[warp][0])[lane >> 1] = part_sum;
      ok = few_agree(good);
      if (!ok) break;
      pa_fence_after();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 t0 = sm.sum[0][q], t1 = sm.sum[1][q], t2 = sm.sum[2][q], t3 = sm.sum[3][q];
        l[4 * q] = (t0.x + t1.x) + (t2.x + t3.x);
        l[4 * q + 1] = (t0.y + t1.y) + (t2.y + t3.y);
        l[4 * q + 2] = (t0.z + t1.z) + (t2.z + t3.z);
        l[4 * q + 3] = (t0.w + t1.w) + (t2.w + t3.w);
      }
      const bool whole = it.begin == 0 && it.end == it.nk;
      if (it.begin == 0 && it.end < it.nk) {
        const int last = u_end - it.end + it.nk - 1;  // the item's last unit, as a position of the call
        const long long e = ((last + 1ll) * sm.range.count - 1) / sm.range.units;
        tail = {it.seq, it.tile, it.head, static_cast<int>(e) - range + 1};
      }
      float* part = a.part + (static_cast<size_t>(range) * 2 + (it.begin == 0 ? 1 : 0)) * few_part_floats(D);
#pragma unroll 1
      for (int blk = 0; blk < kBlocks; ++blk) {
        float o[16], o_rest[16];
        few_ld16(tbase + lanes + kFewColO + 32 * blk, o);
        few_ld16(tbase + lanes + kFewColO + 32 * blk + 16, o_rest);
#pragma unroll
        for (int c = 0; c < 16; ++c) o[c] += o_rest[c];
        if (whole) {
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            if (c >= rows) continue;
            const int rr = it.tile * 16 + c, i = a.by_group.div(rr);
            a.out[(it.s.t0 + i) * a.o_ts + (it.head * a.group + rr - i * a.group) * a.o_hs + 128 * blk + tid] =
                f32_to_bf16(l[c] == 0.f ? 0.f : __fdividef(o[c], l[c]));  // (a NaN sum is not zero: it goes out)
          }
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c)
            if (c < rows) part[c * D + 128 * blk + tid] = o[c];
        }
      }
      if (!whole && tid < 16) {
        float mc = m[0], lc = l[0];
#pragma unroll
        for (int c = 1; c < 16; ++c) {
          mc = tid == c ? m[c] : mc;
          lc = tid == c ? l[c] : lc;
        }
        *reinterpret_cast<float2*>(part + 16 * D + 2 * tid) = make_float2(mc, lc);
      }
      // (sum is written again only past the next tile's agreement; O only after its P)
    }
    pa_fence_before();
    if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
    if (tid == 0) a.tail[range] = ok ? tail : PaTail{-1, 0, 0, 0};
  } else if (warp == 4) {
    // -------------------------------------------------------------- copies
    // A box is 2^log_box rows of one 64-dim block, or all of a stage; a lane copies one.  The lanes
    // meet at every wait: one without a box would hold no stage back, and could lag behind, or run
    // ahead of, the two phases that a parity tells apart.
    PaRing at(0, kFewStages);
    const uint64_t maps[2] = {reinterpret_cast<uint64_t>(&kmap), reinterpret_cast<uint64_t>(&vmap)};
    const int box = 1 << a.log_box, blocks = a.log_box == 7 ? 1 : 2;
    const int slab = lane & (blocks - 1), in_stage = lane / blocks * box;
    const uint32_t dst0 = smem_u32(&sm.ring[0][0]) + slab * 16384u + in_stage * 128u;
    bool ok = true, bad_page = false;
    struct Box {
      int page, row;
      uint32_t bytes;
    };
    auto box_of = [&](int row0) {
      const int low = it.low(), row = row0 + in_stage;
      Box x = {0, -1, 0};
      const int from = max(low - row0, 0) >> a.log_box, to = (min(it.s.kv - row0, kPaKeys) + box - 1) >> a.log_box;
      x.bytes = max(to - from, 0) * (box * 256u);
      if (in_stage < kPaKeys && row < it.s.kv && row + box > low) {
        const int j = a.by_page.div(row);
        x.page = b.tables[it.seq * b.table_stride + j];
        x.row = row - j * b.page_rows;
      }
      return x;
    };
    auto copy = [&](const Box& x, bool is_v, bool edge) {  // a tile's kBlocks stages
#pragma unroll 1
      for (int blk = 0; blk < kBlocks && ok; ++blk) {
        if (at.passed >= kFewStages) ok = pa_wait_warp(&sm.empty[at.stage], at.parity ^ 1u, abort, budget);
        if (!ok) break;
        uint64_t* bar = edge ? &sm.raw[at.stage] : &sm.full[at.stage];
        if (lane == 0) mbar_arrive_expect_tx(bar, x.bytes);
        if (x.row >= 0) {
          int page = x.page;
          if (page < 0 || page >= b.n_pages) {
            bad_page = true;
            page = b.n_pages;  // out of the map's bounds: zeros
          }
          few_tma(dst0 + at.stage * static_cast<uint32_t>(kFewStage), maps[is_v ? 1 : 0], x.row, 2 * blk + slab,
                  it.head, page, smem_u32(bar));
        }
        at.next();
      }
    };
    while (ok && it.next()) {
      Box next = box_of((it.kt0 + it.begin) * kPaKeys), now = next;
      for (int u = it.begin - 1; u < it.end && ok; ++u) {  // K of u + 1, then V of u
        const Box v = now;
        now = next;
        if (u + 2 < it.end) next = box_of((it.kt0 + u + 2) * kPaKeys);
        if (u + 1 < it.end) copy(now, false, false);
        if (u >= it.begin) copy(v, true, it.edge(it.kt0 + u));
      }
    }
    // every stage is free again: no copy or arrival is outstanding when the CTA exits
    for (uint32_t x = at.passed > kFewStages ? at.passed - kFewStages : 0; x < at.passed && ok; ++x)
      ok = pa_wait_warp(&sm.empty[x % kFewStages], (x / kFewStages) & 1, abort, budget);
    if (bad_page) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    if (!ok) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  } else if (warp == 5) {
    // -------------------------------------------------------------- MMA
    PaRing at(0, kFewStages);
    uint32_t g = 0, items = 0;
    bool ok = true;
    const bool leader = pa_elect();
    const uint64_t q_desc = pa_desc(smem_u32(&sm.q[0][0]), 16, 1024), p_desc = pa_desc(smem_u32(&sm.p[0][0]), 16, 1024);
    const uint64_t k_desc = pa_desc(smem_u32(&sm.ring[0][0]), 16, 1024);
    const uint64_t v_desc = pa_desc(smem_u32(&sm.ring[0][0]), 16384, 1024);
    while (ok && it.next()) {
      ok = pa_wait_warp(&sm.q_full, items & 1, abort, budget);
      ++items;
      for (int u = it.begin - 1; u < it.end && ok; ++u) {
        if (u + 1 < it.end) {
          const uint32_t unit = g + (u + 1 - it.begin);
#pragma unroll
          for (int x = 0; x < kBlocks; ++x) {
            ok = ok && pa_wait_warp(&sm.full[at.stage], at.parity, abort, budget);
            if (!ok) break;
            pa_fence_after();
            const uint64_t kd = k_desc + at.stage * static_cast<uint32_t>(kFewStage / 16);
            if (leader) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                few_mma(tbase + 16 * (unit & 1), kd + ((k >> 2) * 16384 + 32 * (k & 3)) / 16,
                        q_desc + ((2 * x + (k >> 2)) * 2048 + 32 * (k & 3)) / 16, kFewIdescS, (x | k) ? 1u : 0u);
              few_commit(&sm.empty[at.stage]);
              if (x == kBlocks - 1) few_commit(&sm.s_full[unit & 1]);
            }
            __syncwarp();
            at.next();
          }
        }
        if (u < it.begin) continue;
        ok = ok && pa_wait_warp(&sm.p_full, (g + (u - it.begin)) & 1, abort, budget);
        const uint32_t more = u > it.begin ? 1u : 0u;
#pragma unroll
        for (int x = 0; x < kBlocks; ++x) {
          ok = ok && pa_wait_warp(&sm.full[at.stage], at.parity, abort, budget);
          if (!ok) break;
          pa_fence_after();
          const uint64_t vd = v_desc + at.stage * static_cast<uint32_t>(kFewStage / 16);
          if (leader) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              few_mma(tbase + kFewColO + 32 * x, vd + 2048 * k / 16,
                      p_desc + ((k >> 2) * kFewPBlock + 32 * (k & 3)) / 16, kFewIdescO, k ? 1u : more);
            few_commit(&sm.empty[at.stage]);
            if (x == kBlocks - 1) few_commit(&sm.pv_done);
          }
          __syncwarp();
          at.next();
        }
      }
      g += it.end - it.begin;
    }
    if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  } else {
    // -------------------------------------------------------------- V rows past the ends
    PaRing at(0, kFewStages);
    uint32_t parity = 0;  // of each stage's `raw`
    bool ok = true;
    while (ok && it.next()) {
      for (int x = 0; x < kBlocks; ++x) at.next();  // K of the first tile
      for (int u = it.begin; u < it.end && ok; ++u) {
        if (u + 1 < it.end)
          for (int x = 0; x < kBlocks; ++x) at.next();
        const int row0 = (it.kt0 + u) * kPaKeys;
        const int front = min(max(it.low() - row0, 0), kPaKeys), back = min(max(it.s.kv - row0, 0), kPaKeys);
        const int n = front + kPaKeys - back;  // rows outside [low, kv)
        for (int x = 0; x < kBlocks; ++x, at.next()) {
          if (!it.edge(it.kt0 + u)) continue;
          ok = ok && pa_wait_warp(&sm.raw[at.stage], (parity >> at.stage) & 1u, abort, budget);
          if (!ok) continue;
          parity ^= 1u << at.stage;
          for (int y = lane; y < 16 * n; y += 32) {
            const int k = y >> 4, ch = y & 15, r = k < front ? k : back + k - front;
            *reinterpret_cast<uint4*>(&sm.ring[at.stage][(ch >> 3) * 16384 + pa_swizzle(r, ch)]) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.full[at.stage]);
        }
      }
    }
    if (!ok && lane == 0) atomicOr(&scr->status, DEV_ERR_TIMEOUT_MBAR);
  }
  __syncthreads();
  if (sm.abort != 0) {  // gave up somewhere: let the copies in flight land (bounded)
    const uint64_t end = global_ns() + 1000000;
    while (global_ns() < end) __nanosleep(1000);
  }
  pa_fence_after();
  if (warp == 5)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(kFewCols));
}

// Joins an item's parts as paged_join_kernel does; a block has one row: D / 4 threads a part,
// kGroups parts at a time, joined in range order within a group and the groups in order.
// kThreads: 512 where one item may be in all CTAs' hands (one token over 8192 rows of a full layer:
// 18.0 us in all, 20.1 with 256), 256 where most have two parts (32 tokens: 56.5 us, 58.5 with 512;
// both before P went in as two bf16).
template <int D, int kThreads>
__global__ void __launch_bounds__(kThreads) paged_few_join_kernel(const __grid_constant__ PaArgs a,
                                                                         const __grid_constant__ PagedBatch b) {
  constexpr int kGroups = kThreads / (D / 4), kBatch = 4;
  __shared__ float4 acc[kGroups][D / 4];
  __shared__ float2 stat[kGroups];
  pdl_wait();
  pdl_launch_dependents();
  const PaTail t = a.tail[blockIdx.x];
  if (t.seq < 0) return;
  bool bad;
  const PagedSeq s = paged_seq(b, t.seq, &bad);
  const int group = threadIdx.x / (D / 4), quad = threadIdx.x % (D / 4);
  const int row = blockIdx.y, rr = t.tile * 16 + row;
  const int i = a.by_group.div(rr), hg = rr - i * a.group;
  if (i >= s.n) return;
  const int per = (t.parts + kGroups - 1) / kGroups, from = group * per, k1 = min(t.parts, from + per);
  const float* base = a.part + static_cast<size_t>(blockIdx.x) * 2 * few_part_floats(D);
  float top = -CUDART_INF_F, l = 0.f, o[4] = {};
  for (int k0 = from; k0 < k1; k0 += kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      ml[k] = make_float2(-CUDART_INF_F, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k < k1) {  // the first part is its range's second slot, the others their first
        const float* p = base + (k0 + k == 0 ? 1 : 2 * (k0 + k)) * few_part_floats(D);
        ml[k] = *reinterpret_cast<const float2*>(p + 16 * D + 2 * row);
        v[k] = *reinterpret_cast<const float4*>(p + row * D + 4 * quad);
      }
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) now = fmaxf(now, ml[k].x);
    const float ref = now == -CUDART_INF_F ? 0.f : now, w0 = pa_exp2(top - ref);
    top = now;
    l *= w0;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= w0;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w = pa_exp2(ml[k].x - ref);
      l = fmaf(w, ml[k].y, l);
      o[0] = fmaf(w, v[k].x, o[0]);
      o[1] = fmaf(w, v[k].y, o[1]);
      o[2] = fmaf(w, v[k].z, o[2]);
      o[3] = fmaf(w, v[k].w, o[3]);
    }
  }
  acc[group][quad] = make_float4(o[0], o[1], o[2], o[3]);
  if (quad == 0) stat[group] = make_float2(top, l);
  __syncthreads();
  if (group != 0) return;
  float all = -CUDART_INF_F;
#pragma unroll
  for (int k = 0; k < kGroups; ++k) all = fmaxf(all, stat[k].x);
  const float ref = all == -CUDART_INF_F ? 0.f : all;
  float sum = 0.f, r[4] = {};
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const float w = pa_exp2(stat[k].x - ref);
    const float4 v = acc[k][quad];
    sum = fmaf(w, stat[k].y, sum);
    r[0] = fmaf(w, v.x, r[0]);
    r[1] = fmaf(w, v.y, r[1]);
    r[2] = fmaf(w, v.z, r[2]);
    r[3] = fmaf(w, v.w, r[3]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.out + (s.t0 + i) * a.o_ts + (t.head * a.group + hg) * a.o_hs + 4 * quad) =
      make_uint2(pa_bf16x2(r[0] * inv, r[1] * inv), pa_bf16x2(r[2] * inv, r[3] * inv));
}

template <int D>
static g4_status launch_few(g4_ctx* ctx, PaArgs a, PagedBatch b, const g4_paged_cache* c) {
  const void* fn = (const void*)paged_few_kernel<D>;
  const size_t smem = sizeof(FewSmem<D>) + 1024;
  g4_status st = allow_max_dynamic_smem(ctx, fn, smem, "paged attention (few rows)");
  if (st != G4_OK) return st;
  a.tile_rows = kPaFewRows;
  a.item_cost = 1;  // (32 single tokens: 59 us with 1, 64 us with 0)
  long long items, keys;
  paged_bounds(b, a, items, keys);
  if (items * (keys + a.item_cost) >= (1ll << 30))
    return fail(ctx, G4_ERR_TOO_LARGE, "paged attention: more than 2^30 tiles in one call");
  a.ranges = ctx->sm_count;
  if (items * keys < a.ranges) a.ranges = static_cast<int>(items * keys);
  const int low = b.page_rows & -b.page_rows;
  a.log_box = 0;
  while ((1 << a.log_box) < low && a.log_box < 7) ++a.log_box;
  CUtensorMap km, vm;
  const int dims[4] = {c->page_rows, D / 64, c->n_kv_heads, c->n_pages};
  const int box[4] = {1 << a.log_box, a.log_box == 7 ? 2 : 1, 1, 1};
  if (!tile_map(&km, c->k, dims, {c->k_row_stride, 64, c->k_head_stride, c->k_page_stride}, box) ||
      !tile_map(&vm, c->v, dims, {c->v_row_stride, 64, c->v_head_stride, c->v_page_stride}, box))
    return fail(ctx, G4_ERR_UNSUPPORTED, "paged attention: the cache's layout has no TMA descriptor");
  Scratch* scr = ctx->buf.scratch;
  uint64_t budget = ctx->wait_budget_ns;
  void* args[] = {(void*)&km, (void*)&vm, (void*)&a, (void*)&b, (void*)&scr, (void*)&budget};
  st = launch_kernel(ctx, fn, dim3(a.ranges), dim3(kFewThreads), smem, args, false, "paged attention (few rows)");
  if (st != G4_OK) return st;
  const long long rows = static_cast<long long>(b.n_tokens) * a.group;
  void* jargs[] = {(void*)&a, (void*)&b};
  const bool many_parts = 4 * items <= a.ranges;
  const void* join = many_parts ? (const void*)paged_few_join_kernel<D, 512> : (const void*)paged_few_join_kernel<D, 256>;
  return launch_kernel(ctx, join, dim3(a.ranges, rows < kPaFewRows ? static_cast<int>(rows) : kPaFewRows),
                       dim3(many_parts ? 512 : 256), 0, jargs, false, "paged attention join (few rows)");
}

g4_status launch_paged_few(g4_ctx* ctx, PaArgs a, const PagedBatch& b, const g4_paged_cache* c) {
  return c->head_dim == DS ? launch_few<DS>(ctx, a, b, c) : launch_few<DF>(ctx, a, b, c);
}

}  // namespace g4
