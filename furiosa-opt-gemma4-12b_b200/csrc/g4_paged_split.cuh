// What the two paged attention kernels share (g4_paged_attn.cu: tiles of 256 rows on CTA pairs;
// g4_paged_few.cu: 16 rows on single CTAs): arguments, bounded waits, tensor-core plumbing and
// the work split.
#pragma once

#include <cuda.h>

#include "g4_paged.cuh"

namespace g4 {

// Division by a number fixed for the call, by multiplication (round-up method; exact for
// 0 <= n < 2^31): a hardware divide goes through the unit that the softmax's exponentials
// keep busy, and took the copying warps over 1000 cycles.
struct PaDiv {
  uint32_t mul, shift;
  __device__ __forceinline__ int div(int n) const {
    const uint32_t u = static_cast<uint32_t>(n);
    return static_cast<int>((__umulhi(u, mul) + u) >> shift);
  }
};
constexpr int kPaFewRows = 16;  // rows of an item of g4_paged_few.cu
constexpr int kPaKeys = 128;    // cache rows per unit
constexpr float kPaLag = 8.f;   // log2 of how far a row's maximum may rise before O is rescaled
struct PaArgs {
  const uint16_t* q;
  long long q_ts, q_hs;
  uint16_t* out;
  long long o_ts, o_hs;
  int group, n_kv, window;  // query heads per KV head, KV heads
  int tile_rows;            // rows of an item
  int item_cost;            // what an item's start and end cost, in units, for the work split
  PaDiv by_group, by_page;  // by group and by the rows of a page
  float scale;              // times log2(e)
  int log_box;              // log2 of the cache rows per TMA box
  int q_tma;                // Q rows come by TMA (the group divides 128), else by the softmax warps
  int ranges;
  float* part;              // partial sums of split items (layout: each kernel's own)
  struct PaTail* tail;      // [ranges]
};
// An item begun in a range and finished by later ones.
struct PaTail {
  int seq, tile, head, parts;  // seq -1: none
};

// ---------------------------------------------------------------------------- PTX
// kWide: the barrier also announces ordinary stores of the other CTA's threads.
template <bool kWide>
__device__ __forceinline__ bool pa_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  if (kWide)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  return ok != 0;
}
// Bounded wait: after the budget, or once another role of the CTA gave up, false.
template <bool kWide = false>
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort, uint64_t budget) {
  for (int i = 0; i < 64; ++i)
    if (pa_try<kWide>(bar, parity)) return true;
  const uint64_t end = global_ns() + budget;
  while (!pa_try<kWide>(bar, parity)) {
    if (*abort != 0u) return false;
    if (global_ns() > end) {
      *abort = 1u;
      return false;
    }
  }
  return true;
}
// The same by a whole warp, with one answer.
__device__ __forceinline__ bool pa_wait_warp(uint64_t* bar, uint32_t parity, volatile uint32_t* abort,
                                             uint64_t budget) {
  return __all_sync(0xffffffffu, pa_wait(bar, parity, abort, budget));
}
__device__ __forceinline__ uint64_t pa_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32) | (static_cast<uint64_t>(1u) << 46) |
         (static_cast<uint64_t>(2u) << 61);
}
__device__ __forceinline__ void pa_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void pa_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pa_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t pa_swizzle(int row, int c) {  // 16-byte chunk c of a 128-byte row
  return static_cast<uint32_t>(row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// ---------------------------------------------------------------------------- work split
// The first row that a token at `pos` sees.  (A position may be negative and a window as large as
// an int holds: nothing is subtracted that could wrap.)
__device__ __forceinline__ int pa_low(int pos, int window) {
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}
// Key tiles of row tile `tile` of a sequence: [kt0, kt0 + n), n >= 1 (a tile nothing is
// visible to still has its zeros to write).
__device__ __forceinline__ int pa_key_tiles(const PagedSeq& s, int tile, const PaArgs& a, int& kt0) {
  const int r0 = tile * a.tile_rows;
  const int i0 = a.by_group.div(r0), i1 = min(s.n - 1, a.by_group.div(r0 + a.tile_rows - 1));
  const int first = s.kv - s.n;
  const int hi = first + i1 + 1;
  kt0 = 0;
  if (hi <= 0) return 1;
  kt0 = pa_low(first + i0, a.window) / kPaKeys;
  return (hi + kPaKeys - 1) / kPaKeys - kt0;
}
__device__ __forceinline__ int pa_tiles(const PagedSeq& s, const PaArgs& a) {
  return (s.n * a.group + a.tile_rows - 1) / a.tile_rows;  // (n * group < 2^30: checked by the host)
}
__device__ __forceinline__ int pa_warp_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Where range r of n starts: r * u / n.
__device__ __forceinline__ int pa_share(int r, int u, int n) {
  return u < (1 << 22) ? static_cast<int>(static_cast<uint32_t>(r) * static_cast<uint32_t>(u) / static_cast<uint32_t>(n))
                       : static_cast<int>(static_cast<long long>(r) * u / n);
}
// Units and items of every sequence into w[]; the whole CTA.  (The call's sum is below 2^30:
// checked by the host.)
struct PaCount {
  int units, items;
};
__device__ __forceinline__ void pa_count(const PagedBatch& b, const PaArgs& a, PaCount* w, Scratch* scr, bool report) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int s0 = 0; s0 < b.n_seqs; s0 += blockDim.x) {
    const int s = s0 + tid;
    PagedSeq q = {0, 0, 0};
    bool bad = false;
    if (s < b.n_seqs) q = paged_seq(b, s, &bad);
    if (report && s == 0 && b.n_seqs > 0 && b.q_start[0] < 0) bad = true;
    if (report && bad) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    const int tiles = pa_tiles(q, a);
    int sum = 0, kt0;
    if (tiles <= 2)
      for (int t = 0; t < tiles; ++t) sum += pa_key_tiles(q, t, a, kt0);
    for (uint32_t left = __ballot_sync(0xffffffffu, tiles > 2); left != 0; left &= left - 1) {
      const int from = __ffs(left) - 1;
      const PagedSeq o = {0, __shfl_sync(0xffffffffu, q.n, from), __shfl_sync(0xffffffffu, q.kv, from)};
      int x = 0;
      for (int t = lane; t < pa_tiles(o, a); t += 32) x += pa_key_tiles(o, t, a, kt0);
      x = __reduce_add_sync(0xffffffffu, x);
      if (lane == from) sum = x;
    }
    if (s < b.n_seqs) w[s] = {sum * a.n_kv, tiles * a.n_kv};
  }
}
// The item that position `want` (< the total) of the weighted order lies in, and how far into
// it: an item weighs its units and `cost`.  One warp, every lane gets the answer.
__device__ __forceinline__ void pa_find(const PagedBatch& b, const PaArgs& a, const PaCount* w, int cost, int want, int lane, int& seq,
                        int& tile, int& head, int& offset) {
  int base = 0;
  seq = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
    const int x = s0 + lane < b.n_seqs ? w[s0 + lane].units + cost * w[s0 + lane].items : 0;
    const int incl = pa_warp_scan(x, lane);
    const uint32_t past = __ballot_sync(0xffffffffu, base + incl > want);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      seq = s0 + at;
      base += __shfl_sync(0xffffffffu, incl - x, at);
      break;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  bool bad;
  const PagedSeq q = paged_seq(b, seq, &bad);
  const int tiles = pa_tiles(q, a);
  tile = 0;
  int weight = 1, kt0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int n = t0 + lane < tiles ? pa_key_tiles(q, t0 + lane, a, kt0) + cost : 0;
    const int x = n * a.n_kv;
    const int incl = pa_warp_scan(x, lane);
    const uint32_t past = __ballot_sync(0xffffffffu, base + incl > want);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      tile = t0 + at;
      weight = __shfl_sync(0xffffffffu, n, at);
      base += __shfl_sync(0xffffffffu, incl - x, at);
      break;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  head = (want - base) / weight;
  offset = want - base - head * weight;
}

// A CTA's (or pair's) share of the call: the weight of all items, where the range starts in it, the
// ranges in use, an item's cost in units, and the item that the range starts in.
struct PaRange {
  int units, first, count, cost;
  int seq, tile, head, offset;
};
// Range `range` of the call, from the counts; one warp.  What the host lets through weighs less
// than 2^30, as long as q_start does not fall: where it does, sequences may share tokens, and a call
// that weighs more by that is not done at all (reported once).
__device__ __forceinline__ PaRange pa_range(const PagedBatch& b, const PaArgs& a, const PaCount* w, int range, int lane,
                                            Scratch* scr) {
  constexpr uint32_t kMost = 1u << 30;  // (a sequence alone stays below it; sums stop there)
  uint32_t units = 0, items = 0;
#pragma unroll 1
  for (int s = lane; s < b.n_seqs; s += 32) {
    units = min(units + w[s].units, kMost);
    items = min(items + w[s].items, kMost);
  }
  // in 32nds, so that the lanes' sum fits: below kMost / 32 what follows is off by no wrap
  const bool most = __reduce_add_sync(0xffffffffu, (units + a.item_cost * items) / 32) >= kMost / 32;
  units = __reduce_add_sync(0xffffffffu, units);
  items = __reduce_add_sync(0xffffffffu, items);
  PaRange r = {0, 0, 0, 0, 0, 0, 0, 0};
  if (most) {
    if (range == 0 && lane == 0) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    return r;
  }
  r.cost = static_cast<int>(units) <= a.ranges ? 0 : a.item_cost;  // with a CTA (pair) for every unit, each gets one
  r.units = static_cast<int>(units + r.cost * items);
  r.count = min(a.ranges, r.units);  // none is empty
  if (range < r.count) {
    r.first = pa_share(range, r.units, r.count);
    pa_find(b, a, w, r.cost, r.first, lane, r.seq, r.tile, r.head, r.offset);
  }
  return r;
}

// The items of a range, in order; every role walks them alike.
struct PaWalk {
  const PagedBatch& b;
  const PaArgs& a;
  const int cost;
  int left;  // weight after the current item
  int seq, tile, head;
  PagedSeq s;
  int kt0, nk, begin, end;  // key tiles of the current item: [begin, end) of its nk are this range's
  int next_offset;
  __device__ PaWalk(const PagedBatch& batch, const PaArgs& args, const PaRange& r, int weight)
      : b(batch), a(args), cost(r.cost), left(weight), seq(r.seq), tile(r.tile), head(r.head - 1), next_offset(r.offset) {
    bool bad;
    s = left > 0 ? paged_seq(b, seq, &bad) : PagedSeq{0, 0, 0};
  }
  __device__ bool next() {
    if (left <= 0) return false;
    if (++head == a.n_kv) {
      head = 0;
      if (++tile >= pa_tiles(s, a)) {
        bool bad;
        tile = 0;
        do {
          // (never past the last one, as long as nobody writes the batch during the call)
          if (++seq >= b.n_seqs) {
            left = 0;
            return false;
          }
          s = paged_seq(b, seq, &bad);
        } while (s.n == 0);
      }
    }
    nk = pa_key_tiles(s, tile, a, kt0);
    // the item's first `cost` positions are its overhead, the others its units
    const int offset = next_offset;
    const int to = min(nk + cost, offset + left);
    next_offset = 0;
    begin = max(0, offset - cost);
    end = max(0, to - cost);
    left -= to - offset;
    return end > begin;  // (no unit: the range ends within the overhead)
  }
  // the first cache row any new token of the sequence sees
  __device__ int low() const { return pa_low(s.kv - s.n, a.window); }
  // a V tile that reaches past the sequence's visible rows
  __device__ bool edge(int kt) const { return (kt + 1) * kPaKeys > s.kv || kt * kPaKeys < low(); }
};

// A position in a ring of stages [first, first + n): the stage, the parity of the barrier phase
// that its use ends, and the uses before it.
struct PaRing {
  const int first, n;
  int stage;
  uint32_t parity = 0, passed = 0;
  __device__ __forceinline__ PaRing(int first_, int n_) : first(first_), n(n_), stage(first_) {}
  __device__ __forceinline__ void next() {
    ++passed;
    if (++stage == first + n) {
      stage = first;
      parity ^= 1u;
    }
  }
};
__device__ __forceinline__ bool pa_elect() {  // one lane of a converged warp
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// ---------------------------------------------------------------------------- host
inline PaDiv divisor(int d) {
  uint32_t shift = 0;
  while ((1ull << shift) < static_cast<uint64_t>(d)) ++shift;
  return {static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// A 5-D tensor of 64-dim rows with the 128-byte swizzle; `stride` in elements.
inline bool tile_map(CUtensorMap* m, const uint16_t* base, const int (&n)[4], const int64_t (&stride)[4],
                     const int (&box)[4]) {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
               ? reinterpret_cast<EncodeFn>(p)
               : nullptr;
  }();
  if (fn == nullptr) return false;
  cuuint64_t dims[5] = {64}, strides[4];
  cuuint32_t boxes[5] = {64};
  for (int i = 0; i < 4; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(n[i]);
    // the stride of a dimension of size one is never used, but has to be a legal one
    strides[i] = static_cast<cuuint64_t>(n[i] > 1 ? stride[i] : 64) * 2;
    boxes[i + 1] = static_cast<cuuint32_t>(box[i]);
  }
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<uint16_t*>(base), dims, strides, boxes, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


// Scratch of split items (tails and partial sums), allocated at the first call; both kernels use it,
// one after the other on the context's stream.
g4_status paged_scratch(g4_ctx* ctx, PaArgs& a);
// The kernel of g4_paged_few.cu.
g4_status launch_paged_few(g4_ctx* ctx, PaArgs a, const PagedBatch& b, const g4_paged_cache* c);
// No more items than this, and 128-row key tiles of the longest cache there can be.
inline void paged_bounds(const PagedBatch& b, const PaArgs& a, long long& items, long long& keys) {
  const long long rows = static_cast<long long>(b.n_tokens) * a.group;
  items = (rows / a.tile_rows + (b.n_seqs < b.n_tokens ? b.n_seqs : b.n_tokens)) * a.n_kv;
  keys = (static_cast<long long>(b.max_pages) * b.page_rows + kPaKeys - 1) / kPaKeys;
  if (keys < 1) keys = 1;
  if (keys > (1 << 24)) keys = 1 << 24;  // (a sequence is cut off below 2^31 rows)
}

}  // namespace g4
