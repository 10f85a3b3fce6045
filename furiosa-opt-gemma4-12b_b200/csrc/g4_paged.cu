// Paged KV caches: storing a chunk's K and V rows (with the norms and rotary positions the
// single-token projections apply), copying pages, and compaction.  The attention over the
// pages is g4_paged_attn.cu.
#include <climits>
#include <string>

#include "g4_paged.cuh"

namespace g4 {

// ---------------------------------------------------------------------------- host checks
static bool bad_stride(int64_t s) { return s < 0 || s % 8 != 0 || s > (int64_t(1) << 38); }

g4_status check_paged_cache(g4_ctx* ctx, const g4_paged_cache* c) {
  if (c == nullptr) return fail(ctx, G4_ERR_BAD_ARG, "paged cache: null descriptor");
  if (!aligned16(c->k) || !aligned16(c->v))
    return fail(ctx, G4_ERR_BAD_ARG, "paged cache: k or v is null or not 16-byte aligned");
  if (c->head_dim != DS && c->head_dim != DF)
    return fail(ctx, G4_ERR_UNSUPPORTED, "paged cache: head_dim must be 256 or 512");
  if (c->page_rows < 8 || c->page_rows > 65536 || c->page_rows % 8 != 0)
    return fail(ctx, G4_ERR_BAD_ARG, "paged cache: page_rows must be a multiple of 8 in [8, 65536]");
  if (c->n_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 1024)
    return fail(ctx, G4_ERR_BAD_ARG, "paged cache: no pages, or n_kv_heads not in [1, 1024]");
  if (bad_stride(c->k_page_stride) || bad_stride(c->k_row_stride) || bad_stride(c->k_head_stride) ||
      bad_stride(c->v_page_stride) || bad_stride(c->v_row_stride) || bad_stride(c->v_head_stride))
    return fail(ctx, G4_ERR_BAD_ARG, "paged cache: strides must be multiples of 8 elements, not negative");
  const int64_t along[][3] = {{c->n_pages, c->k_page_stride, c->v_page_stride},
                              {c->page_rows, c->k_row_stride, c->v_row_stride},
                              {c->n_kv_heads, c->k_head_stride, c->v_head_stride}};
  for (const auto& d : along)
    if (d[0] > 1 && (d[1] < c->head_dim || d[2] < c->head_dim))
      return fail(ctx, G4_ERR_BAD_ARG, "paged cache: a stride below head_dim makes rows overlap");
  return G4_OK;
}
g4_status check_paged_batch(g4_ctx* ctx, const g4_paged_batch* b) {
  if (b == nullptr) return fail(ctx, G4_ERR_BAD_ARG, "paged batch: null descriptor");
  if (b->n_seqs < 0 || b->n_seqs > G4_PAGED_MAX_SEQS || b->n_tokens < 0 || b->max_pages < 0 ||
      b->n_tokens > (1 << 22) || b->table_stride < b->max_pages)
    return fail(ctx, G4_ERR_BAD_ARG, "paged batch: n_seqs, n_tokens, max_pages or table_stride out of range");
  const void* ptrs[] = {b->q_start, b->kv_len, b->tables};  // no tables where no sequence can have a page
  for (int i = 0; i < (b->max_pages > 0 ? 3 : 2); ++i)
    if (b->n_seqs > 0 && (ptrs[i] == nullptr || (reinterpret_cast<uintptr_t>(ptrs[i]) & 3u)))
      return fail(ctx, G4_ERR_BAD_ARG, "paged batch: tables, q_start or kv_len is null or misaligned");
  return G4_OK;
}
g4_status check_rows(g4_ctx* ctx, const void* p, int64_t token_stride, int64_t head_stride, const char* what) {
  if (!aligned16(p)) return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + " is null or not 16-byte aligned");
  if (bad_stride(token_stride) || bad_stride(head_stride))
    return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + ": strides must be multiples of 8 elements, not negative");
  return G4_OK;
}
g4_status check_out_rows(g4_ctx* ctx, const void* p, int64_t token_stride, int64_t head_stride, int tokens, int heads,
                         int head_dim, const char* what) {
  const g4_status st = check_rows(ctx, p, token_stride, head_stride, what);
  if (st == G4_OK && ((tokens > 1 && token_stride < head_dim) || (heads > 1 && head_stride < head_dim)))
    return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + ": a stride below head_dim makes rows overlap");
  return st;
}
PagedBatch paged_batch(const g4_paged_batch* b, const g4_paged_cache* c) {
  return {b->tables,  static_cast<long long>(b->table_stride), b->q_start, b->kv_len, b->max_pages,
          b->n_seqs, b->n_tokens, c->n_pages, c->page_rows};
}

// ---------------------------------------------------------------------------- norm, rotate, store
// out[d] = n[d] cos[d] + n[d +- D/2] sin[d], n = x rsqrt(mean x^2 + eps) w.  D / 16 lanes have a
// head: a lane its dims 8 l .. 8 l + 7 and D / 2 + 8 l .. , so the pairs that turn into each
// other meet in one lane, and a warp has two heads of 256 or one of 512 at a time.  A warp takes
// kIter such steps of one token's q, k or v heads: q, k and v are read once and written once,
// the token's cos/sin row and the norm weights once per warp.  The heads' loads go out first,
// ahead of the chain token -> sequence -> page, whose two round trips they hide (the sequence is
// found by a scan, 32 a round trip: more than 32 sequences make that chain longer).  4096 sliding
// tokens keep DRAM 38 % and the SMs' pipes 36 % busy: what bounds them is how much 16 warps an SM (110
// registers) have in flight.
struct StoreArgs {
  const uint16_t *q, *k, *v;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const uint16_t *qw, *kw, *cos, *sin;
  int n_heads, n_kv, n_positions;
  uint16_t *kc, *vc;
  long long kp, kr, kh, vp, vr, vh;
  uint16_t* out;
  long long o_ts, o_hs;
};
constexpr int kStoreThreads = 128;

__device__ __forceinline__ uint4 ldg128(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }
// Eight bf16 as four pairs of f32, and back.
__device__ __forceinline__ void unpack8(const uint4 w, uint64_t (&f)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pa_pair(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    pa_unpair(f[i], a, b);
    u[i] = pa_bf16x2(a, b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// The sequence whose new tokens include token t (-1: none), 32 sequences at a time, and its
// position; bad: its numbers had to be cut off.
__device__ __forceinline__ int seq_of_token(const PagedBatch& b, int t, int lane, int& pos, bool& bad) {
  for (int s0 = 0; s0 < b.n_seqs; s0 += 32) {
    PagedSeq q = {0, 0, 0};
    bool cut = false;
    if (s0 + lane < b.n_seqs) q = paged_seq(b, s0 + lane, &cut);
    const uint32_t hit = __ballot_sync(0xffffffffu, q.t0 <= t && t < q.t0 + q.n);
    if (hit != 0) {
      const int from = __ffs(hit) - 1;
      pos = __shfl_sync(0xffffffffu, q.kv - q.n + (t - q.t0), from);
      bad = __shfl_sync(0xffffffffu, static_cast<int>(cut), from) != 0;
      return s0 + from;
    }
  }
  return -1;
}

template <int D, int kIter>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const __grid_constant__ StoreArgs a,
                                                                    const __grid_constant__ PagedBatch b,
                                                                    Scratch* scr) {
  constexpr int kLanes = D / 16, kAtOnce = 32 / kLanes, kPer = kIter * kAtOnce;  // lanes a head; heads a step, a warp
  pdl_wait();
  const int lane = threadIdx.x & 31, hl = lane % kLanes, sub = lane / kLanes;
  const int q_groups = (a.n_heads + kPer - 1) / kPer, kv_groups = (a.n_kv + kPer - 1) / kPer;
  const int groups = q_groups + 2 * kv_groups;  // of q heads, of k heads, of v heads
  const int unit = blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5);
  const int t = unit / groups, group = unit - t * groups;
  if (unit == 0) paged_check_batch(b, lane, scr);
  if (t >= b.n_tokens) return;
  const bool is_q = group < q_groups, is_v = group >= q_groups + kv_groups;
  const int head0 = (is_q ? group : (group - q_groups) % kv_groups) * kPer + sub, heads = is_q ? a.n_heads : a.n_kv;
  const uint16_t* src = is_q ? a.q + t * a.q_ts : (is_v ? a.v + t * a.v_ts : a.k + t * a.k_ts);
  const long long src_hs = is_q ? a.q_hs : (is_v ? a.v_hs : a.k_hs);
  uint4 x[kIter][2];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int head = head0 + i * kAtOnce;
    if (head >= heads) continue;
    x[i][0] = ldg128(src + head * src_hs + 8 * hl);
    x[i][1] = ldg128(src + head * src_hs + D / 2 + 8 * hl);
  }
  uint64_t w[2][4];
  if (!is_v) {
    const uint16_t* weight = is_q ? a.qw : a.kw;
    unpack8(ldg128(weight + 8 * hl), w[0]);
    unpack8(ldg128(weight + D / 2 + 8 * hl), w[1]);
  }
  int pos = -1;
  bool bad = false;
  const int s = seq_of_token(b, t, lane, pos, bad);
  if (s < 0) return;
  bool live = pos >= 0 && !bad;  // (of a sequence that was cut off, the positions are not known)
  if (pos >= a.n_positions) live = false, bad = true;
  int page = 0, row = 0;
  if (live) {  // (pos < kv <= max_pages * page_rows)
    const int j = pos / b.page_rows;
    page = b.tables[s * b.table_stride + j];
    row = pos - j * b.page_rows;
  }
  uint64_t cs[2][4], sn[2][4];
  if (live) {
    if (!is_v) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        unpack8(ldg128(a.cos + static_cast<long long>(pos) * D + c * (D / 2) + 8 * hl), cs[c]);
        unpack8(ldg128(a.sin + static_cast<long long>(pos) * D + c * (D / 2) + 8 * hl), sn[c]);
      }
    }
    if (page < 0 || page >= b.n_pages) live = false, bad = true;
  }
  if (bad && lane == 0) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
  if (!live && !is_q) return;
  uint16_t* dst = is_q ? a.out + t * a.o_ts : (is_v ? a.vc + page * a.vp + row * a.vr : a.kc + page * a.kp + row * a.kr);
  const long long dst_hs = is_q ? a.o_hs : (is_v ? a.vh : a.kh);
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int head = head0 + i * kAtOnce;
    const bool mine = head < heads;
    uint64_t f[2][4], ss = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      unpack8(mine ? x[i][c] : make_uint4(0, 0, 0, 0), f[c]);
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = pa_fma2(f[c][j], f[c][j], ss);
    }
    float s0, s1;
    pa_unpair(ss, s0, s1);
    s0 += s1;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    const float r = rsqrtf(fmaf(s0, 1.f / D, EPS));  // (2 ulp: far below the one rounding to bf16)
    const uint64_t rr = pa_pair(r, r);
    uint4 y0, y1;
    if (is_v) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[c][j] = pa_mul2(f[c][j], rr);
      y0 = pack8(f[0]);
      y1 = pack8(f[1]);
    } else {
      uint64_t y[2][4];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[c][j] = pa_mul2(pa_mul2(f[c][j], rr), w[c][j]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[c][j] = pa_fma2(f[c][j], cs[c][j], pa_mul2(f[c ^ 1][j], sn[c][j]));
      y0 = live ? pack8(y[0]) : make_uint4(0, 0, 0, 0);
      y1 = live ? pack8(y[1]) : make_uint4(0, 0, 0, 0);
    }
    if (mine) {
      *reinterpret_cast<uint4*>(dst + head * dst_hs + 8 * hl) = y0;
      *reinterpret_cast<uint4*>(dst + head * dst_hs + D / 2 + 8 * hl) = y1;
    }
  }
}
// Steps a warp: kStoreIter where that still gives every SM 32 warps, else one.  4096 sliding tokens
// (138 MB): 29.6 us with 4, 33.6 with 2, 36.5 with 8; one token 2.5 us with 1.
constexpr int kStoreIter = 4;
template <int D>
static const void* store_kernel(bool many) {
  return many ? (const void*)paged_store_kernel<D, kStoreIter> : (const void*)paged_store_kernel<D, 1>;
}

// ---------------------------------------------------------------------------- page copies
// One block per (layer and K/V, move, slice of the page's rows); pure traffic, 2 x the bytes.
constexpr int kCopyThreads = 256;
constexpr int kCopyLayers = 56;  // per launch: the descriptors travel in the 4 KB of kernel arguments
struct CopyLayer {
  uint16_t* base[2];  // K, V
  long long page_stride[2];
  int row_stride[2], head_stride[2];
  int n_kv, log_chunks;  // 16-byte chunks per head: 1 << log_chunks
};
struct CopyArgs {
  const int32_t *src, *dst, *rows;  // rows null: whole pages
  int n, n_layers, n_pages, page_rows, slices;
  int32_t* tables;  // null: none
  long long table_stride;
  int n_seqs, max_pages;
  const int32_t* page_map;
  CopyLayer layer[kCopyLayers];
};
static_assert(sizeof(CopyArgs) + 16 <= 4096, "kernel arguments");

__global__ void __launch_bounds__(kCopyThreads) paged_copy_kernel(const __grid_constant__ CopyArgs a, Scratch* scr) {
  pdl_wait();
  const int tid = threadIdx.x;
  if (blockIdx.z == 2u * a.n_layers) {  // the block tables
    const long long total = static_cast<long long>(a.n_seqs) * a.max_pages;
    const long long step = static_cast<long long>(gridDim.x) * gridDim.y * kCopyThreads;
    for (long long i = (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * kCopyThreads + tid; i < total;
         i += step) {
      int32_t* e = a.tables + i / a.max_pages * a.table_stride + i % a.max_pages;
      const int p = *e;
      if (p < 0) continue;
      const int to = p < a.n_pages ? a.page_map[p] : -1;
      if (to >= 0 && to < a.n_pages)
        *e = to;
      else
        atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    }
    return;
  }
  const CopyLayer& l = a.layer[blockIdx.z >> 1];
  const int kv = blockIdx.z & 1;
  for (int m = blockIdx.y; m < a.n; m += gridDim.y) {
    const int s = a.src[m], d = a.dst[m];
    int rows = a.rows != nullptr ? a.rows[m] : a.page_rows;
    const bool ok = s >= 0 && s < a.n_pages && d >= 0 && d < a.n_pages && rows >= 0 && rows <= a.page_rows;
    if (!ok && tid == 0) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
    if (s < 0 || s >= a.n_pages || d < 0 || d >= a.n_pages || s == d) continue;
    rows = min(max(rows, 0), a.page_rows);
    const uint16_t* from = l.base[kv] + s * l.page_stride[kv];
    uint16_t* to = l.base[kv] + d * l.page_stride[kv];
    const int per_row = l.n_kv << l.log_chunks;
    const int per_slice = (a.page_rows + a.slices - 1) / a.slices;
    const int r0 = blockIdx.x * per_slice, r1 = min(rows, r0 + per_slice);
    for (long long i = static_cast<long long>(r0) * per_row + tid; i < static_cast<long long>(r1) * per_row;
         i += kCopyThreads) {
      const int r = static_cast<int>(i / per_row), in_row = static_cast<int>(i % per_row);
      const int h = in_row >> l.log_chunks, c = in_row & ((1 << l.log_chunks) - 1);
      const long long off = static_cast<long long>(r) * l.row_stride[kv] +
                            static_cast<long long>(h) * l.head_stride[kv] + 8 * c;
      *reinterpret_cast<uint4*>(to + off) = ldg128(from + off);
    }
  }
}

static g4_status launch_copies(g4_ctx* ctx, const g4_paged_cache* caches, int n_layers, CopyArgs a) {
  for (int l0 = 0; l0 < n_layers; l0 += kCopyLayers) {
    CopyArgs p = a;
    p.n_layers = n_layers - l0 < kCopyLayers ? n_layers - l0 : kCopyLayers;
    int row_bytes = 0;
    for (int i = 0; i < p.n_layers; ++i) {
      const g4_paged_cache& c = caches[l0 + i];
      p.layer[i] = {{c.k, c.v},
                    {c.k_page_stride, c.v_page_stride},
                    {static_cast<int>(c.k_row_stride), static_cast<int>(c.v_row_stride)},
                    {static_cast<int>(c.k_head_stride), static_cast<int>(c.v_head_stride)},
                    c.n_kv_heads,
                    c.head_dim == DS ? 5 : 6};
      if (c.n_kv_heads * c.head_dim * 2 > row_bytes) row_bytes = c.n_kv_heads * c.head_dim * 2;
    }
    const bool last = l0 + kCopyLayers >= n_layers;
    if (!last) p.tables = nullptr;
    // slices of about 32 KB of the widest layer
    const long long slices = (static_cast<long long>(p.page_rows) * row_bytes + 32767) / 32768;
    p.slices = static_cast<int>(slices < p.page_rows ? slices : p.page_rows);
    if (p.slices < 1) p.slices = 1;
    const dim3 grid(p.slices, p.n < 1 ? 1 : (p.n > 32768 ? 32768 : p.n), 2 * p.n_layers + (p.tables != nullptr ? 1 : 0));
    Scratch* scr = ctx->buf.scratch;
    void* args[] = {(void*)&p, (void*)&scr};
    const g4_status st = launch_kernel(ctx, (const void*)paged_copy_kernel, grid, dim3(kCopyThreads), 0, args, false,
                                       "paged copy");
    if (st != G4_OK) return st;
  }
  return G4_OK;
}

static g4_status check_layers(g4_ctx* ctx, const g4_paged_cache* caches, int n_layers) {
  if (caches == nullptr || n_layers < 1) return fail(ctx, G4_ERR_BAD_ARG, "no layers");
  for (int i = 0; i < n_layers; ++i) {
    const g4_status st = check_paged_cache(ctx, caches + i);
    if (st != G4_OK) return st;
    const g4_paged_cache& c = caches[i];
    if (c.page_rows != caches[0].page_rows || c.n_pages != caches[0].n_pages)
      return fail(ctx, G4_ERR_BAD_ARG, "layers differ in page_rows or n_pages");
    if (c.k_row_stride > INT_MAX || c.v_row_stride > INT_MAX || c.k_head_stride > INT_MAX || c.v_head_stride > INT_MAX)
      return fail(ctx, G4_ERR_BAD_ARG, "row or head stride of 2^31 elements or more");
  }
  return G4_OK;
}
static bool bad_words(const void* p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 3u) != 0; }

}  // namespace g4

using namespace g4;

extern "C" {

g4_status g4_paged_store_qkv(g4_ctx* ctx, const g4_bf16* q, int64_t q_token_stride, int64_t q_head_stride,
                             int n_heads, const g4_bf16* k, int64_t k_token_stride, int64_t k_head_stride,
                             const g4_bf16* v, int64_t v_token_stride, int64_t v_head_stride,
                             const g4_bf16* q_rms_weight, const g4_bf16* k_rms_weight, const g4_bf16* cos,
                             const g4_bf16* sin, int n_positions, const g4_paged_cache* cache,
                             const g4_paged_batch* batch, g4_bf16* q_out, int64_t out_token_stride,
                             int64_t out_head_stride) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_paged_cache(ctx, cache);
  if (st == G4_OK) st = check_paged_batch(ctx, batch);
  if (st != G4_OK) return st;
  if (n_heads < 1 || n_heads > 4096) return fail(ctx, G4_ERR_BAD_ARG, "n_heads must be in [1, 4096]");
  if (n_positions < 1) return fail(ctx, G4_ERR_BAD_ARG, "n_positions must be positive");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return G4_OK;
  if ((st = check_rows(ctx, q, q_token_stride, q_head_stride, "q")) != G4_OK) return st;
  if ((st = check_rows(ctx, k, k_token_stride, k_head_stride, "k")) != G4_OK) return st;
  if ((st = check_rows(ctx, v, v_token_stride, v_head_stride, "v")) != G4_OK) return st;
  if ((st = check_out_rows(ctx, q_out, out_token_stride, out_head_stride, batch->n_tokens, n_heads, cache->head_dim,
                           "q_out")) != G4_OK)
    return st;
  if (!aligned16(q_rms_weight) || !aligned16(k_rms_weight) || !aligned16(cos) || !aligned16(sin))
    return fail(ctx, G4_ERR_BAD_ARG, "a norm weight, cos or sin is null or not 16-byte aligned");
  StoreArgs a = {q, k, v, q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                 q_rms_weight, k_rms_weight, cos, sin, n_heads, cache->n_kv_heads, n_positions, cache->k, cache->v,
                 cache->k_page_stride, cache->k_row_stride, cache->k_head_stride, cache->v_page_stride,
                 cache->v_row_stride, cache->v_head_stride, q_out, out_token_stride, out_head_stride};
  PagedBatch b = paged_batch(batch, cache);
  Scratch* scr = ctx->buf.scratch;
  const int at_once = 512 / cache->head_dim;
  const long long all = static_cast<long long>(batch->n_tokens) * (n_heads + 2 * cache->n_kv_heads);
  const bool many = all >= 32ll * kStoreIter * at_once * ctx->sm_count;
  const int per = (many ? kStoreIter : 1) * at_once;
  const void* fn = cache->head_dim == DS ? store_kernel<DS>(many) : store_kernel<DF>(many);
  const int groups = (n_heads + per - 1) / per + 2 * ((cache->n_kv_heads + per - 1) / per);
  const long long warps = static_cast<long long>(batch->n_tokens) * groups;
  const long long blocks = (warps + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
  if (blocks > INT_MAX / (kStoreThreads / 32)) return fail(ctx, G4_ERR_BAD_ARG, "too many tokens times heads for one call");
  void* args[] = {(void*)&a, (void*)&b, (void*)&scr};
  return launch_kernel(ctx, fn, dim3(static_cast<unsigned>(blocks)), dim3(kStoreThreads), 0, args, false,
                       "paged store");
}

g4_status g4_paged_copy(g4_ctx* ctx, const g4_paged_cache* caches, int n_layers, const int32_t* src,
                        const int32_t* dst, const int32_t* rows, int n) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_layers(ctx, caches, n_layers);
  if (st != G4_OK) return st;
  if (n < 0) return fail(ctx, G4_ERR_BAD_ARG, "negative copy count");
  if (n == 0) return G4_OK;
  if (bad_words(src) || bad_words(dst) || bad_words(rows))
    return fail(ctx, G4_ERR_BAD_ARG, "src, dst or rows is null or misaligned");
  CopyArgs a = {src, dst, rows, n, 0, caches[0].n_pages, caches[0].page_rows, 1, nullptr, 0, 0, 0, nullptr, {}};
  return launch_copies(ctx, caches, n_layers, a);
}

g4_status g4_paged_compact(g4_ctx* ctx, const g4_paged_cache* caches, int n_layers, const int32_t* src,
                           const int32_t* dst, int n, int32_t* tables, int64_t table_stride, int n_seqs,
                           int max_pages, const int32_t* page_map) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_layers(ctx, caches, n_layers);
  if (st != G4_OK) return st;
  if (n < 0 || n_seqs < 0 || max_pages < 0 || table_stride < max_pages)
    return fail(ctx, G4_ERR_BAD_ARG, "negative count, or table_stride below max_pages");
  const bool has_tables = n_seqs > 0 && max_pages > 0;
  if (n > 0 && (bad_words(src) || bad_words(dst)))
    return fail(ctx, G4_ERR_BAD_ARG, "src or dst is null or misaligned");
  if (has_tables && (bad_words(tables) || bad_words(page_map)))
    return fail(ctx, G4_ERR_BAD_ARG, "tables or page_map is null or misaligned");
  if (n == 0 && !has_tables) return G4_OK;
  CopyArgs a = {src, dst, nullptr, n, 0, caches[0].n_pages, caches[0].page_rows, 1,
                has_tables ? tables : nullptr, table_stride, n_seqs, max_pages, page_map, {}};
  return launch_copies(ctx, caches, n_layers, a);
}

}  // extern "C"
