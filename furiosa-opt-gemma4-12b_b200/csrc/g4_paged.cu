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
// A warp takes a token and kPer of its q, k and v heads; a head's D values stay in its
// registers (8 per lane and 16-byte chunk), so q, k and v are read once and written once.
// Memory bound: 4 B per element, and the token's cos/sin row, loaded once per warp.  The heads'
// loads go out first, ahead of the chain token -> sequence -> page, whose two L2 round trips
// they hide.  kPer = 4 where that still gives every SM 64 warps, else 1: a single token's heads
// then go to as many warps.  4096 sliding tokens (138 MB): 33.6 us with 4, 34.7 with 8, 37.5 with
// 2, 77 with 1; one token: 2.3 us with 1.
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
constexpr int kStoreThreads = 256;

__device__ __forceinline__ void unpack8(const uint4 w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]), bf16x2(f[4], f[5]), bf16x2(f[6], f[7]));
}
__device__ __forceinline__ uint4 ldg128(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }

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

template <int D, int kPer>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(const __grid_constant__ StoreArgs a,
                                                                    const __grid_constant__ PagedBatch b,
                                                                    Scratch* scr) {
  constexpr int C = D / 256;  // 16-byte chunks per lane: chunk c holds dims 256 c + 8 lane ..
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int slots = a.n_heads + 2 * a.n_kv, groups = (slots + kPer - 1) / kPer;  // q heads, k heads, v heads
  const int unit = blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5);
  const int t = unit / groups, slot0 = unit % groups * kPer;
  if (unit == 0) paged_check_batch(b, lane, scr);
  if (t >= b.n_tokens) return;
  uint4 x[kPer][C];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int slot = slot0 + i, k = slot - a.n_heads, v = k - a.n_kv;
    if (slot >= slots) continue;
    const uint16_t* src = k < 0 ? a.q + t * a.q_ts + slot * a.q_hs
                                : (v < 0 ? a.k + t * a.k_ts + k * a.k_hs : a.v + t * a.v_ts + v * a.v_hs);
#pragma unroll
    for (int c = 0; c < C; ++c) x[i][c] = ldg128(src + 256 * c + 8 * lane);
  }
  int pos = -1;
  bool bad = false;
  const int s = seq_of_token(b, t, lane, pos, bad);
  if (s < 0) return;
  bool live = pos >= 0;
  if (pos >= a.n_positions) live = false, bad = true;
  int page = 0, row = 0;
  if (live) {  // (pos < kv <= max_pages * page_rows)
    page = b.tables[s * b.table_stride + pos / b.page_rows];
    row = pos % b.page_rows;
  }
  float cf[C][8], sf[C][8];
  if (live) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      unpack8(ldg128(a.cos + static_cast<long long>(pos) * D + 256 * c + 8 * lane), cf[c]);
      unpack8(ldg128(a.sin + static_cast<long long>(pos) * D + 256 * c + 8 * lane), sf[c]);
    }
    if (page < 0 || page >= b.n_pages) live = false, bad = true;
  }
  if (bad && lane == 0) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int slot = slot0 + i, k = slot - a.n_heads, v = k - a.n_kv;
    if (slot >= slots || (!live && k >= 0)) continue;
    uint16_t* dst = k < 0 ? a.out + t * a.o_ts + slot * a.o_hs
                          : (v < 0 ? a.kc + page * a.kp + row * a.kr + k * a.kh
                                   : a.vc + page * a.vp + row * a.vr + v * a.vh);
    if (!live) {
#pragma unroll
      for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(dst + 256 * c + 8 * lane) = make_uint4(0, 0, 0, 0);
      continue;
    }
    float f[C][8], ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      unpack8(x[i][c], f[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(f[c][j], f[c][j], ss);
    }
    const float r = rsqrtf(fmaf(warp_sum(ss), 1.f / D, EPS));  // (2 ulp: far below the one rounding to bf16)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[c][j] *= r;
    if (v < 0) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float wf[8];
        unpack8(ldg128((k < 0 ? a.qw : a.kw) + 256 * c + 8 * lane), wf);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[c][j] *= wf[j];
      }
      // out[d] = x[d] cos[d] + x[d +- D/2] sin[d]: the other half is chunk c ^ 1 of this lane
      // (D = 512) or chunk 0 of lane ^ 16 (D = 256)
      float y[C][8];
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = C == 2 ? f[(c ^ 1) & (C - 1)][j] : __shfl_xor_sync(0xffffffffu, f[c][j], 16);
          y[c][j] = fmaf(f[c][j], cf[c][j], other * sf[c][j]);
        }
#pragma unroll
      for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(dst + 256 * c + 8 * lane) = pack8(y[c]);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(dst + 256 * c + 8 * lane) = pack8(f[c]);
    }
  }
}
constexpr int kStorePer = 4;
template <int kPer>
static const void* store_kernel(int head_dim) {
  return head_dim == DS ? (const void*)paged_store_kernel<DS, kPer> : (const void*)paged_store_kernel<DF, kPer>;
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
  const int slots = n_heads + 2 * cache->n_kv_heads;
  const int per = static_cast<long long>(batch->n_tokens) * slots >= 64ll * kStorePer * ctx->sm_count ? kStorePer : 1;
  const long long warps = static_cast<long long>(batch->n_tokens) * ((slots + per - 1) / per);
  const long long blocks = (warps + kStoreThreads / 32 - 1) / (kStoreThreads / 32);
  if (blocks > INT_MAX / (kStoreThreads / 32)) return fail(ctx, G4_ERR_BAD_ARG, "too many tokens times heads for one call");
  void* args[] = {(void*)&a, (void*)&b, (void*)&scr};
  const void* fn = per == 1 ? store_kernel<1>(cache->head_dim) : store_kernel<kStorePer>(cache->head_dim);
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
