// Attention of a chunk of new tokens over the pages of their sequences.
//   o = sum_j softmax_j(scale q.k_j) v_j over the visible rows j of the token's sequence
// One warp per (token, query head): lane l holds dims 8 l .. (and 256 + 8 l .. for D = 512),
// one pass over the visible rows with the running maximum and sum of the softmax.
#include <cmath>
#include <string>

#include "g4_paged.cuh"

namespace g4 {

struct PaArgs {
  const uint16_t* q;
  long long q_ts, q_hs;
  uint16_t* out;
  long long o_ts, o_hs;
  const uint16_t *kc, *vc;
  long long kp, kr, kh, vp, vr, vh;
  int n_heads, n_kv, window;
  float scale;
};
constexpr int kPaThreads = 256;

__device__ __forceinline__ void pa_unpack8(const uint4 w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}

template <int D>
__global__ void __launch_bounds__(kPaThreads) paged_attn_kernel(const PaArgs a, const PagedBatch b, Scratch* scr) {
  constexpr int C = D / 256;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * (kPaThreads / 32) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / a.n_heads), h = static_cast<int>(unit % a.n_heads);
  if (unit == 0) paged_check_batch(b, lane, scr);
  if (t >= b.n_tokens) return;
  int s = -1;
  for (int s0 = 0; s0 < b.n_seqs && s < 0; s0 += 32) {
    const int i = s0 + lane;
    const bool mine = i < b.n_seqs && b.q_start[i] <= t && t < b.q_start[i + 1];
    const uint32_t hit = __ballot_sync(0xffffffffu, mine);
    if (hit != 0) s = s0 + __ffs(hit) - 1;
  }
  if (s < 0) return;
  bool bad;
  const PagedSeq sq = paged_seq(b, s, &bad);
  const int pos = sq.kv - sq.n + (t - sq.t0);
  const int hk = h / (a.n_heads / a.n_kv);
  float q[C][8], o[C][8] = {}, m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
    pa_unpack8(*reinterpret_cast<const uint4*>(a.q + t * a.q_ts + h * a.q_hs + 256 * c + 8 * lane), q[c]);
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  for (int j = lo; j <= pos; ++j) {
    const int page = b.tables[s * b.table_stride + j / b.page_rows];
    if (page < 0 || page >= b.n_pages) {
      bad = true;
      continue;
    }
    const long long row = j % b.page_rows;
    const uint16_t* kr = a.kc + page * a.kp + row * a.kr + hk * a.kh;
    const uint16_t* vr = a.vc + page * a.vp + row * a.vr + hk * a.vh;
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float k[8];
      pa_unpack8(*reinterpret_cast<const uint4*>(kr + 256 * c + 8 * lane), k);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(q[c][i], k[i], dot);
    }
    dot = warp_sum(dot) * a.scale;
    const float mn = fmaxf(m, dot);
    const float corr = m == -CUDART_INF_F ? 0.f : __expf(m - mn), p = __expf(dot - mn);
    l = l * corr + p;
    m = mn;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v[8];
      pa_unpack8(*reinterpret_cast<const uint4*>(vr + 256 * c + 8 * lane), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[c][i] = fmaf(p, v[i], o[c][i] * corr);
    }
  }
  if (bad && lane == 0) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
    *reinterpret_cast<uint4*>(a.out + t * a.o_ts + h * a.o_hs + 256 * c + 8 * lane) =
        make_uint4(pack_bf16x2(o[c][0] * inv, o[c][1] * inv), pack_bf16x2(o[c][2] * inv, o[c][3] * inv),
                   pack_bf16x2(o[c][4] * inv, o[c][5] * inv), pack_bf16x2(o[c][6] * inv, o[c][7] * inv));
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
  if (!std::isfinite(scale)) return fail(ctx, G4_ERR_BAD_ARG, "scale is not finite");
  if (batch->n_tokens == 0 || batch->n_seqs == 0) return G4_OK;
  if ((st = check_rows(ctx, q, q_token_stride, q_head_stride, "q")) != G4_OK) return st;
  if ((st = check_out_rows(ctx, out, out_token_stride, out_head_stride, batch->n_tokens, n_heads, cache->head_dim,
                           "out")) != G4_OK)
    return st;
  PaArgs a = {q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride, cache->k, cache->v,
              cache->k_page_stride, cache->k_row_stride, cache->k_head_stride, cache->v_page_stride,
              cache->v_row_stride, cache->v_head_stride, n_heads, cache->n_kv_heads, window, scale};
  PagedBatch b = paged_batch(batch, cache);
  Scratch* scr = ctx->buf.scratch;
  const long long warps = static_cast<long long>(batch->n_tokens) * n_heads;
  void* args[] = {(void*)&a, (void*)&b, (void*)&scr};
  const void* fn = cache->head_dim == DS ? (const void*)paged_attn_kernel<DS> : (const void*)paged_attn_kernel<DF>;
  return launch_kernel(ctx, fn, dim3(static_cast<unsigned>((warps + 7) / 8)), dim3(kPaThreads), 0, args, false,
                       "paged attention");
}

}  // extern "C"
