// Beam search's selection: the n_select best (beam, token) of each group by
//   s = scores[beam] + logit - logsumexp(the beam's logits)
//
// A row's order is its logits' order, so one pass over the logits is enough: each block takes a stretch
// of one row, adds up its exponentials beside the running maximum and keeps the stretch's n_select best
// logits; a second kernel, a block per group, joins the sums and picks among the lists by score.
//
// The n_select best of many values, without sorting them: of the best values of disjoint parts (one
// part per thread, or the lists' heads), the n_select-th bounds the answer from below, and every value
// above that bound lies in one of the n_select parts whose best is.  What is left is ranked by
// counting, so results hang on no order of arrival.  Keys (order-preserving logit bits, then
// the inverted index) are all different: equal logits rank by lower token, and the bound is sharp.
#include <string>

#include "g4_internal.h"
#include "g4_common.cuh"

namespace g4 {

constexpr int kBmThreads = 256, kBmJoinThreads = 512;
constexpr int kBmStretch = 65536;  // logits a block may take: 16 bits of index in a key
constexpr int kBmMaxLists = 1024;  // lists of a group (64 beams of 2^20 logits)
constexpr float kBmLog2e = 1.4426950408889634f;

struct BeamSum {  // a stretch's maximum and its sum of exp(l - maximum)
  double sum;
  float top;
};
struct BeamArgs {
  const uint16_t* logits;
  long long group_stride, beam_stride;
  const float* scores;
  int n_beams, vocab, k, stretch, stretches;
  BeamSum* sums;   // [group][beam][stretch]
  uint32_t* keys;  // [group][beam][stretch][k], best first, 0 past a short list's end
  float* out_scores;
  int32_t* out_beams;
  int32_t* out_tokens;
};

// Order-preserving 16 bits of a bf16 (-0 as 0, and none is 0).
__device__ __forceinline__ uint32_t bm_order(uint32_t bits) {
  return (bits & 0x8000u) ? 0x8000u - (bits & 0x7FFFu) : (bits | 0x8000u);
}
__device__ __forceinline__ float bm_logit(uint32_t order) {
  return bf16_to_f32(static_cast<uint16_t>((order & 0x8000u) ? (order & 0x7FFFu) : 0x8000u | (0x8000u - order)));
}
__device__ __forceinline__ uint32_t bm_key(uint32_t bits, int i) { return bm_order(bits) << 16 | (0xFFFFu - i); }
__device__ __forceinline__ uint32_t bm_max2(uint32_t a, uint32_t b) {  // of two bf16 each; a NaN loses
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A thread takes every 256th 16-byte piece of the stretch; what lies before the first 16-byte border and
// behind the last is one element each of the first threads.
//
// What bounds it at many rows: the exponentials (one of the conversion unit's operations a logit) beside the
// bytes; at few, the chain of load, maximum, ranks and the pieces looked at again.
__global__ void __launch_bounds__(kBmThreads) beam_lists_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ uint32_t found[];  // [k * the logits of a thread]
  __shared__ __align__(16) uint32_t keys[kBmThreads];
  __shared__ float red_top[kBmThreads / 32];
  __shared__ double red_sum[kBmThreads / 32];
  __shared__ uint32_t n_found, bound;
  const int tid = threadIdx.x, lane = tid & 31, part = blockIdx.x, beam = blockIdx.y;
  const long long row = static_cast<long long>(blockIdx.z) * a.n_beams + beam;
  const int first = part * a.stretch, n = min(a.stretch, a.vocab - first);
  if (tid == 0) n_found = 0, bound = 1;
  pdl_wait();
  const uint16_t* x = a.logits + blockIdx.z * a.group_stride + beam * a.beam_stride + first;
  const int head = min(n, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / 2);
  const int pieces = (n - head) / 8, tail = head + 8 * pieces;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  // a thread's element outside the body, or none
  auto single = [&](int t) { return t < 8 ? (t < head ? t : -1) : (t < 16 && tail + t - 8 < n ? tail + t - 8 : -1); };

  float m = -CUDART_INF_F, sum = 0.f;
  int at = -1;  // where the first m is: an element, or a piece's first element
  bool whole = false;
  auto raise = [&](float v, int i, bool piece) {
    if (v > m) {
      sum *= exp2f((m - v) * kBmLog2e);  // (-inf - v: 0; never -inf - -inf)
      m = v;
      at = i;
      whole = piece;
    }
  };
  auto take = [&](const uint4& v, int j) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint32_t two = bm_max2(bm_max2(w[0], w[1]), bm_max2(w[2], w[3]));
    const float top = fmaxf(__uint_as_float(two << 16), __uint_as_float(two & 0xFFFF0000u));
    raise(top, head + 8 * j, true);
    if (m == -CUDART_INF_F) {
      if (top != top) sum = top;  // nothing but NaN
      if (at < 0) at = head + 8 * j, whole = true;
      return;
    }
    float more = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      more += exp2f((__uint_as_float(w[e] << 16) - m) * kBmLog2e);
      more += exp2f((__uint_as_float(w[e] & 0xFFFF0000u) - m) * kBmLog2e);
    }
    sum += more;
  };
  const int mine = single(tid);
  if (mine >= 0) {
    const float v = bf16_to_f32(x[mine]);
    raise(v, mine, false);
    if (at < 0) at = mine;
    if (v != -CUDART_INF_F) sum += exp2f((v - m) * kBmLog2e);
  }
  int j = tid;
  for (; j + 3 * kBmThreads < pieces; j += 4 * kBmThreads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __ldg(body + j + u * kBmThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u) take(v[u], j + u * kBmThreads);
  }
  for (; j < pieces; j += kBmThreads) take(__ldg(body + j), j);
  uint32_t best = 0;
  if (at >= 0) {
    if (whole) {  // which of the piece's elements
      int e = 7;
#pragma unroll
      for (int i = 7; i >= 0; --i)
        if (bf16_to_f32(x[at + i]) == m) e = i;
      at += e;
    }
    best = bm_key(__float_as_uint(m) >> 16, at);
  }
  keys[tid] = best;
  // (a NaN has to stay one: nothing here compares sums)
  const float wm = warp_max(m);
  double wide = sum == 0.f ? 0.0 : static_cast<double>(sum) * exp2f((m - wm) * kBmLog2e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
  if (lane == 0) red_top[tid >> 5] = wm, red_sum[tid >> 5] = wide;
  __syncthreads();
  int rank = 0;
#pragma unroll 8
  for (int i = 0; i < kBmThreads; i += 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(keys + i);
    rank += (v.x > best) + (v.y > best) + (v.z > best) + (v.w > best);
  }
  if (rank == a.k - 1 && best != 0u) bound = best;
  __syncthreads();
  const uint32_t least = bound;
  // the pieces of the threads whose best is in, each looked at by its whole warp
  for (uint32_t in = __ballot_sync(0xffffffffu, best >= least); in != 0u; in &= in - 1) {
    const int t = (tid & ~31) + __ffs(in) - 1;
    for (int p = t + lane * kBmThreads; p < pieces; p += 32 * kBmThreads) {
      const uint4 v = __ldg(body + p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = bm_key((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, head + 8 * p + e);
        if (key >= least) found[atomicAdd(&n_found, 1u)] = key;
      }
    }
    const int one = single(t);
    if (lane == 0 && one >= 0) {
      const uint32_t key = bm_key(x[one], one);
      if (key >= least) found[atomicAdd(&n_found, 1u)] = key;
    }
  }
  __syncthreads();
  const int have = n_found;
  const long long list = row * a.stretches + part;
  for (int i = tid; i < have; i += kBmThreads) {
    int above = 0;
    for (int o = 0; o < have && above < a.k; ++o) above += found[o] > found[i];
    if (above < a.k) a.keys[list * a.k + above] = found[i];
  }
  if (tid >= have && tid < a.k) a.keys[list * a.k + tid] = 0u;
  if (tid == 0) {
    float top = -CUDART_INF_F;
    double total = 0.0;
    for (int w = 0; w < kBmThreads / 32; ++w) top = fmaxf(top, red_top[w]);
    for (int w = 0; w < kBmThreads / 32; ++w)
      if (!(red_sum[w] == 0.0)) total += red_sum[w] * exp2f((red_top[w] - top) * kBmLog2e);
    a.sums[list] = {total, top};
  }
}

// What is compared: the score, then the lower beam, the higher logit (scores that 64 bits cannot tell
// apart), the lower token.
struct BeamItem {
  double score;
  uint64_t rest;  // beam inverted : 16 | logit order : 16 | token inverted : 32
};
__device__ __forceinline__ bool bm_above(const BeamItem& a, const BeamItem& b) {
  return a.score > b.score || (a.score == b.score && a.rest > b.rest);
}
__device__ __forceinline__ BeamItem bm_item(const BeamArgs& a, double base, int beam, int part, uint32_t key) {
  const uint32_t token = part * a.stretch + (0xFFFFu - (key & 0xFFFFu));
  const bool none = base == -CUDART_INF;  // no order of logits among the continuations of such a beam
  return {none ? base : base + static_cast<double>(bm_logit(key >> 16)),
          static_cast<uint64_t>(0xFFFFu - beam) << 48 | static_cast<uint64_t>(none ? 0u : key >> 16) << 32 |
              (0xFFFFFFFFu - token)};
}

__global__ void __launch_bounds__(kBmJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  BeamItem* heads = reinterpret_cast<BeamItem*>(raw);            // [lists]
  BeamItem* found = heads + kBmMaxLists;                         // [k * k]
  __shared__ double base[G4_BEAM_MAX];
  __shared__ BeamItem bound;
  __shared__ uint32_t n_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row0 = static_cast<long long>(blockIdx.x) * a.n_beams;
  const int lists = a.n_beams * a.stretches;
  if (tid == 0) {
    n_found = 0;
    bound = {-CUDART_INF, 0ull};
  }
  pdl_wait();
  // base = scores[beam] - logsumexp, -inf for a beam that does not count
  for (int b = warp; b < a.n_beams; b += kBmJoinThreads / 32) {
    const BeamSum* st = a.sums + (row0 + b) * a.stretches;
    float top = -CUDART_INF_F;
    for (int i = lane; i < a.stretches; i += 32) top = fmaxf(top, st[i].top);
    top = warp_max(top);
    double total = 0.0;
    for (int i = lane; i < a.stretches; i += 32)
      if (!(st[i].sum == 0.0)) total += st[i].sum * exp(static_cast<double>(st[i].top) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      const double v = static_cast<double>(a.scores[row0 + b]) - (static_cast<double>(top) + log(total));
      base[b] = isfinite(v) ? v : -CUDART_INF;
    }
  }
  __syncthreads();
  // (a beam that does not count has one list, its first k tokens)
  auto list_key = [&](int list, int i) -> uint32_t {
    const int beam = list / a.stretches, part = list % a.stretches;
    if (base[beam] != -CUDART_INF) return a.keys[(row0 * a.stretches + list) * a.k + i];
    return part == 0 && i < min(a.vocab, a.k) ? 0x10000u | (0xFFFFu - i) : 0u;
  };
  for (int i = tid; i < lists; i += kBmJoinThreads) {
    const uint32_t key = list_key(i, 0);
    const int beam = i / a.stretches;
    heads[i] = key ? bm_item(a, base[beam], beam, i % a.stretches, key) : BeamItem{-CUDART_INF, 0ull};
  }
  __syncthreads();
  for (int i = tid; i < lists; i += kBmJoinThreads) {
    if (heads[i].rest == 0ull) continue;
    int rank = 0;
    for (int j = 0; j < lists; ++j) rank += bm_above(heads[j], heads[i]);
    if (rank == a.k - 1) bound = heads[i];
  }
  __syncthreads();
  for (int c = tid; c < lists * a.k; c += kBmJoinThreads) {
    const int list = c / a.k;
    if (heads[list].rest == 0ull || bm_above(bound, heads[list])) continue;
    const uint32_t key = list_key(list, c % a.k);
    if (key == 0u) continue;
    const int beam = list / a.stretches;
    const BeamItem item = bm_item(a, base[beam], beam, list % a.stretches, key);
    if (!bm_above(bound, item)) found[atomicAdd(&n_found, 1u)] = item;
  }
  __syncthreads();
  const int have = n_found;
  for (int i = tid; i < have; i += kBmJoinThreads) {
    int rank = 0;
    for (int j = 0; j < have && rank < a.k; ++j) rank += bm_above(found[j], found[i]);
    if (rank < a.k) {
      const long long at = static_cast<long long>(blockIdx.x) * a.k + rank;
      a.out_scores[at] = static_cast<float>(found[i].score);
      a.out_beams[at] = 0xFFFF - static_cast<int>(found[i].rest >> 48);
      a.out_tokens[at] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(found[i].rest));
    }
  }
}

}  // namespace g4

using namespace g4;

extern "C" g4_status g4_beam_select(g4_ctx* ctx, const g4_bf16* logits, int64_t group_stride, int64_t beam_stride,
                                    const float* scores, int n_groups, int n_beams, int vocab, int n_select,
                                    float* out_scores, int32_t* out_beams, int32_t* out_tokens) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  if (n_groups < 0 || n_beams < 1 || n_beams > G4_BEAM_MAX || vocab < 1 || vocab > (1 << 20) || n_select < 1 ||
      n_select > G4_BEAM_MAX || n_select > static_cast<long long>(n_beams) * vocab)
    return fail(ctx, G4_ERR_BAD_ARG, "beam_select: n_groups, n_beams, vocab or n_select out of range");
  if (n_groups == 0) return G4_OK;
  const int64_t most = int64_t(1) << 38;
  if ((n_groups > 1 && (group_stride < 0 || group_stride > most)) || (n_beams > 1 && (beam_stride < 0 || beam_stride > most)))
    return fail(ctx, G4_ERR_BAD_ARG, "beam_select: a stride is negative or too large");
  if (logits == nullptr || (reinterpret_cast<uintptr_t>(logits) & 1u))
    return fail(ctx, G4_ERR_BAD_ARG, "beam_select: logits is null or misaligned");
  const void* words[] = {scores, out_scores, out_beams, out_tokens};
  for (const void* p : words)
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 3u))
      return fail(ctx, G4_ERR_BAD_ARG, "beam_select: scores or an output is null or misaligned");
  DeviceGuard on(ctx);
  const long long rows = static_cast<long long>(n_groups) * n_beams;
  BeamArgs a = {logits, n_groups > 1 ? group_stride : 0, n_beams > 1 ? beam_stride : 0, scores, n_beams, vocab, n_select,
                0, 0, nullptr, nullptr, out_scores, out_beams, out_tokens};
  // stretches of a row: enough blocks to fill the device, none of few logits, within both limits
  const int least = (vocab + kBmStretch - 1) / kBmStretch, useful = (vocab + 4095) / 4096;
  const long long fill = (4ll * ctx->sm_count + rows - 1) / rows;
  int parts = fill < useful ? static_cast<int>(fill) : useful;
  if (parts > kBmMaxLists / n_beams) parts = kBmMaxLists / n_beams;
  if (parts < least) parts = least;  // (at most 16: kBmMaxLists / 64)
  a.stretch = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  a.stretches = (vocab + a.stretch - 1) / a.stretch;
  const size_t lists = static_cast<size_t>(n_beams) * a.stretches;
  const size_t bytes = lists * (sizeof(BeamSum) + 4 * n_select);
  const size_t list_smem = 4 * static_cast<size_t>(n_select) * (8 * ((a.stretch / 8 + kBmThreads - 1) / kBmThreads) + 1);
  const size_t join_smem = sizeof(BeamItem) * (kBmMaxLists + static_cast<size_t>(n_select) * n_select);
  g4_status st = allow_max_dynamic_smem(ctx, (const void*)beam_lists_kernel, list_smem, "beam lists");
  if (st == G4_OK) st = allow_max_dynamic_smem(ctx, (const void*)beam_join_kernel, join_smem, "beam join");
  // as many groups at a time as the context's lists have room for
  const long long at_once = kBeamWords * 8 / bytes < 65535 ? kBeamWords * 8 / bytes : 65535;
  for (long long done = 0; done < n_groups && st == G4_OK; done += at_once) {
    const int n = static_cast<int>(n_groups - done < at_once ? n_groups - done : at_once);
    a.logits = logits + done * a.group_stride;
    a.scores = scores + done * n_beams;
    a.out_scores = out_scores + done * n_select;
    a.out_beams = out_beams + done * n_select;
    a.out_tokens = out_tokens + done * n_select;
    a.sums = reinterpret_cast<BeamSum*>(ctx->buf.beam);
    a.keys = reinterpret_cast<uint32_t*>(a.sums + n * lists);
    void* args[] = {(void*)&a};
    st = launch_kernel(ctx, (const void*)beam_lists_kernel, dim3(a.stretches, n_beams, n), dim3(kBmThreads), list_smem,
                       args, false, "beam lists");
    if (st == G4_OK)
      st = launch_kernel(ctx, (const void*)beam_join_kernel, dim3(n), dim3(kBmJoinThreads), join_smem, args, false,
                         "beam join");
  }
  return st;
}
