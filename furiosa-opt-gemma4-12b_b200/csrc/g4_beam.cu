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
constexpr int kBmQuads = 16;       // up to as many selected, four threads are a part
constexpr int kBmNear = 8192;      // keys of a group that are copied to shared memory
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
__device__ __forceinline__ float bm_exp2(float x) {  // x <= 0 (or next to it): what underflows counts for nothing
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float bm_exp(float x) { return bm_exp2(x * kBmLog2e); }
__device__ __forceinline__ uint32_t bm_max2(uint32_t a, uint32_t b) {  // of two bf16 each; a NaN stays one
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
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
  __shared__ uint32_t n_found, n_who, bound;
  __shared__ uint8_t who[kBmThreads];
  const int tid = threadIdx.x, lane = tid & 31, part = blockIdx.x, beam = blockIdx.y;
  const long long row = static_cast<long long>(blockIdx.z) * a.n_beams + beam;
  const int first = part * a.stretch, n = min(a.stretch, a.vocab - first);
  if (tid == 0) n_found = 0, n_who = 0, bound = 1;
  pdl_wait();
  const uint16_t* x = a.logits + blockIdx.z * a.group_stride + beam * a.beam_stride + first;
  const int head = min(n, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / 2);
  const int pieces = (n - head) / 8, tail = head + 8 * pieces;
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  // a thread's element outside the body, or none
  auto single = [&](int t) { return t < 8 ? (t < head ? t : -1) : (t < 16 && tail + t - 8 < n ? tail + t - 8 : -1); };

  float m = -CUDART_INF_F, sum = 0.f;
  int at = -1;  // where the first m is: an element, or the first of four pieces
  bool whole = false;
  // The sum is of 2^(l log2 e - ref), one FMA a logit, where ref is m log2 e rounded to f32: what the rounding
  // took is put back (in 64 bits) when the sum leaves the thread.  Where m is beyond 2^100 (rows masked with
  // the lowest number there is) ref might not be finite: the difference to m comes first there.
  float ref = 0.f;
  auto far = [](float v) { return fabsf(v) > 0x1p100f; };
  auto raise = [&](float v, int i, bool pieces_of_it) {
    if (v > m) {
      const float to = v * kBmLog2e;
      if (m != -CUDART_INF_F) sum *= far(m) || far(v) ? bm_exp(m - v) : bm_exp2(ref - to);
      ref = to;
      m = v;
      at = i;
      whole = pieces_of_it;
    } else if (at < 0) {  // (nothing but -inf so far)
      at = i;
      whole = pieces_of_it;
    }
    if (v != v) sum = v;
  };
  const int mine = single(tid);
  if (mine >= 0) {
    const float v = bf16_to_f32(x[mine]);
    raise(v, mine, false);
    if (m != -CUDART_INF_F) sum += bm_exp(v - m);
  }
  // four pieces are on their way while four are looked at; what is not there counts as -inf
  uint4 now[4], next[4];
  auto fetch = [&](uint4 (&v)[4], int j) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t none = 0xFF80FF80u;
      v[u] = j + u * kBmThreads < pieces ? __ldg(body + j + u * kBmThreads) : make_uint4(none, none, none, none);
    }
  };
  fetch(now, tid);
  for (int j = tid; j < pieces; j += 4 * kBmThreads) {
    fetch(next, j + 4 * kBmThreads);
    uint32_t two = bm_max2(bm_max2(now[0].x, now[0].y), bm_max2(now[0].z, now[0].w));
#pragma unroll
    for (int u = 1; u < 4; ++u)
      two = bm_max2(two, bm_max2(bm_max2(now[u].x, now[u].y), bm_max2(now[u].z, now[u].w)));
    const uint32_t both = bm_max2(two, __byte_perm(two, 0, 0x1032));
    raise(__uint_as_float(both << 16), j, true);
    if (far(m) && m != -CUDART_INF_F) {
      for (int u = 0; u < 4; ++u)
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = e == 0 ? now[u].x : e == 1 ? now[u].y : e == 2 ? now[u].z : now[u].w;
          sum += bm_exp(__uint_as_float(w << 16) - m) + bm_exp(__uint_as_float(w & 0xFFFF0000u) - m);
        }
    } else if (m != -CUDART_INF_F) {
      const float2 scale = make_float2(kBmLog2e, kBmLog2e), off = make_float2(-ref, -ref);
      float2 more[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t w[4] = {now[u].x, now[u].y, now[u].z, now[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x2 =
              fma_f32x2(make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u)), scale, off);
          more[e & 1] = add_f32x2(more[e & 1], make_float2(bm_exp2(x2.x), bm_exp2(x2.y)));
        }
      }
      more[0] = add_f32x2(more[0], more[1]);
      sum += more[0].x + more[0].y;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) now[u] = next[u];
  }
  pdl_launch_dependents();  // (the join waits for all of this kernel)
  uint32_t best = 0;
  if (at >= 0) {
    if (whole) {  // which of the four pieces' elements
      const int j = at;
      at = -1;
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const int p = j + u * kBmThreads;
        if (p >= pieces) continue;
        const uint4 v = __ldg(body + p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if (__uint_as_float((w[e >> 1] >> (16 * (e & 1))) << 16) == m) at = head + 8 * p + e;
      }
    }
    if (at >= 0) best = bm_key(__float_as_uint(m) >> 16, at);  // (none: all are NaN)
  }
  // parts of a thread each, or of four where so few are wanted that ranking a quarter of the parts does
  const int parts = a.k <= kBmQuads ? kBmThreads / 4 : kBmThreads;
  uint32_t part_best = best;
  if (a.k <= kBmQuads) {
    part_best = max(part_best, __shfl_xor_sync(0xffffffffu, part_best, 1));
    part_best = max(part_best, __shfl_xor_sync(0xffffffffu, part_best, 2));
    if ((tid & 3) == 0) keys[tid >> 2] = part_best;
  } else {
    keys[tid] = part_best;
  }
  // (a NaN has to stay one: nothing here compares sums)
  const float wm = warp_max(m);
  const double lost = far(m) ? 0.0 : (static_cast<double>(ref) - static_cast<double>(m) * kBmLog2e) * 0.6931471805599453;
  double wide = sum == 0.f ? 0.0 : static_cast<double>(sum) * (1.0 + lost) * bm_exp(m - wm);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
  if (lane == 0) red_top[tid >> 5] = wm, red_sum[tid >> 5] = wide;
  __syncthreads();
  if (tid < parts) {
    const uint32_t key = keys[tid];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < parts; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(keys + i);
      rank += (v.x > key) + (v.y > key) + (v.z > key) + (v.w > key);
    }
    if (rank == a.k - 1 && key != 0u) bound = key;
  }
  __syncthreads();
  const uint32_t least = bound;
  // the threads whose best is in, and then all of their pieces by all threads
  if (best >= least) who[atomicAdd(&n_who, 1u)] = static_cast<uint8_t>(tid);
  __syncthreads();
  const int turns = (pieces + kBmThreads - 1) / kBmThreads + 1;  // pieces of a thread, and the element outside
  for (int c = tid; c < static_cast<int>(n_who) * turns; c += kBmThreads) {
    const int q = c / turns, turn = c - q * turns, t = who[q], p = t + turn * kBmThreads;
    if (turn == turns - 1) {
      const int one = single(t);
      if (one < 0) continue;
      const uint32_t key = bm_key(x[one], one);
      if (key >= least) found[atomicAdd(&n_found, 1u)] = key;
    } else if (p < pieces) {
      const uint4 v = __ldg(body + p);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      // (most pieces have nothing: their largest says so)
      const uint32_t two = bm_max2(bm_max2(w[0], w[1]), bm_max2(w[2], w[3]));
      if (max(bm_order(two & 0xFFFFu), bm_order(two >> 16)) < least >> 16) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = bm_key((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, head + 8 * p + e);
        if (key >= least) found[atomicAdd(&n_found, 1u)] = key;
      }
    }
  }
  __syncthreads();
  const int have = n_found;
  const long long list = row * a.stretches + part;
  for (int i = tid; i < have; i += kBmThreads) {
    int above = 0;
#pragma unroll 4
    for (int o = 0; o < have; ++o) above += found[o] > found[i];
    if (above < a.k) a.keys[list * a.k + above] = found[i];
  }
  if (tid >= have && tid < a.k) a.keys[list * a.k + tid] = 0u;
  if (tid < kBmThreads / 32) {
    constexpr uint32_t kAll = (1u << (kBmThreads / 32)) - 1;
    const float mine_top = red_top[tid];
    float top = mine_top;
#pragma unroll
    for (int o = kBmThreads / 64; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    double total = red_sum[tid];
    if (!(total == 0.0)) total *= bm_exp(mine_top - top);
#pragma unroll
    for (int o = kBmThreads / 64; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    if (tid == 0) a.sums[list] = {total, top};
  }
}

// What is compared: the score, then the lower beam, the higher logit (scores that 64 bits cannot tell
// apart), the lower token.
struct BeamItem {
  uint64_t score;  // order-preserving bits of the f64
  uint64_t rest;   // beam inverted : 16 | logit order : 16 | token inverted : 32 (never 0)
};
__device__ __forceinline__ uint64_t bm_bits(double s) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(s + 0.0));  // (-0 as 0)
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double bm_score(uint64_t bits) {
  return __longlong_as_double(static_cast<long long>((bits >> 63) ? bits & ~(1ull << 63) : ~bits));
}
__device__ __forceinline__ bool bm_above(const BeamItem& a, const BeamItem& b) {
  return a.score > b.score || (a.score == b.score && a.rest > b.rest);
}
struct BeamBase {  // of a beam: its largest logit, and scores[beam] - log sum exp(l - largest), -inf if it does not count
  double top, rest;
};
__device__ __forceinline__ BeamItem bm_item(const BeamArgs& a, const BeamBase& base, int beam, int part, uint32_t key) {
  const uint32_t token = part * a.stretch + (0xFFFFu - (key & 0xFFFFu));
  const bool none = base.rest == -CUDART_INF;  // no order of logits among the continuations of such a beam
  return {bm_bits(none ? base.rest : base.rest + (static_cast<double>(bm_logit(key >> 16)) - base.top)),
          static_cast<uint64_t>(0xFFFFu - beam) << 48 | static_cast<uint64_t>(none ? 0u : key >> 16) << 32 |
              (0xFFFFFFFFu - token)};
}

__global__ void __launch_bounds__(kBmJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  BeamItem* heads = reinterpret_cast<BeamItem*>(raw);              // [kBmMaxLists]
  BeamItem* found = heads + kBmMaxLists;                           // [k * k]
  uint32_t* near = reinterpret_cast<uint32_t*>(found + a.k * a.k);  // the lists' keys where they have room
  __shared__ BeamBase base[G4_BEAM_MAX];
  __shared__ int in[G4_BEAM_MAX];  // the lists whose heads are among the k best
  __shared__ uint32_t n_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row0 = static_cast<long long>(blockIdx.x) * a.n_beams;
  const int lists = a.n_beams * a.stretches;
  if (tid == 0) n_found = 0;
  if (tid < a.k) in[tid] = -1;
  pdl_wait();
  const uint32_t* keys = a.keys + row0 * a.stretches * a.k;
  if (lists * a.k <= kBmNear) {
    for (int i = tid; i < lists * a.k; i += kBmJoinThreads) near[i] = keys[i];
    keys = near;
  }
  for (int b = warp; b < a.n_beams; b += kBmJoinThreads / 32) {
    const BeamSum* st = a.sums + (row0 + b) * a.stretches;
    const float score = a.scores[row0 + b];
    float top = -CUDART_INF_F;
    for (int i = lane; i < a.stretches; i += 32) top = fmaxf(top, st[i].top);
    top = warp_max(top);
    double total = 0.0;
    for (int i = lane; i < a.stretches; i += 32)
      if (!(st[i].sum == 0.0)) total += st[i].sum * exp(static_cast<double>(st[i].top) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      const double v = static_cast<double>(score) - log(total);
      base[b] = {static_cast<double>(top), isfinite(v) && isfinite(top) ? v : -CUDART_INF};
    }
  }
  __syncthreads();
  // (a beam that does not count has one list, its first k tokens)
  auto key_of = [&](int beam, int part, int i, uint32_t key) -> uint32_t {
    if (base[beam].rest != -CUDART_INF) return key;
    return part == 0 && i < a.vocab ? 0x10000u | (0xFFFFu - i) : 0u;
  };
  for (int i = tid; i < lists; i += kBmJoinThreads) {
    const int beam = i / a.stretches, part = i - beam * a.stretches;
    const uint32_t key = key_of(beam, part, 0, keys[i * a.k]);
    heads[i] = key ? bm_item(a, base[beam], beam, part, key) : BeamItem{0ull, 0ull};
  }
  __syncthreads();
  // `each` threads, neighbours of one warp, rank a head
  int each = 32;
  while (each > 1 && each * lists > kBmJoinThreads) each >>= 1;
  for (int i0 = 0; i0 < lists; i0 += kBmJoinThreads / each) {
    const int i = i0 + tid / each;
    const BeamItem mine = i < lists ? heads[i] : BeamItem{0ull, 0ull};
    int rank = 0;
    if (mine.rest != 0ull) {
#pragma unroll 4
      for (int j = tid & (each - 1); j < lists; j += each) rank += bm_above(heads[j], mine);
    }
    for (int o = 1; o < each; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if ((tid & (each - 1)) == 0 && mine.rest != 0ull && rank < a.k) in[rank] = i;
  }
  __syncthreads();
  // nothing below the last head that is in can be (with fewer lists than that, everything can)
  const int last = in[a.k - 1];
  const BeamItem bound = last >= 0 ? heads[last] : BeamItem{0ull, 0ull};
  for (int c = tid; c < a.k * a.k; c += kBmJoinThreads) {
    const int list = in[c / a.k], i = c % a.k;
    if (list < 0) continue;
    const int beam = list / a.stretches, part = list - beam * a.stretches;
    const uint32_t key = key_of(beam, part, i, keys[list * a.k + i]);
    if (key == 0u) continue;
    const BeamItem item = bm_item(a, base[beam], beam, part, key);
    if (!bm_above(bound, item)) found[atomicAdd(&n_found, 1u)] = item;
  }
  __syncthreads();
  const int have = n_found;
  for (int i = tid; i < have; i += kBmJoinThreads) {
    const BeamItem mine = found[i];
    int rank = 0;
    for (int j = 0; j < have && rank < a.k; ++j) rank += bm_above(found[j], mine);
    if (rank < a.k) {
      const long long at = static_cast<long long>(blockIdx.x) * a.k + rank;
      a.out_scores[at] = static_cast<float>(bm_score(mine.score));
      a.out_beams[at] = 0xFFFF - static_cast<int>(mine.rest >> 48);
      a.out_tokens[at] = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(mine.rest));
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
  // Stretches of a row: more of them keep the SMs busier, fewer leave the join less.  Of 262144 logits, one row
  // takes 7.6 us in 32 stretches (8.2 in 16), 4 rows 9.3 in 16 (10.6 in 8 and in 32), 64 rows 18.4 in 8 (20.6 in
  // 16), 128 rows 26.4 in 4 (27.9 in 8); 4 rows of 32000 8.5 in 16 (10.2 in 4).
  const int least = (vocab + kBmStretch - 1) / kBmStretch, useful = (vocab + 2047) / 2048;
  int parts = rows <= 2 ? 32 : rows <= 32 ? 16 : rows < 96 ? 8 : 4;
  if (parts > useful) parts = useful;
  if (parts > kBmMaxLists / n_beams) parts = kBmMaxLists / n_beams;
  if (parts < least) parts = least;  // (at most 16: kBmMaxLists / 64)
  a.stretch = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  a.stretches = (vocab + a.stretch - 1) / a.stretch;
  const size_t lists = static_cast<size_t>(n_beams) * a.stretches;
  const size_t bytes = lists * (sizeof(BeamSum) + 4 * n_select);
  const size_t list_smem = 4 * static_cast<size_t>(n_select) * (8 * ((a.stretch / 8 + kBmThreads - 1) / kBmThreads) + 1) *
                            (n_select <= kBmQuads ? 4 : 1);
  const size_t join_smem = sizeof(BeamItem) * (kBmMaxLists + static_cast<size_t>(n_select) * n_select) +
                           (lists * n_select <= kBmNear ? 4 * lists * n_select : 0);
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
