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
// the inverted index) are all different: equal logits rank by lower token.
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
  uint32_t room, room_groups;  // of a stretch's candidates, and of its groups that may have some
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

// A stretch as its block's threads take it: every kBmThreads-th 16-byte piece, four of them (a group) at a time;
// what lies before the first 16-byte border and behind the last is one element each of the first threads.
struct BmStretch {
  const uint16_t* x;
  int n, head, pieces, groups, tail;
  __device__ __forceinline__ const uint4* body() const { return reinterpret_cast<const uint4*>(x + head); }
  // a thread's element before the body or behind it, or none
  __device__ __forceinline__ int before(int t) const { return t < head ? t : -1; }
  __device__ __forceinline__ int behind(int t) const { return tail + t < n ? tail + t : -1; }
};
constexpr int kBmGroups = kBmStretch / (32 * kBmThreads);
constexpr uint32_t kBmOf = 31u;  // a group's place in a key: earlier groups hold lower tokens
struct BmShared {
  __align__(16) uint32_t keys[kBmThreads];
  uint16_t most[kBmGroups][kBmThreads];  // the largest of each thread's groups
  uint32_t n_groups, n_found, bound;
};
// Value and place, comparable.
__device__ __forceinline__ uint32_t bm_place(uint32_t bits, int group) { return bm_order(bits) << 8 | (kBmOf - group); }

// The k-th of the parts' best keys (all different; 0: none), 1 if there are fewer.  Parts are a thread each, or
// four where so few are wanted that ranking a quarter of the parts does.
__device__ __forceinline__ uint32_t bm_bound(BmShared& s, int k, uint32_t best) {
  const int tid = threadIdx.x;
  int parts = kBmThreads;
  if (k <= kBmQuads) {
    parts = kBmThreads / 4;
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 1));
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 2));
    if ((tid & 3) == 0) s.keys[tid >> 2] = best;
  } else {
    s.keys[tid] = best;
  }
  __syncthreads();
  if (tid < parts) {
    const uint32_t key = s.keys[tid];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < parts; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(s.keys + i);
      rank += (v.x > key) + (v.y > key) + (v.z > key) + (v.w > key);
    }
    if (rank == k - 1 && key != 0u) s.bound = key;
  }
  __syncthreads();
  return s.bound;
}

__device__ __forceinline__ uint32_t bm_max8(const uint4& v) { return bm_max2(bm_max2(v.x, v.y), bm_max2(v.z, v.w)); }

// Calls f(bits, index) for each element of a piece.
template <class F>
__device__ __forceinline__ void bm_each(const uint4& v, int i, F f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) f((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu, i + e);
}

// The candidates where too many groups reach the bound `least` (a place, of values that are all alike): the best
// key of each thread's groups that do, the bound of those, and what reaches that one.
__device__ __noinline__ void bm_again(BmShared& s, const BmStretch& r, int k, uint32_t least, uint32_t* found) {
  const int tid = threadIdx.x;
  auto each = [&](auto f) {
    const int one[2] = {r.before(tid), r.behind(tid)};
    for (int o = 0; o < 2; ++o)
      if (one[o] >= 0 && bm_place(r.x[one[o]], o == 0 ? 0 : static_cast<int>(kBmOf)) >= least) f(r.x[one[o]], one[o]);
    for (int g = 0; g < r.groups; ++g) {
      if (bm_place(s.most[g][tid], g) < least) continue;
      for (int p = tid + 4 * g * kBmThreads; p < min(r.pieces, 4 * (g + 1) * kBmThreads); p += kBmThreads)
        bm_each(__ldg(r.body() + p), r.head + 8 * p, f);
    }
  };
  uint32_t best = 0;
  each([&](uint32_t bits, int i) { best = max(best, bm_key(bits, i)); });
  __syncthreads();
  if (tid == 0) s.n_found = 0, s.bound = 1;
  const uint32_t sharp = bm_bound(s, k, best);
  if (best >= sharp)
    each([&](uint32_t bits, int i) {
      if (bm_key(bits, i) >= sharp) found[atomicAdd(&s.n_found, 1u)] = bm_key(bits, i);
    });
  __syncthreads();
}

// One pass: sums, and the largest value of each thread's groups.  Of the threads' largest (with the group where
// they first come) the k-th is the bound, and the few groups that reach it are looked at again.
//
// What bounds it at many rows (18 us of 128 x 262144, 3.7 TB/s): the bytes and the exponentials, 16 us with the first
// loads' latency and SMs that have four blocks where others have three; bounds, second look and ranks are 2 us behind
// them.  (Collecting candidates as they pass, above the bound of the first group, takes 21 us; finding each thread's
// best exactly first, and then looking through all of the best threads' pieces, 21 us.)  At few rows: the
// chain of latencies, 4.6 us of 4 x 262144.
__global__ void __launch_bounds__(kBmThreads) beam_lists_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ uint32_t shared[];
  __shared__ BmShared s;
  __shared__ float red_top[kBmThreads / 32];
  __shared__ double red_sum[kBmThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, part = blockIdx.x, beam = blockIdx.y;
  const long long row = static_cast<long long>(blockIdx.z) * a.n_beams + beam;
  const int first = part * a.stretch;
  if (tid == 0) s.n_groups = 0, s.n_found = 0, s.bound = 1;
  pdl_wait();
  BmStretch r;
  r.x = a.logits + blockIdx.z * a.group_stride + beam * a.beam_stride + first;
  r.n = min(a.stretch, a.vocab - first);
  r.head = min(r.n, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(r.x) & 15u)) & 15u) / 2);
  r.pieces = (r.n - r.head) / 8;
  r.groups = (r.pieces + 4 * kBmThreads - 1) / (4 * kBmThreads);
  r.tail = r.head + 8 * r.pieces;
  const uint4* body = r.body();
  const int pieces = r.pieces;

  const int lo = r.before(tid), hi = r.behind(tid);
  float m = -CUDART_INF_F, sum = 0.f;
  // The group where m first is.  What raises it is above -inf: a thread of nothing else has its first element's, so
  // that what the thread stands for in the bound is an element that reaches it.
  int in = tid < pieces || lo >= 0 ? 0 : static_cast<int>(kBmOf);
  // The sum is of 2^((l - m) log2 e) as 2^(fma(l, log2 e, -ref) - rest), where ref is m log2 e rounded to f32 and rest
  // what the rounding took: m itself counts as 1 exactly.  Where m is beyond 2^100 (rows masked with the lowest
  // number there is) ref might not be finite: the difference to m comes first there.
  float ref = 0.f, rest = 0.f;
  auto far = [](float v) { return fabsf(v) > 0x1p100f; };
  auto raise = [&](float v, int group) {
    if (v > m) {
      if (m != -CUDART_INF_F) sum *= bm_exp(m - v);
      ref = v * kBmLog2e;
      rest = fmaf(v, kBmLog2e, -ref);
      m = v;
      in = group;
    }
    if (v != v) sum = v;
  };
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
  const uint32_t lo_bits = lo >= 0 ? r.x[lo] : 0xFF80u, hi_bits = hi >= 0 ? r.x[hi] : 0xFF80u;
  if (lo >= 0) {
    const float v = __uint_as_float(lo_bits << 16);
    raise(v, 0);
    if (m != -CUDART_INF_F) sum += bm_exp(v - m);
  }
  for (int g = 0, j = tid; j < pieces; ++g, j += 4 * kBmThreads) {
    fetch(next, j + 4 * kBmThreads);
    uint32_t two = bm_max8(now[0]);
#pragma unroll
    for (int u = 1; u < 4; ++u) two = bm_max2(two, bm_max8(now[u]));
    const uint32_t both = bm_max2(two, __byte_perm(two, 0, 0x1032));
    s.most[g][tid] = static_cast<uint16_t>(both);
    raise(__uint_as_float(both << 16), g);
    if (far(m) && m != -CUDART_INF_F) {
      for (int u = 0; u < 4; ++u)
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = e == 0 ? now[u].x : e == 1 ? now[u].y : e == 2 ? now[u].z : now[u].w;
          sum += bm_exp(__uint_as_float(w << 16) - m) + bm_exp(__uint_as_float(w & 0xFFFF0000u) - m);
        }
    } else if (m != -CUDART_INF_F) {
      const float2 scale = make_float2(kBmLog2e, kBmLog2e), off = make_float2(-ref, -ref),
                   less = make_float2(-rest, -rest);
      float2 more[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t w[4] = {now[u].x, now[u].y, now[u].z, now[u].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 l2 = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u));
          const float2 x2 = add_f32x2(fma_f32x2(l2, scale, off), less);
          more[e & 1] = add_f32x2(more[e & 1], make_float2(bm_exp2(x2.x), bm_exp2(x2.y)));
        }
      }
      more[0] = add_f32x2(more[0], more[1]);
      sum += more[0].x + more[0].y;
    }
    if (j + 4 * kBmThreads >= pieces) break;  // (the last group stays)
#pragma unroll
    for (int u = 0; u < 4; ++u) now[u] = next[u];
  }
  pdl_launch_dependents();  // (the join waits for all of this kernel)
  if (hi >= 0) {
    const float v = __uint_as_float(hi_bits << 16);
    raise(v, static_cast<int>(kBmOf));
    if (m != -CUDART_INF_F) sum += bm_exp(v - m);
  }
  const bool any = tid < pieces || lo >= 0 || hi >= 0;
  const uint32_t best = any ? bm_place(__float_as_uint(m) >> 16, in) << 8 | (0xFFu - tid) : 0u;
  const uint32_t least = bm_bound(s, a.k, best) >> 8;
  uint32_t* found = shared;
  uint16_t* which = reinterpret_cast<uint16_t*>(found + a.room);  // groups: place in the stretch : 8 | thread : 8
  auto take = [&](uint32_t bits, int i) {
    const uint32_t at = atomicAdd(&s.n_found, 1u);
    if (at < a.room) found[at] = bm_key(bits, i);
  };
  if (lo >= 0 && bm_place(lo_bits, 0) >= least) take(lo_bits, lo);
  if (hi >= 0 && bm_place(hi_bits, static_cast<int>(kBmOf)) >= least) take(hi_bits, hi);
  auto look = [&](const uint4& v, int p, int g) {
    const uint32_t two = bm_max8(v);  // (most pieces have nothing: their largest says so)
    if (max(bm_place(two & 0xFFFFu, g), bm_place(two >> 16, g)) < least) return;
    bm_each(v, r.head + 8 * p, [&](uint32_t bits, int at) {
      if (bm_place(bits, g) >= least) take(bits, at);
    });
  };
  const bool mine = best >> 8 >= least;  // (no group of a thread's is above its best)
  if (r.groups > 1) {
    if (mine)
      for (int g = 0, j = tid; j < pieces; ++g, j += 4 * kBmThreads)
        if (bm_place(s.most[g][tid], g) >= least) {
          const uint32_t at = atomicAdd(&s.n_groups, 1u);
          if (at < a.room_groups) which[at] = static_cast<uint16_t>(g << 8 | tid);
        }
    __syncthreads();
  } else if (mine) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (tid + u * kBmThreads < pieces) look(now[u], tid + u * kBmThreads, 0);
  }
  // (the sums are joined while the first of the pieces comes back)
  const int again = s.n_groups <= a.room_groups ? 4 * s.n_groups : 0;
  auto piece = [&](int i, int& g) {
    g = which[i >> 2] >> 8;
    return (which[i >> 2] & 0xFF) + (4 * g + (i & 3)) * kBmThreads;
  };
  int g0 = 0, p0 = tid < again ? piece(tid, g0) : pieces;
  if (p0 < pieces) now[0] = __ldg(body + p0);
  // (a NaN has to stay one: nothing here compares sums)
  const float wm = warp_max(m);
  double wide = sum == 0.f ? 0.0 : static_cast<double>(sum) * bm_exp(m - wm);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wide += __shfl_xor_sync(0xffffffffu, wide, o);
  if (lane == 0) red_top[tid >> 5] = wm, red_sum[tid >> 5] = wide;
  if (p0 < pieces) look(now[0], p0, g0);
  for (int i = tid + kBmThreads; i < again; i += kBmThreads) {
    int g;
    const int p = piece(i, g);
    if (p < pieces) look(__ldg(body + p), p, g);
  }
  __syncthreads();
  if (s.n_groups > a.room_groups || s.n_found > a.room) bm_again(s, r, a.k, least, found);
  const int have = s.n_found;
  const long long list = row * a.stretches + part;
  for (int i = tid; i < have; i += kBmThreads) {
    int above = 0;
#pragma unroll 4
    for (int o = 0; o < have; ++o) above += found[o] > found[i];
    if (above < a.k) a.keys[list * a.k + above] = found[i];
  }
  if (tid >= have && tid < a.k) a.keys[list * a.k + tid] = 0u;
  if (tid >= kBmThreads - kBmThreads / 32) {  // (not the warp that ranks)
    constexpr uint32_t kAll = ~((1u << (32 - kBmThreads / 32)) - 1);
    const float mine_top = red_top[tid - (kBmThreads - kBmThreads / 32)];
    float top = mine_top;
#pragma unroll
    for (int o = kBmThreads / 64; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    double total = red_sum[tid - (kBmThreads - kBmThreads / 32)];
    if (!(total == 0.0)) total *= bm_exp(mine_top - top);
#pragma unroll
    for (int o = kBmThreads / 64; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    if (tid == kBmThreads - 1) a.sums[list] = {total, top};
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

// One block per group.  What bounds it: latencies in a chain (the lists and sums come back, sums joined in 64 bits,
// heads ranked, what is left ranked), 4 to 5 us behind the lists of 4 beams of 262144, 16 lists or 64 of them.
__global__ void __launch_bounds__(kBmJoinThreads) beam_join_kernel(const __grid_constant__ BeamArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  BeamItem* heads = reinterpret_cast<BeamItem*>(raw);              // [kBmMaxLists]
  BeamItem* found = heads + kBmMaxLists;                           // [k * k]
  uint32_t* near = reinterpret_cast<uint32_t*>(found + a.k * a.k);  // the lists' keys where they have room
  __shared__ BeamBase base[G4_BEAM_MAX];
  __shared__ BeamItem deep[8];
  __shared__ int in[G4_BEAM_MAX];  // the lists whose heads are among the k best
  __shared__ uint32_t n_found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row0 = static_cast<long long>(blockIdx.x) * a.n_beams;
  const int lists = a.n_beams * a.stretches;
  if (tid == 0) n_found = 0;
  if (tid < a.k) in[tid] = -1;
  pdl_wait();
  const uint32_t* keys = a.keys + row0 * a.stretches * a.k;
  // (all that comes from memory is asked for at once)
  auto sum_of = [&](int b) {
    return b < a.n_beams && lane < a.stretches ? a.sums[(row0 + b) * a.stretches + lane] : BeamSum{0.0, -CUDART_INF_F};
  };
  const BeamSum own0 = sum_of(warp);
  const float score0 = warp < a.n_beams ? a.scores[row0 + warp] : 0.f;
  if (lists * a.k <= kBmNear) {
    for (int i = tid; i < lists * a.k; i += kBmJoinThreads) near[i] = keys[i];
    keys = near;
  }
  for (int b = warp; b < a.n_beams; b += kBmJoinThreads / 32) {
    const BeamSum* st = a.sums + (row0 + b) * a.stretches;
    const BeamSum own = b == warp ? own0 : sum_of(b);
    const float score = b == warp ? score0 : a.scores[row0 + b];
    float top = own.top;
    for (int i = lane + 32; i < a.stretches; i += 32) top = fmaxf(top, st[i].top);
    top = warp_max(top);
    double total = own.sum == 0.0 ? 0.0 : own.sum * exp(static_cast<double>(own.top) - top);
    for (int i = lane + 32; i < a.stretches; i += 32)
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
  // so many threads, neighbours of one warp, rank one of n
  auto sharing = [](int n) {
    int each = 32;
    while (each > 1 && each * n > kBmJoinThreads) each >>= 1;
    return each;
  };
  int share = sharing(lists);
  for (int i0 = 0; i0 < lists; i0 += kBmJoinThreads / share) {
    const int i = i0 + tid / share;
    const BeamItem mine = i < lists ? heads[i] : BeamItem{0ull, 0ull};
    int rank = 0;
    if (mine.rest != 0ull) {
#pragma unroll 4
      for (int j = tid & (share - 1); j < lists; j += share) rank += bm_above(heads[j], mine);
    }
    for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if ((tid & (share - 1)) == 0 && mine.rest != 0ull && rank < a.k) in[rank] = i;
  }
  __syncthreads();
  // nothing below the last head that is in can be (with fewer lists than that, everything can)
  const int last = in[a.k - 1];
  BeamItem bound = last >= 0 ? heads[last] : BeamItem{0ull, 0ull};
  auto item_of = [&](int list, int i) {
    if (list < 0) return BeamItem{0ull, 0ull};
    const int beam = list / a.stretches, part = list - beam * a.stretches;
    const uint32_t key = key_of(beam, part, i, keys[list * a.k + i]);
    return key ? bm_item(a, base[beam], beam, part, key) : BeamItem{0ull, 0ull};
  };
  // nor can what is below the (k/d)-th best of those lists' d-th: where many are selected and one beam leads, the
  // heads alone leave thousands to rank (64 of 32 beams of 262144: 420 us, and 37 us so)
  if (a.k > kBmQuads) {
    int depths = 0;
    while ((2 << depths) <= a.k) ++depths;
    for (int c = tid; c < depths * a.k; c += kBmJoinThreads) found[c] = item_of(in[c % a.k], (2 << c / a.k) - 1);
    if (tid < 8) deep[tid] = BeamItem{0ull, 0ull};
    __syncthreads();
    for (int c = tid; c < depths * a.k; c += kBmJoinThreads) {
      const int t = c / a.k, d = 2 << t;
      const BeamItem mine = found[c];
      int rank = 0;
      for (int j = 0; j < a.k; ++j) rank += bm_above(found[t * a.k + j], mine);
      if (mine.rest != 0ull && rank == (a.k + d - 1) / d - 1) deep[t] = mine;
    }
    __syncthreads();
    for (int t = 0; t < depths; ++t)
      if (bm_above(deep[t], bound)) bound = deep[t];
  }
  for (int c = tid; c < a.k * a.k; c += kBmJoinThreads) {
    const BeamItem item = item_of(in[c / a.k], c % a.k);
    if (item.rest != 0ull && !bm_above(bound, item)) found[atomicAdd(&n_found, 1u)] = item;
  }
  __syncthreads();
  const int have = n_found;
  share = sharing(have);
  for (int i0 = 0; i0 < have; i0 += kBmJoinThreads / share) {
    const int i = i0 + tid / share;
    const BeamItem mine = i < have ? found[i] : BeamItem{0ull, 0ull};
    int rank = 0;
    for (int j = tid & (share - 1); j < have && rank < a.k; j += share) rank += bm_above(found[j], mine);
    for (int o = 1; o < share; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if ((tid & (share - 1)) == 0 && i < have && rank < a.k) {
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
                0, 0, 0, 0, nullptr, nullptr, out_scores, out_beams, out_tokens};
  // Stretches of a row: more of them keep the SMs busier, fewer leave the join less.  Of 262144 logits, one row
  // takes 7.4 us in 32 stretches (7.9 in 16), 4 rows 8.8 in 16 (9.5 in 8, 9.8 in 32), 64 rows 16.0 in 8 (16.3 in
  // 4, 18.6 in 16), 80 rows 19.1 in 4 (20.4 in 8), 128 rows 22.7 in 4 (24.9 in 8).  And of a group no more lists
  // than 128, or 64 where they are long: 32 selected of 8 beams in 4 groups take 20.0 us in 8 (29.6 in 16).
  const int least = (vocab + kBmStretch - 1) / kBmStretch, useful = (vocab + 2047) / 2048;
  const int few = (n_select <= kBmQuads ? 128 : 64) / n_beams;
  int parts = rows <= 2 ? 32 : rows <= 32 ? 16 : rows < 72 ? 8 : 4;
  if (parts > useful) parts = useful;
  if (parts > few) parts = few;
  if (parts < least) parts = least;  // (at most 16, which is kBmMaxLists / 64)
  a.stretch = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  a.stretches = (vocab + a.stretch - 1) / a.stretch;
  const size_t lists = static_cast<size_t>(n_beams) * a.stretches;
  const size_t bytes = lists * (sizeof(BeamSum) + 4 * n_select);
  // the candidates of a stretch: as many as there are in the groups of n_select parts, should it come to that
  const int threads = n_select * (n_select <= kBmQuads ? 4 : 1), turns = (a.stretch / 8 + kBmThreads - 1) / kBmThreads;
  const int worst = threads * (8 * turns + 2);
  a.room = 16 * n_select + 384;
  a.room_groups = 8 * n_select + 64;
  const size_t once = 4 * static_cast<size_t>(a.room) + 2 * a.room_groups;
  const size_t list_smem = 4 * static_cast<size_t>(worst) > once ? 4 * static_cast<size_t>(worst) : once;
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
