// What the paged-cache kernels share (g4_paged.cu, g4_paged_attn.cu): the batch as a kernel
// argument, with its device-resident contents read through bounds, and the host checks.
#pragma once

#include "g4_common.cuh"
#include "g4_internal.h"

namespace g4 {

// Two f32 at a time.
__device__ __forceinline__ uint64_t pa_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void pa_unpair(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t pa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pa_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pa_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pa_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
struct PagedBatch {
  const int32_t* tables;
  long long table_stride;
  const int32_t* q_start;
  const int32_t* kv_len;
  int max_pages, n_seqs, n_tokens;
  int n_pages, page_rows;  // the cache's
};

// One sequence of a batch: new tokens [t0, t0 + n), cache rows [0, kv), first position
// kv - n.  Values outside their range are cut off; *bad reports it.
struct PagedSeq {
  int t0, n, kv;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s, bool* bad) {
  const int a = b.q_start[s], e = b.q_start[s + 1], l = b.kv_len[s];
  const long long room = min(static_cast<long long>(b.max_pages) * b.page_rows, 0x7fffff00ll);
  PagedSeq q;
  q.t0 = min(max(a, 0), b.n_tokens);
  q.n = min(max(e, q.t0), b.n_tokens) - q.t0;
  q.kv = static_cast<int>(min(static_cast<long long>(max(l, 0)), room));
  *bad = q.t0 != a || q.t0 + q.n != e || q.kv != l;
  return q;
}
// One warp of a launch looks over the whole batch, sequences without tokens included.
__device__ __forceinline__ void paged_check_batch(const PagedBatch& b, int lane, Scratch* scr) {
  bool any = false;
  for (int s = lane; s < b.n_seqs; s += 32) {
    bool bad;
    paged_seq(b, s, &bad);
    any |= bad;
  }
  if (lane == 0 && b.n_seqs > 0 && b.q_start[0] < 0) any = true;
  if (any) atomicOr(&scr->status, DEV_ERR_BAD_OFFSET);
}

// Host checks of the two descriptors (messages through g4_ctx_last_error).
g4_status check_paged_cache(g4_ctx* ctx, const g4_paged_cache* c);
g4_status check_paged_batch(g4_ctx* ctx, const g4_paged_batch* b);
PagedBatch paged_batch(const g4_paged_batch* b, const g4_paged_cache* c);
// A [tokens, heads, head_dim] operand: 16-byte aligned, strides multiples of 8.
g4_status check_rows(g4_ctx* ctx, const void* p, int64_t token_stride, int64_t head_stride, const char* what);
// The same for one that is written: its rows must not overlap.
g4_status check_out_rows(g4_ctx* ctx, const void* p, int64_t token_stride, int64_t head_stride, int tokens, int heads,
                         int head_dim, const char* what);

}  // namespace g4
