// Row operators of a batch: embedding rows of many tokens (ops::embed_token, src/ops.rs:9-36) and
// the norm and residual add behind an output projection (src/ops.rs:138-158).
#include <string>

#include "g4_internal.h"
#include "g4_common.cuh"

namespace g4 {

g4_status check_matrix(g4_ctx* ctx, const void* p, int64_t stride, int rows, int cols, const char* what) {
  if (!aligned16(p)) return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + " is null or not 16-byte aligned");
  if (rows > 1 && (stride < cols || stride % 8 != 0 || stride > (int64_t(1) << 38)))
    return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + ": the row stride must be a multiple of 8 and at least the row");
  return G4_OK;
}

// One block per token, 16 bytes a thread and step.  A token's row is 7.5 KB: with four loads a thread
// under way the blocks of a prompt keep the memory busy, and one token is one round trip for its
// id and one for its row.  What bounds it: the bytes, 9.9 us of 4096 tokens of 3840 (6.4 TB/s, a copy's rate);
// 1.4 us of one token.
__global__ void __launch_bounds__(128) embed_rows_kernel(const uint16_t* __restrict__ table, int vocab, int vecs,
                                                         const int32_t* __restrict__ tokens, float scale,
                                                         uint16_t* __restrict__ out, long long out_stride,
                                                         uint32_t* status) {
  pdl_wait();
  const long long t = blockIdx.x;
  const int id = __ldg(tokens + t);
  const bool in = id >= 0 && id < vocab;
  if (!in && threadIdx.x == 0) atomicOr(status, DEV_ERR_BAD_OFFSET);
  const uint4* row = reinterpret_cast<const uint4*>(table) + static_cast<long long>(in ? id : 0) * vecs;
  uint4* to = reinterpret_cast<uint4*>(out + t * out_stride);
  for (int i0 = threadIdx.x; i0 < vecs; i0 += 4 * blockDim.x) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * blockDim.x;
      v[j] = in && i < vecs ? __ldg(row + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * blockDim.x;
      if (i >= vecs) break;
      uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack_bf16x2(__uint_as_float(w[e] << 16) * scale, __uint_as_float(w[e] & 0xFFFF0000u) * scale);
      to[i] = in ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0, 0, 0, 0);  // (not 0 x scale: it may be inf)
    }
  }
}

// One block of T threads per row; a thread holds up to NB 16-byte pieces of x, of the residual and of
// the weight, all requested before the sum of squares is joined: one pass, 16.4 us of 4096 x 3840 (5.8 TB/s, what
// bounds it), 1.6 us of 32 rows (one round trip to memory and one join).
template <int T, int NB>
__global__ void __launch_bounds__(T) residual_norm_kernel(const uint16_t* x, long long x_stride,
                                                          const uint16_t* __restrict__ w, const uint16_t* residual,
                                                          long long r_stride, int vecs, uint16_t* out,
                                                          long long out_stride) {
  __shared__ float red[T / 32];
  const long long row = blockIdx.x;
  pdl_wait();
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * x_stride);
  const uint4* rr = reinterpret_cast<const uint4*>(residual + row * r_stride);
  uint4* to = reinterpret_cast<uint4*>(out + row * out_stride);
  uint4 xv[NB], rv[NB], wv[NB];
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int i = threadIdx.x + j * T;
    xv[j] = i < vecs ? xr[i] : none;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int i = threadIdx.x + j * T;
    rv[j] = i < vecs ? rr[i] : none;
    wv[j] = i < vecs ? __ldg(reinterpret_cast<const uint4*>(w) + i) : none;
  }
  auto squares = [&](float scale) {  // of x times scale, added up over the block
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const uint32_t v[4] = {xv[j].x, xv[j].y, xv[j].z, xv[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = __uint_as_float(v[e] << 16) * scale, b = __uint_as_float(v[e] & 0xFFFF0000u) * scale;
        ss = fmaf(a, a, ss);
        ss = fmaf(b, b, ss);
      }
    }
    ss = warp_sum(ss);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) total += red[i];
    return total;
  };
  float total = squares(1.f), r = rms_factor(total, 8 * vecs);
  if (!(total <= 3e38f)) {  // (beyond f32, where 1e-6 counts for nothing; what is not finite stays so)
    total = squares(0x1p-80f);
    r = 0x1p-80f / sqrtf(total / static_cast<float>(8 * vecs));
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int i = threadIdx.x + j * T;
    if (i >= vecs) break;
    const uint32_t a[4] = {xv[j].x, xv[j].y, xv[j].z, xv[j].w}, b[4] = {rv[j].x, rv[j].y, rv[j].z, rv[j].w},
                   c[4] = {wv[j].x, wv[j].y, wv[j].z, wv[j].w};
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = pack_bf16x2(fmaf(__uint_as_float(a[e] << 16) * r, __uint_as_float(c[e] << 16), __uint_as_float(b[e] << 16)),
                         fmaf(__uint_as_float(a[e] & 0xFFFF0000u) * r, __uint_as_float(c[e] & 0xFFFF0000u),
                              __uint_as_float(b[e] & 0xFFFF0000u)));
    to[i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace g4

using namespace g4;

extern "C" {

g4_status g4_embed_tokens(g4_ctx* ctx, const g4_bf16* table, int vocab, int dim, const int32_t* tokens, int n_tokens,
                          float scale, g4_bf16* out, int64_t out_stride) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  if (vocab < 1 || dim < 8 || dim % 8 != 0 || n_tokens < 0)
    return fail(ctx, G4_ERR_BAD_ARG, "embed_tokens: vocab, dim (a multiple of 8) or n_tokens out of range");
  if (n_tokens == 0) return G4_OK;
  g4_status st = check_matrix(ctx, table, dim, vocab, dim, "table");
  if (st == G4_OK) st = check_matrix(ctx, out, out_stride, n_tokens, dim, "out");
  if (st != G4_OK) return st;
  if (tokens == nullptr || (reinterpret_cast<uintptr_t>(tokens) & 3u))
    return fail(ctx, G4_ERR_BAD_ARG, "tokens is null or misaligned");
  DeviceGuard on(ctx);
  int vecs = dim / 8;
  long long os = out_stride;
  uint32_t* status = &ctx->buf.scratch->status;
  void* a[] = {(void*)&table, (void*)&vocab, (void*)&vecs, (void*)&tokens,
               (void*)&scale, (void*)&out,   (void*)&os,   (void*)&status};
  const int threads = vecs >= 128 ? 128 : (vecs + 31) / 32 * 32;
  return launch_kernel(ctx, (const void*)embed_rows_kernel, dim3(n_tokens), dim3(threads), 0, a, false, "embed tokens");
}

g4_status g4_residual_norm(g4_ctx* ctx, const g4_bf16* x, int64_t x_stride, const g4_bf16* rms_weight,
                           const g4_bf16* residual, int64_t residual_stride, int n_rows, int dim, g4_bf16* out,
                           int64_t out_stride) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  if (dim < 8 || dim % 8 != 0 || dim > 16384 || n_rows < 0)
    return fail(ctx, G4_ERR_BAD_ARG, "residual_norm: dim must be a multiple of 8 up to 16384, n_rows not negative");
  if (n_rows == 0) return G4_OK;
  g4_status st = check_matrix(ctx, x, x_stride, n_rows, dim, "x");
  if (st == G4_OK) st = check_matrix(ctx, residual, residual_stride, n_rows, dim, "residual");
  if (st == G4_OK) st = check_matrix(ctx, out, out_stride, n_rows, dim, "out");
  if (st == G4_OK) st = check_matrix(ctx, rms_weight, dim, 1, dim, "rms_weight");
  if (st != G4_OK) return st;
  DeviceGuard on(ctx);
  int vecs = dim / 8;
  long long xs = x_stride, rs = residual_stride, os = out_stride;
  void* a[] = {(void*)&x,    (void*)&xs,  (void*)&rms_weight, (void*)&residual, (void*)&rs,
               (void*)&vecs, (void*)&out, (void*)&os};
  const void* fn;
  int threads = 128;
  if (vecs <= 128) fn = (const void*)residual_norm_kernel<128, 1>;
  else if (vecs <= 256) fn = (const void*)residual_norm_kernel<128, 2>;
  else if (vecs <= 512) fn = (const void*)residual_norm_kernel<128, 4>;
  else if (vecs <= 1024) fn = (const void*)residual_norm_kernel<256, 4>, threads = 256;
  else fn = (const void*)residual_norm_kernel<512, 4>, threads = 512;
  return launch_kernel(ctx, fn, dim3(n_rows), dim3(threads), 0, a, false, "residual norm");
}

}  // extern "C"
