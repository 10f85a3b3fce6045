// NVFP4 activations of a batch: quantising rows (as they are or RMSNorm'ed), reading them back, and
// the checks of the products over them (g4_nvfp4_mm.cu).
//
// The recipe (include/g4.h) takes a power of two where the checkpoint's weights and the prefill MLP
// take 2688 / max|row| itself: E4M3 and E2M1 are floating point, so the power of two costs no
// precision, and every step but the two roundings becomes exact (x g has x's 8 bits; y - c s needs
// fewer than 24).  A row's codes then do not hang on the order of any arithmetic: bf16
// activations meet ties of both formats all the time (0.4 % of the blocks of a prompt's rows changed
// their scale between 32- and 64-bit arithmetic with the recipe of the weights).
#include <string>
#include <type_traits>

#include "g4_nvfp4.cuh"
#include "g4_paged_split.cuh"

namespace g4 {

__device__ __forceinline__ float2 nv_halves(uint32_t h) {
  return make_float2(__half2float(__ushort_as_half(static_cast<uint16_t>(h))),
                     __half2float(__ushort_as_half(static_cast<uint16_t>(h >> 16))));
}
__device__ __forceinline__ uint32_t nv_abs_max2(uint32_t a, uint32_t b) {  // of two bf16 each, its sign of no meaning
  uint32_t d;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Values as E2M1 codes, the first in the low nibble.  (Four bytes packed by one mov.b32 came out right in
// the word but not where the same word was taken apart again: pairs of bytes do.)
__device__ __forceinline__ uint32_t nv_e2m1x4(float2 a, float2 b) {
  uint16_t r;
  asm("{\n\t.reg .b8 t0, t1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t1, %4, %3;\n\t"
      "mov.b16 %0, {t0, t1};\n\t}"
      : "=h"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ uint32_t nv_e2m1x8(float2 a, float2 b, float2 c, float2 d) {
  return __byte_perm(nv_e2m1x4(a, b), nv_e2m1x4(c, d), 0x5410);
}
// Quotients by multiplication, right in every tie.  What is divided has at most 11 significant bits (x g has 8,
// y - c s at most 11: it is a multiple of 2^-9 of the scale's power of two and no larger than the scale), the
// borders of both formats have few (3 bits of E2M1's by 4 of the scale; 6 by 5 bits of E4M3's).  So a quotient
// that is not on a border is at least 2^-11 of itself away from it, and one that is has come out within
// 2^-22 of it: rounding the approximate quotient to 2^-16 (E2M1: by adding 192 and taking it off again) or to
// 16 significant bits (E4M3) puts the second on the border and leaves the first on its side.
// E4M3 with integers: at 2^-120 of its value an f32 has the format's exponents, subnormal ones among them, and
// its leading bits are the code.  (By conversions, with the borders between the codes, 51 us where this took 49.)
__device__ __forceinline__ uint32_t nv_scale_of(float top) {
  const uint32_t q = __float_as_uint(top * (1.0f / 6.0f));
  const uint32_t b = __float_as_uint(__uint_as_float((q + 0x80u) & ~0xFFu) * 0x1p-120f);
  return (b + 0x7FFFFu + ((b >> 20) & 1u)) >> 20;  // (at most 448: max|y| is at most 2688)
}
__device__ __forceinline__ float nv_scale_value(uint32_t code) { return __uint_as_float(code << 20) * 0x1p120f; }
__device__ __forceinline__ float nv_rcp(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return r;
}
__device__ __forceinline__ float lo_f32(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_f32(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

struct QuantArgs {
  const uint16_t* x;
  long long x_stride;
  const uint16_t* norm_w;
  int nb, kblocks;  // 16-column blocks of a row, scale blocks across
  uint8_t* codes;
  size_t code_row, code_piece;
  uint8_t* scales;
  size_t scale_piece;
  float* factor;
};

// What bounds it: instructions, and among them the integer pipe's (62 % busy when 4096 x 15360 in two pieces took 49
// us, now 40 us, with more of its rows on an SM; the bytes alone are 30 us): unpacking, maxima, codes and their
// bytes.  Beside the 49 us, rows through shared memory, the next one on its way, took 54 us; one f32 an
// instruction 58 us; back from codes by byte tables 53 us.
// With the norm 4096 x 3840 in two pieces take 19.7 us (12.4 without), 4096 x 15360 77 us: a conversion to f64 and an
// f64 FMA an element, and the instances of two blocks and more a thread spill (8 to 208 bytes).
//
// One block of T threads per row; thread t holds the row's 16-element blocks t and t + T (at most NB).
template <int T, int NB, int P, int kPerSm, bool kNorm>
__global__ void __launch_bounds__(T, kPerSm) nv_quant_kernel(const __grid_constant__ QuantArgs a) {
  __shared__ uint32_t redu[T / 32];
  __shared__ double redd[T / 32];
  const int row = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  if (P > 1) pdl_launch_dependents();  // (a product may read a constant weight meanwhile; one piece may be a weight)
  const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.x_stride);
  uint32_t w[NB][8];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int b = tid + i * T;
    const uint4 none = make_uint4(0, 0, 0, 0);
    const uint4 u = b < a.nb ? x[2 * b] : none, v = b < a.nb ? x[2 * b + 1] : none;
    w[i][0] = u.x, w[i][1] = u.y, w[i][2] = u.z, w[i][3] = u.w;
    w[i][4] = v.x, w[i][5] = v.y, w[i][6] = v.z, w[i][7] = v.w;
  }
  if (kNorm) {
    // 64-bit sums: a factor that is the same however it is added up leaves no element on the other side of
    // a rounding border
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double p = lo_f32(w[i][e]), q = hi_f32(w[i][e]);
        ss = fma(p, p, ss);
        ss = fma(q, q, ss);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((tid & 31) == 0) redd[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) ss += redd[i];
    const float r = static_cast<float>(1.0 / sqrt(ss / (16.0 * a.nb) + 1e-6));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int b = tid + i * T;
      if (b < a.nb) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(a.norm_w) + 2 * b),
                    v = __ldg(reinterpret_cast<const uint4*>(a.norm_w) + 2 * b + 1);
        const uint32_t nw[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[i][e] = pack_bf16x2(__fmul_rn(__fmul_rn(lo_f32(w[i][e]), r), lo_f32(nw[e])),
                                __fmul_rn(__fmul_rn(hi_f32(w[i][e]), r), hi_f32(nw[e])));
      }
    }
  }
  // |x| orders like its low 15 bits
  uint32_t own[NB], top = 0u;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    uint32_t m = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = nv_abs_max2(m, w[i][e]);
    m &= 0x7FFF7FFFu;
    own[i] = max(m & 0xFFFFu, m >> 16);
    top = max(top, own[i]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) redu[tid >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, redu[tid & (T / 32 - 1)]);
  const bool finite = top < 0x7F80u, live = finite && top != 0u;
  // g's biased exponent: 2688 = 1.3125 * 2^11, and 1.3125 is 40 of the 128 steps of a bf16 mantissa
  const uint32_t ge = min(253u, ((top & 0x7Fu) <= 40u ? 265u : 264u) - (live ? top >> 7 : 0u));
  const float g = live ? __uint_as_float(ge << 23) : 0.f;
  if (tid == 0) a.factor[row] = live ? __uint_as_float((254u - ge) << 23) : (finite ? 0.f : CUDART_NAN_F);
  if (!live) {  // nothing to divide by (and an infinity times 0 would be NaN)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      own[i] = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] = 0u;
    }
  }
  const float2 g2 = make_float2(g, g), snap = make_float2(192.f, 192.f), unsnap = make_float2(-192.f, -192.f);
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int b = tid + i * T;
    if (i > 0 && i * T >= 4 * a.kblocks) break;  // (of all threads)
    float2 y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = mul_f32x2(make_float2(lo_f32(w[i][e]), hi_f32(w[i][e])), g2);
    float m = lo_f32(own[i]) * g;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t sc = nv_scale_of(m);
      const float sf = nv_scale_value(sc), rcp = sc != 0u ? nv_rcp(sf) : 0.f;
      const float2 r2 = make_float2(rcp, rcp);
      float2 q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = add_f32x2(fma_f32x2(y[e], r2, snap), unsnap);
      const uint2 c = make_uint2(nv_e2m1x8(q[0], q[1], q[2], q[3]), nv_e2m1x8(q[4], q[5], q[6], q[7]));
      if (p + 1 < P) {  // what the piece leaves, and its largest
        const float2 s2 = make_float2(-sf, -sf);
        uint32_t h[8];
        cvt_e2m1x8(c.x, h[0], h[1], h[2], h[3]);
        cvt_e2m1x8(c.y, h[4], h[5], h[6], h[7]);
        m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = fma_f32x2(nv_halves(h[e]), s2, y[e]);
          m = pa_max3(m, fabsf(y[e].x), fabsf(y[e].y));
        }
      }
      if (b < a.nb) *reinterpret_cast<uint2*>(a.codes + p * a.code_piece + row * a.code_row + 8 * b) = c;
      // four lanes' scales are neighbours in a scale block (zeros past the row's end)
      uint32_t four = sc | __shfl_down_sync(0xffffffffu, sc, 1) << 8;
      four |= __shfl_down_sync(0xffffffffu, four, 2) << 16;
      if ((tid & 3) == 0 && b < 4 * a.kblocks)
        *reinterpret_cast<uint32_t*>(a.scales + p * a.scale_piece + nv_scale_at(row, b, a.kblocks)) = four;
    }
  }
}

// One thread per 16-column block of a row: 35 us of 4096 x 15360 in two pieces, whose 197 MB (5.6 TB/s) bound it.
template <int P>
__global__ void __launch_bounds__(256) nv_dequant_kernel(const __grid_constant__ QuantArgs a, uint16_t* out,
                                                         long long out_stride) {
  const int row = blockIdx.x, b = blockIdx.y * 256 + threadIdx.x;
  pdl_wait();
  if (b >= a.nb) return;
  const float f = a.factor[row];
  float v[16];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint2 c = *reinterpret_cast<const uint2*>(a.codes + p * a.code_piece + row * a.code_row + 8 * b);
    const float s = e4m3_value(a.scales[p * a.scale_piece + nv_scale_at(row, b, a.kblocks)]);
    uint32_t h[8];
    cvt_e2m1x8(c.x, h[0], h[1], h[2], h[3]);
    cvt_e2m1x8(c.y, h[4], h[5], h[6], h[7]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float lo = __half2float(__ushort_as_half(static_cast<uint16_t>(h[e]))) * s;
      const float hi = __half2float(__ushort_as_half(static_cast<uint16_t>(h[e] >> 16))) * s;
      v[2 * e] = p ? v[2 * e] + lo : lo;
      v[2 * e + 1] = p ? v[2 * e + 1] + hi : hi;
    }
  }
  uint32_t o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = pack_bf16x2(v[2 * e] * f, v[2 * e + 1] * f);
  uint4* to = reinterpret_cast<uint4*>(out + row * out_stride) + 2 * b;
  to[0] = make_uint4(o[0], o[1], o[2], o[3]);
  to[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// Four scales a thread; rows and columns past the matrix are zeros.
__global__ void __launch_bounds__(256) nv_scale_blocks_kernel(const uint8_t* __restrict__ in, int rows, int nb,
                                                              int kblocks, size_t words, uint32_t* out) {
  pdl_wait();
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= words) return;
  const size_t block = i >> 7;
  const int at = static_cast<int>(i & 127);  // 32 lanes of 4 row groups
  const long long row = static_cast<long long>(block / kblocks) * 128 + (at & 3) * 32 + (at >> 2);
  const int b0 = 4 * static_cast<int>(block % kblocks);
  uint32_t v = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (row < rows && b0 + j < nb) v |= static_cast<uint32_t>(in[row * nb + b0 + j]) << (8 * j);
  out[i] = v;
}

// ---------------------------------------------------------------------------- host side
static g4_status check_cols(g4_ctx* ctx, int cols, const char* what) {
  if (cols < 32 || cols % 32 != 0 || cols > kNvMaxCols)
    return fail(ctx, G4_ERR_BAD_ARG, std::string(what) + ": cols must be a multiple of 32 up to 16384");
  return G4_OK;
}
static g4_status check_nv_rows(g4_ctx* ctx, const g4_nvfp4_rows* r, int n_rows) {
  if (r == nullptr) return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 rows: null descriptor");
  const g4_status st = check_cols(ctx, r->cols, "nvfp4 rows");
  if (st != G4_OK) return st;
  if (r->pieces < 1 || r->pieces > 3) return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 rows: 1 to 3 pieces");
  if (r->max_rows < 1 || r->max_rows > kNvMaxRows || n_rows < 0 || n_rows > r->max_rows)
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 rows: max_rows or the call's rows out of range");
  if (!aligned16(r->codes) || !aligned16(r->scales) || !aligned16(r->factor))
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 rows: codes, scales or factor is null or not 16-byte aligned");
  return G4_OK;
}
static QuantArgs quant_args(const g4_nvfp4_rows* r) {
  QuantArgs a = {};
  a.nb = r->cols / 16;
  a.kblocks = (r->cols + 63) / 64;
  a.codes = r->codes;
  a.code_row = r->cols / 2;
  a.code_piece = static_cast<size_t>(r->max_rows) * (r->cols / 2);
  a.scales = r->scales;
  a.scale_piece = nv_scale_bytes(r->max_rows, r->cols);
  a.factor = r->factor;
  return a;
}
// Threads to a row, blocks to a thread and rows to an SM (which is registers to a thread).  Many rows want several
// on an SM, each at another point of its way from load to codes; no more rows than SMs want all threads that
// have work for each.  Two pieces: 1024 rows of 3840 take 4.1 us as 128 x 2, 8 to an SM (5.5 with 12 to an SM; 4096 of
// them 12.4 and 12.6, 16.2 as 256 x 2); 2048 rows of 8192 12.7 as 256 x 2 (12.8 as 128 x 4, 18.7 as 512 x 2); 4096
// rows of 15360 40 as 256 x 4 (44 with 5 to an SM, 42 as 128 x 8, 49 as 512 x 2).  One row of 15360 takes 2.8 as 512 x 2 (3.2 as
// 256 x 4), one of 3840 with its norm 2.7 as 256 x 1 (2.9 as 128 x 2).
template <int P, bool kNorm>
static const void* quant_kernel(int nb4, int rows, int sm_count, int& threads) {
  if (rows <= sm_count) {
    threads = nb4 <= 128 ? 128 : nb4 <= 256 ? 256 : 512;
    if (nb4 <= 128) return (const void*)nv_quant_kernel<128, 1, P, 8, kNorm>;
    if (nb4 <= 256) return (const void*)nv_quant_kernel<256, 1, P, 4, kNorm>;
    if (nb4 <= 512) return (const void*)nv_quant_kernel<512, 1, P, 2, kNorm>;
    return (const void*)nv_quant_kernel<512, 2, P, 2, kNorm>;
  }
  threads = nb4 <= 256 ? 128 : 256;
  if (nb4 <= 128) return (const void*)nv_quant_kernel<128, 1, P, 8, kNorm>;
  if (nb4 <= 256) return (const void*)nv_quant_kernel<128, 2, P, 8, kNorm>;
  if (nb4 <= 512) return (const void*)nv_quant_kernel<256, 2, P, 5, kNorm>;
  return (const void*)nv_quant_kernel<256, 4, P, 4, kNorm>;
}

}  // namespace g4

using namespace g4;

extern "C" {

uint64_t g4_nvfp4_scale_bytes(int rows, int cols) { return rows < 0 || cols < 0 ? 0 : nv_scale_bytes(rows, cols); }

g4_status g4_nvfp4_scale_blocks(g4_ctx* ctx, const g4_f8e4m3* block_scale, int rows, int cols, g4_f8e4m3* out) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  const g4_status st = check_cols(ctx, cols, "scale blocks");
  if (st != G4_OK) return st;
  if (rows < 0 || rows > kNvMaxRows) return fail(ctx, G4_ERR_BAD_ARG, "scale blocks: rows out of range");
  if (rows == 0) return G4_OK;
  if (block_scale == nullptr || !aligned16(out))
    return fail(ctx, G4_ERR_BAD_ARG, "scale blocks: null scales, or out is null or not 16-byte aligned");
  DeviceGuard on(ctx);
  int nb = cols / 16, kblocks = (cols + 63) / 64;
  size_t words = nv_scale_bytes(rows, cols) / 4;
  void* a[] = {(void*)&block_scale, (void*)&rows, (void*)&nb, (void*)&kblocks, (void*)&words, (void*)&out};
  return launch_kernel(ctx, (const void*)nv_scale_blocks_kernel, dim3(static_cast<unsigned>((words + 255) / 256)),
                       dim3(256), 0, a, false, "scale blocks");
}

g4_status g4_nvfp4_quantize(g4_ctx* ctx, const g4_bf16* x, int64_t x_stride, int n_rows, const g4_bf16* rms_weight,
                            const g4_nvfp4_rows* out) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_nv_rows(ctx, out, n_rows);
  if (st != G4_OK || n_rows == 0) return st;
  if ((st = check_matrix(ctx, x, x_stride, n_rows, out->cols, "x")) != G4_OK) return st;
  if (rms_weight != nullptr && (st = check_matrix(ctx, rms_weight, out->cols, 1, out->cols, "rms_weight")) != G4_OK)
    return st;
  DeviceGuard on(ctx);
  QuantArgs a = quant_args(out);
  a.x = x;
  a.x_stride = x_stride;
  a.norm_w = rms_weight;
  int threads = 0;
  auto kernel = [&](auto norm) {
    const int nb4 = 4 * a.kblocks;
    return out->pieces == 1   ? quant_kernel<1, decltype(norm)::value>(nb4, n_rows, ctx->sm_count, threads)
           : out->pieces == 2 ? quant_kernel<2, decltype(norm)::value>(nb4, n_rows, ctx->sm_count, threads)
                              : quant_kernel<3, decltype(norm)::value>(nb4, n_rows, ctx->sm_count, threads);
  };
  const void* fn = rms_weight != nullptr ? kernel(std::true_type()) : kernel(std::false_type());
  void* args[] = {(void*)&a};
  st = launch_kernel(ctx, fn, dim3(n_rows), dim3(threads), 0, args, false, "nvfp4 quantize");
  ctx->quantised = st == G4_OK && ctx->pdl_ok && out->pieces > 1 ? launches_on(ctx).load() : 0;
  return st;
}

g4_status g4_nvfp4_dequantize(g4_ctx* ctx, const g4_nvfp4_rows* rows, int n_rows, g4_bf16* out, int64_t out_stride) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_nv_rows(ctx, rows, n_rows);
  if (st != G4_OK || n_rows == 0) return st;
  if ((st = check_matrix(ctx, out, out_stride, n_rows, rows->cols, "out")) != G4_OK) return st;
  DeviceGuard on(ctx);
  QuantArgs a = quant_args(rows);
  long long os = out_stride;
  void* args[] = {(void*)&a, (void*)&out, (void*)&os};
  const void* fn = rows->pieces == 1   ? (const void*)nv_dequant_kernel<1>
                   : rows->pieces == 2 ? (const void*)nv_dequant_kernel<2>
                                       : (const void*)nv_dequant_kernel<3>;
  return launch_kernel(ctx, fn, dim3(n_rows, (a.nb + 255) / 256), dim3(256), 0, args, false, "nvfp4 dequantize");
}

g4_status g4_nvfp4_matmul(g4_ctx* ctx, const g4_nvfp4_rows* rows, int n_rows, const g4_nvfp4_weight* weight, void* out,
                          int64_t out_stride, int out_f32) {
  if (ctx == nullptr) return G4_ERR_BAD_ARG;
  g4_status st = check_nv_rows(ctx, rows, n_rows);
  if (st != G4_OK) return st;
  if (weight == nullptr) return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: null descriptor");
  if (weight->rows < 1 || weight->rows > kNvMaxRows || weight->cols != rows->cols)
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: rows out of range, or cols other than the activations'");
  if (weight->constant != 0 && weight->constant != 1)
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: constant is 0 or 1");
  if (weight->n_factors != 1 && weight->n_factors != weight->rows)
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: one factor, or one for each row");
  if (!aligned16(weight->codes) || !aligned16(weight->scales))
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: codes or scales is null or not 16-byte aligned");
  if (weight->factor == nullptr || (reinterpret_cast<uintptr_t>(weight->factor) & 3u))
    return fail(ctx, G4_ERR_BAD_ARG, "nvfp4 weight: factor is null or misaligned");
  if (n_rows == 0) return G4_OK;
  if ((st = check_matrix(ctx, out, out_stride, n_rows, weight->rows, "out")) != G4_OK) return st;
  if (n_rows == 1) out_stride = (static_cast<int64_t>(weight->rows) + 7) / 8 * 8;  // (of no meaning, but tensor maps want one)
  DeviceGuard on(ctx);
  // Nothing behind that quantisation on the stream: no launch of any context (one may have laid this weight out, or be
  // about to overwrite it as one of its rows' pieces), and no kernel of the caller's that could write a constant weight.
  const bool early = weight->constant != 0 && ctx->quantised != 0 && ctx->quantised == launches_on(ctx).load();
  return launch_nvfp4_matmul(ctx, {rows->codes, rows->scales, rows->factor, weight->codes, weight->scales, weight->factor,
                                   n_rows, weight->rows, rows->cols, rows->pieces, rows->max_rows, weight->n_factors,
                                   out_f32 != 0, early, out, out_stride});
}

}  // extern "C"
