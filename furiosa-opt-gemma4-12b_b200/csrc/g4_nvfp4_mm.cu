// Products of NVFP4 rows and weights:
//   out[m][n] = fx[m] * fw[n] * sum_k (sum_p cx[p][m][k] sx[p][m][k / 16]) cw[n][k] sw[n][k / 16]
#include "g4_nvfp4.cuh"

namespace g4 {

// One warp per output: lanes take the 16-column blocks in turn.
__global__ void __launch_bounds__(256) nv_matmul_kernel(const __grid_constant__ NvMatmulArgs a) {
  const int lane = threadIdx.x & 31, n = blockIdx.y * 8 + (threadIdx.x >> 5), m = blockIdx.x;
  pdl_wait();
  if (n >= a.n) return;
  const int nb = a.k / 16, kblocks = (a.k + 63) / 64;
  float sum = 0.f;
  for (int b = lane; b < nb; b += 32) {
    const uint2 wc = *reinterpret_cast<const uint2*>(a.w_codes + static_cast<size_t>(n) * (a.k / 2) + 8 * b);
    uint32_t w[8];
    cvt_e2m1x8(wc.x, w[0], w[1], w[2], w[3]);
    cvt_e2m1x8(wc.y, w[4], w[5], w[6], w[7]);
    const float ws = e4m3_value(a.w_scales[nv_scale_at(n, b, kblocks)]);
    for (int p = 0; p < a.pieces; ++p) {
      const uint2 xc = *reinterpret_cast<const uint2*>(
          a.x_codes + (static_cast<size_t>(p) * a.max_rows + m) * (a.k / 2) + 8 * b);
      uint32_t x[8];
      cvt_e2m1x8(xc.x, x[0], x[1], x[2], x[3]);
      cvt_e2m1x8(xc.y, x[4], x[5], x[6], x[7]);
      const float xs = e4m3_value(a.x_scales[p * nv_scale_bytes(a.max_rows, a.k) + nv_scale_at(m, b, kblocks)]);
      float dot = 0.f;  // exact: 16 products of two small numbers
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t q = hmul2_u32(w[e], x[e]);
        dot += __half2float(__ushort_as_half(static_cast<uint16_t>(q))) +
               __half2float(__ushort_as_half(static_cast<uint16_t>(q >> 16)));
      }
      sum = fmaf(dot, ws * xs, sum);
    }
  }
  sum = warp_sum(sum);
  if (lane == 0) {
    const float v = sum * a.x_factor[m] * a.w_factor[a.n_factors > 1 ? n : 0];
    const size_t at = static_cast<size_t>(m) * a.out_stride + n;
    if (a.out_f32)
      static_cast<float*>(a.out)[at] = v;
    else
      static_cast<uint16_t*>(a.out)[at] = f32_to_bf16(v);
  }
}

g4_status launch_nvfp4_matmul(g4_ctx* ctx, const NvMatmulArgs& args) {
  NvMatmulArgs a = args;
  void* p[] = {(void*)&a};
  return launch_kernel(ctx, (const void*)nv_matmul_kernel, dim3(a.m, (a.n + 7) / 8), dim3(256), 0, p, false, "nvfp4 matmul");
}

}  // namespace g4
