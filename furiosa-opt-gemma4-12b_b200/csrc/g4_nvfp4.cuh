// NVFP4 rows and weights of the batched projections (g4_nvfp4.cu, g4_nvfp4_mm.cu).
#pragma once

#include "g4_common.cuh"
#include "g4_internal.h"

namespace g4 {

constexpr int kNvMaxCols = 16384;
constexpr int kNvMaxRows = 1 << 22;

// Scale blocks of one [rows, cols] matrix: bytes, and where the scale of (row, 16-column block b) is.
__host__ __device__ inline size_t nv_scale_bytes(int rows, int cols) {
  return static_cast<size_t>((rows + 127) / 128) * ((cols + 63) / 64) * 512;
}
__device__ __forceinline__ size_t nv_scale_at(int row, int b, int kblocks) {
  return (static_cast<size_t>(row >> 7) * kblocks + (b >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (b & 3);
}

struct NvMatmulArgs {
  const uint8_t* x_codes;
  const uint8_t* x_scales;
  const float* x_factor;
  const uint8_t* w_codes;
  const uint8_t* w_scales;
  const float* w_factor;
  int m, n, k, pieces, max_rows, n_factors, out_f32;
  int early;  // the weights may be fetched before the previous kernel is done
  void* out;
  long long out_stride;
};
g4_status launch_nvfp4_matmul(g4_ctx* ctx, const NvMatmulArgs& a);

}  // namespace g4
