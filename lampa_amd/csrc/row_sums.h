// Column sums of fp32 rows in a fixed order: what the gradients of weights that every token shares end with, after each
// workgroup has left one row.
#pragma once
#include "gdr_common.h"

#define RS_BLOCK 256
#define RS_COLS 64

// out[z, c] = sum_r rows[z, r, c]: 64 columns a workgroup, its 4 waves take the rows in turn.
template <typename OT>
__global__ void __launch_bounds__(RS_BLOCK) row_sums_kernel(const float* __restrict__ rows, int64_t n_rows, int64_t n_cols,
                                                            int64_t row_stride, int64_t z_stride, OT* __restrict__ out, int64_t out_stride) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * RS_COLS + lane;
  const float* src = rows + blockIdx.y * z_stride + c;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < n_cols) {
    int64_t r = wave;
    for (; r + 12 < n_rows; r += 16) {
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += src[(r + 4 * k) * row_stride];
    }
    for (; r < n_rows; r += 4) sum[0] += src[r * row_stride];
  }
  __shared__ float part[4][RS_COLS];
  part[wave][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (wave == 0 && c < n_cols)
    out[blockIdx.y * out_stride + c] =
        GdrElem<OT>::from_float((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

// `batch` sets of rows, z_stride floats apart; rows row_stride floats apart.
template <typename OT>
static int row_sums_launch(const float* rows, int64_t n_rows, int64_t n_cols, int64_t row_stride, int64_t z_stride, int batch,
                           OT* out, int64_t out_stride, hipStream_t s) {
  if (batch > 65535) return LAMPA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((n_cols + RS_COLS - 1) / RS_COLS), (unsigned)batch);
  hipLaunchKernelGGL((row_sums_kernel<OT>), grid, dim3(RS_BLOCK), 0, s, rows, n_rows, n_cols, row_stride, z_stride, out,
                     out_stride);
  LAMPA_PROF(s, "row_sums_kernel");
  return lampa_launch_status();
}
