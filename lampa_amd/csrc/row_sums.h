// Column sums of fp32 rows in a fixed order: what the gradients of weights that every token shares end with, after each
// workgroup has left one row.
#pragma once
#include "gdr_common.h"

#define RS_BLOCK 1024
#define RS_WAVES (RS_BLOCK / 64)
#define RS_COLS 64

// Where the sums of set z go: out[z], or, where out[1] is null, out[0] + z * stride.
template <typename OT>
struct RowSumsOut {
  OT* out[3];
  int64_t stride;
};

// Set z: sum_r rows[z_stride * z + row_stride * r + c] for every column c; 64 columns a workgroup, its 16 waves take the rows in
// turn, four under way each.
template <typename OT>
__global__ void __launch_bounds__(RS_BLOCK) row_sums_kernel(const float* __restrict__ rows, int64_t n_rows, int64_t n_cols,
                                                            int64_t row_stride, int64_t z_stride, RowSumsOut<OT> to) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * RS_COLS + lane;
  const float* src = rows + blockIdx.y * z_stride + c;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < n_cols) {
    int64_t r = wave;
    for (; r + 3 * RS_WAVES < n_rows; r += 4 * RS_WAVES) {
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] += src[(r + k * RS_WAVES) * row_stride];
    }
    for (; r < n_rows; r += RS_WAVES) sum[0] += src[r * row_stride];
  }
  __shared__ float part[RS_WAVES][RS_COLS];
  part[wave][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (wave == 0 && c < n_cols) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < RS_WAVES; ++k) total += part[k][lane];
    OT* out = to.out[1] ? to.out[blockIdx.y] : to.out[0] + blockIdx.y * to.stride;
    out[c] = GdrElem<OT>::from_float(total);
  }
}

// `sets` sets of rows, z_stride floats apart; rows row_stride floats apart.
template <typename OT>
static int row_sums_launch(const float* rows, int64_t n_rows, int64_t n_cols, int64_t row_stride, int64_t z_stride, int sets,
                           RowSumsOut<OT> to, hipStream_t s) {
  if (sets > 65535) return LAMPA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((n_cols + RS_COLS - 1) / RS_COLS), (unsigned)sets);
  hipLaunchKernelGGL((row_sums_kernel<OT>), grid, dim3(RS_BLOCK), 0, s, rows, n_rows, n_cols, row_stride, z_stride, to);
  LAMPA_PROF(s, "row_sums_kernel");
  return lampa_launch_status();
}
