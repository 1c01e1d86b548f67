// The gated feed-forward block for any width: tiled matrix products whose epilogues hold what is elementwise (ff_common.h has the
// mathematics). Hidden values go through memory between the products.
//   hidden:  S from x, Wg and Wu in one kernel (both products share x's tiles);
//   grads:   G, U from x and dS from dy and Wd^T in one kernel, which leaves S, dG and dU;
//   product: y = S Wd^T; dx = dG Wg + dU Wu as one sum over both (on transposed weights: all operands then lie along their
//            contraction);
//   weights: dWg, dWu, dWd over the rows, split over the rows where that fills the GPU, the parts summed in a fixed order.
// A workgroup has 4 waves in 2 x 2 over a tile of 128 (or 64) x 128 of the output (64 hidden columns of each product for `hidden` and
// `grads`), tiles of 128 bytes of the contraction in LDS, double buffered, the next one on its way from memory to LDS past the registers
// (through them: hidden 72 us, grads 134, weights 138). A product with few tiles has its contraction shared out and the parts summed
// in order. Rows of 128 bytes are stored with their 16-byte pieces permuted by the row (piece ^ row / 2 % 8): 16 rows of an operand
// read, 8 even and 8 odd ones, fill the 256 bytes of the banks once.
//
// Measured, 8 192 x 768, 2 048 hidden columns, bf16 (the library's 8 192 x 4 096 x 768 product alone 0.88 PFLOP/s): hidden 61 us (51.5 GFLOP,
// 0.84 PFLOP/s), grads 116 us (77 GFLOP), y 35 and dx 62 us (77 GFLOP together), weights 125 us (77 GFLOP; medians of a kernel trace). The matrix cores are
// busy for half of the time. It is neither LDS alone (without the conflicts of piece ^ row % 8, half of its cycles, hidden and grads
// take 1% less), nor the loads: steps of 64 bytes, three ahead, take 72 and 136 us against 69 and 122, tiles of 256 rows by 8 waves, two
// steps ahead, 72 and 125. fp32, 1 501 x 96, 256 hidden columns: hidden 7, grads 12, y 9, dx 13, weights 22 us.
#include "ff_common.h"

#define MM_BLOCK 256
#define MM_ROW_BYTES 128  // of the contraction
#define MM_STAGE(MB) ((64 * (MB) + 128) * MM_ROW_BYTES)  // one step's tiles: 64 MB rows of x against 128 of the weights

template <typename T>
__device__ __forceinline__ f32x16 mm_mac(ff_u32x4 a, ff_u32x4 b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    return mfma32(__builtin_bit_cast(typename OpVec<T>::x8, a), __builtin_bit_cast(typename OpVec<T>::x8, b), c);
  } else {  // 8 values of the contraction: lane half hh holds 4 hh .. + 3, step j pairs j and 4 + j
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
}

// A tile's operand: 64 rows (or 128) of a row-major matrix, `step` elements apart.
struct MmSide {
  __amdgpu_buffer_rsrc_t buf;  // from the tile's first row to the end of its last one
  unsigned step;               // bytes between rows
};
template <typename T>
__device__ __forceinline__ MmSide mm_side(const T* base, int64_t first, int64_t rows, int64_t stride, int K) {
  const int64_t left = rows - first;
  const int64_t n = left < 0 ? 0 : (left < 128 ? left : 128);
  return {ff_buffer(base + (n ? first * stride : 0), n ? ((n - 1) * stride + K) * (int64_t)sizeof(T) : 0), (unsigned)(stride * sizeof(T))};
}

// 16 bytes of each lane from memory to LDS: lane l's go to p + 16 l, zeros where its offset is out of range.
__device__ __forceinline__ void mm_load_lds(__amdgpu_buffer_rsrc_t buf, unsigned char* p, unsigned offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (__attribute__((address_space(3))) void*)p, 16, offset, 0, 0, 0);
}

// acc[m][b] += (B rows b) . (A rows m) over K: register r of a lane is B row 8 (r / 4) + 4 hh + r % 4 of its block, A row = lane % 32.
// The wave's MB A blocks are rows 32 (MB wm + m), its B blocks rows 32 wn and 64 + 32 wn (the second from b1).
template <typename T, int MB, int NB>
__device__ __forceinline__ void mm_phase(const MmSide& a, const MmSide& b0, const MmSide& b1, int K, unsigned char* lds,
                                         f32x16 (&acc)[MB][NB]) {
  constexpr int BR = 64 * NB, BCH = BR * 8 / MM_BLOCK, AR = 64 * MB, ACH = AR * 8 / MM_BLOCK, ATILE = AR * MM_ROW_BYTES;
  constexpr int STAGE = MM_STAGE(MB);
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int steps = (K * (int)sizeof(T) + MM_ROW_BYTES - 1) / MM_ROW_BYTES;
  // A wave's load of 64 pieces of 16 bytes fills 8 rows of 128 bytes in LDS, lane by lane; which piece of the row a lane asks for makes
  // the permutation.
  auto fetch = [&](int step, int which) {
    unsigned char* p = lds + which * STAGE + __builtin_amdgcn_readfirstlane(wave) * 1024;
    const int row = tid >> 3, at = step * MM_ROW_BYTES + ((tid & 7) ^ (row >> 1 & 7)) * 16;
    const bool in = at < K * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < ACH; ++i) mm_load_lds(a.buf, p + i * 4096, in ? (row + 32 * i) * a.step + at : FF_OFF);
#pragma unroll
    for (int i = 0; i < BCH; ++i)
      mm_load_lds(i >= 2 ? b1.buf : b0.buf, p + ATILE + i * 4096, in ? (row + 32 * (i & 1)) * b0.step + at : FF_OFF);
  };
  fetch(0, 0);
  for (int step = 0; step < steps; ++step) {
    // this step's tiles are there for all waves, and the last step's are free
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (step + 1 < steps) fetch(step + 1, (step + 1) & 1);
    const unsigned char* p = lds + (step & 1) * STAGE;
    // operands are read a step ahead of their products, held there by the barriers
    ff_u32x4 fa[2][MB], fb[2][NB];
    auto read = [&](int ks) {
      const int piece = ((ks * 2 + hh) ^ (ln >> 1 & 7)) * 16;
#pragma unroll
      for (int m = 0; m < MB; ++m) fa[ks & 1][m] = *reinterpret_cast<const ff_u32x4*>(p + (32 * (MB * wm + m) + ln) * MM_ROW_BYTES + piece);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        fb[ks & 1][b] = *reinterpret_cast<const ff_u32x4*>(p + ATILE + (64 * b + 32 * wn + ln) * MM_ROW_BYTES + piece);
    };
    read(0);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks + 1 < 4) read(ks + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[m][b] = mm_mac<T>(fb[ks & 1][b], fa[ks & 1][m], acc[m][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  lds_barrier();  // the tiles are free
}

template <int M, int N>
__device__ __forceinline__ void mm_clear(f32x16 (&acc)[M][N]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[m][b][r] = 0.0f;
}

// Workgroup -> tile of the output. Workgroups go round robin over the 8 XCDs, each with an L2 of its own.
// mm_place: an XCD takes every 8th row tile and all columns, a strip of 8 row tiles at a time: its rows stay in L2 while the columns pass.
__device__ __forceinline__ void mm_place(int64_t row_tiles, int col_tiles, int64_t& rt, int& ct) {
  const int64_t per = 8 * (int64_t)col_tiles, strip = blockIdx.x / per, in = blockIdx.x % per;
  const int64_t high = row_tiles - strip * 8 < 8 ? row_tiles - strip * 8 : 8;
  rt = strip * 8 + in % high;
  ct = (int)(in / high);
}
// mm_place_columns: an XCD takes every 8th column tile and all rows, row tile by row tile: its part of the weights stays in L2 while the rows
// pass. For weights that L2 does not hold as a whole. The grid is 8 x column tiles of an XCD x row tiles; false: no tile.
__device__ __forceinline__ bool mm_place_columns(int col_tiles, int64_t& rt, int& ct) {
  const int each = (col_tiles + 7) / 8, in = blockIdx.x / 8;
  ct = (int)(blockIdx.x % 8) + 8 * (in % each);
  rt = in / each;
  return ct < col_tiles;
}

// Four hidden values (or their gradients), and, where `low` is not 0, what their rounding leaves as many elements on.
template <typename T>
__device__ __forceinline__ void mm_store_parts(T* p, int64_t low, const float (&v)[4]) {
  ff_store4(p, v[0], v[1], v[2], v[3]);
  if (low) ff_store4(p + low, ff_rest<T>(v[0]), ff_rest<T>(v[1]), ff_rest<T>(v[2]), ff_rest<T>(v[3]));
}

// ------------------------------------------------------------------------------------------------ S = act(x Wg^T) (x Wu^T)
template <typename T, int ACT, int MB>
__global__ void __launch_bounds__(MM_BLOCK, 2) ff_hidden_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ wg,
                                                             const T* __restrict__ wu, int64_t rows, int D, int F,
                                                             T* __restrict__ hidden, int64_t low, bool columns) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * MM_STAGE(MB)];
  int64_t rt;
  int ct;
  if (columns) {
    if (!mm_place_columns((F + 63) / 64, rt, ct)) return;
  } else {
    mm_place((rows + 64 * MB - 1) / (64 * MB), (F + 63) / 64, rt, ct);
  }
  const int64_t r0 = rt * (64 * MB);
  const int f0 = ct * 64;
  f32x16 acc[MB][2];
  mm_clear(acc);
  mm_phase<T, MB, 2>(mm_side(x, r0, rows, x_stride, D), mm_side(wg, f0, F, D, D), mm_side(wu, f0, F, D, D), D, lds, acc);
  const int lane = threadIdx.x & 63, ln = lane & 31, hh = lane >> 5, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int64_t row = r0 + 32 * (MB * wm + m) + ln;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int f = f0 + 32 * wn + 8 * q + 4 * hh;
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = ff_act<ACT>(acc[m][0][4 * q + k]) * acc[m][1][4 * q + k];
      if (row < rows && f < F) mm_store_parts(hidden + row * F + f, low, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ S, dG, dU
template <typename T, int ACT, int MB>
__global__ void __launch_bounds__(MM_BLOCK, 2) ff_grads_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy,
                                                            const T* __restrict__ wg, const T* __restrict__ wu,
                                                            const T* __restrict__ wd_t, int64_t rows, int D, int F,
                                                            T* __restrict__ hidden, T* __restrict__ dg, T* __restrict__ du,
                                                            int64_t low, bool columns) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * MM_STAGE(MB)];
  int64_t rt;
  int ct;
  if (columns) {
    if (!mm_place_columns((F + 63) / 64, rt, ct)) return;
  } else {
    mm_place((rows + 64 * MB - 1) / (64 * MB), (F + 63) / 64, rt, ct);
  }
  const int64_t r0 = rt * (64 * MB);
  const int f0 = ct * 64;
  f32x16 acc[MB][2], ds[MB][1];
  mm_clear(acc);
  mm_clear(ds);
  mm_phase<T, MB, 2>(mm_side(x, r0, rows, x_stride, D), mm_side(wg, f0, F, D, D), mm_side(wu, f0, F, D, D), D, lds, acc);
  const MmSide wd = mm_side(wd_t, f0, F, D, D);
  mm_phase<T, MB, 1>(mm_side(dy, r0, rows, D, D), wd, wd, D, lds, ds);
  const int lane = threadIdx.x & 63, ln = lane & 31, hh = lane >> 5, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int64_t row = r0 + 32 * (MB * wm + m) + ln;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int f = f0 + 32 * wn + 8 * q + 4 * hh;
      float v[4], g[4], u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float value, slope;
        ff_act_slope<ACT>(acc[m][0][4 * q + k], value, slope);
        const float up = acc[m][1][4 * q + k], d = ds[m][0][4 * q + k];
        v[k] = value * up;
        g[k] = d * up * slope;
        u[k] = d * value;
      }
      if (row < rows && f < F) {
        if (hidden) mm_store_parts(hidden + row * F + f, low, v);
        mm_store_parts(dg + row * F + f, low, g);
        mm_store_parts(du + row * F + f, low, u);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ out = A0 B0^T (+ A1 B1^T)
// Part blockIdx.y takes `span` of the contraction's columns (of both products); with more than one part the sums go to parts
// [splits, rows, N] in fp32. `low` not 0: A0 and A1 have a second part as many elements on.
template <typename T, int MB>
__global__ void __launch_bounds__(MM_BLOCK, 2) ff_product_kernel(const T* __restrict__ a0, const T* __restrict__ b0,
                                                                              const T* __restrict__ a1, const T* __restrict__ b1,
                                                                              int64_t low, int64_t rows, int N, int K, int span, T* __restrict__ out,
                                                                              float* __restrict__ parts) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * MM_STAGE(MB)];
  int64_t rt;
  int ct;
  mm_place((rows + 64 * MB - 1) / (64 * MB), (N + 127) / 128, rt, ct);
  const int64_t r0 = rt * (64 * MB);
  const int n0 = ct * 128, k0 = blockIdx.y * span, width = K - k0 < span ? K - k0 : span;
  f32x16 acc[MB][2];
  mm_clear(acc);
  const int products = a1 ? 2 : 1;
  for (int i = 0; i < (low ? 2 * products : products); ++i) {
    const int p = low ? i >> 1 : i;
    const T *a = (p ? a1 : a0) + (low && i & 1 ? low : 0) + k0, *b = (p ? b1 : b0) + k0;
    mm_phase<T, MB, 2>(mm_side(a, r0, rows, K, width), mm_side(b, n0, N, K, width), mm_side(b, n0 + 64, N, K, width), width, lds, acc);
  }
  const int lane = threadIdx.x & 63, ln = lane & 31, hh = lane >> 5, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int64_t row = r0 + 32 * (MB * wm + m) + ln;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + 64 * b + 32 * wn + 8 * q + 4 * hh;
        if (row >= rows || n >= N) continue;
        const f32x4 v = {acc[m][b][4 * q], acc[m][b][4 * q + 1], acc[m][b][4 * q + 2], acc[m][b][4 * q + 3]};
        if (parts) *reinterpret_cast<f32x4*>(parts + ((int64_t)blockIdx.y * rows + row) * N + n) = v;
        else ff_store4(out + row * N + n, v[0], v[1], v[2], v[3]);
      }
  }
}

// ------------------------------------------------------------------------------------------------ weights' gradients
// Up to three products C[M, N] = sum over rows t of A[t, m] B[t, n], one behind the other in the grid; part `split` of a product goes
// over rows [split * per, ..) and leaves its sums in parts + split * part_step + at. `twice`: A or B has a second part, a_low or b_low
// elements on.
struct FfWeightJob {
  const void *A, *B;
  int64_t a_stride, b_stride, a_low, b_low, at;
  int M, N, tiles;  // tiles of 128 x 128
};
struct FfWeightJobs {
  FfWeightJob job[3];
  int n, splits;
  bool twice;
  int64_t rows, per, part_step;
};

template <typename T>
__global__ void __launch_bounds__(MM_BLOCK, 2) ff_weights_kernel(const FfWeightJobs jobs, float* __restrict__ parts) {
  constexpr int BK = 128 / sizeof(T);  // rows of a step
  constexpr int EPC = 16 / sizeof(T), CPR = 128 / EPC, CH = BK * CPR / MM_BLOCK;
  __shared__ __attribute__((aligned(16))) T lds[2][2][BK * 128];
  int tile = blockIdx.x, j = 0;
  while (j + 1 < jobs.n && tile >= jobs.job[j].tiles) tile -= jobs.job[j++].tiles;
  const FfWeightJob& job = jobs.job[j];
  const int ntiles = (job.N + 127) / 128, m0 = tile / ntiles * 128, n0 = tile % ntiles * 128;
  const int64_t begin = (int64_t)blockIdx.y * jobs.per, end = begin + jobs.per < jobs.rows ? begin + jobs.per : jobs.rows;
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  f32x16 acc[2][2];
  mm_clear(acc);
  // Rows of 128 columns in LDS, their pieces permuted so that the rows of an operand read meet in no bank. 16 bits: a read takes 64
  // bytes of each of 8 rows, 16 lanes 32 bytes of 4 rows; 32 bytes of row r go to place ^ twist(r % 4) of 8, different in
  // any 128 bytes for the 4 rows and in 256 for both halves. fp32: the lane halves read 128 bytes of rows 4 apart.
  auto twist = [](int r) { return (r << 1) ^ (r & 1) ^ (r >> 1); };
  const T *A = (const T*)job.A, *B = (const T*)job.B;
  auto fetch = [&](int64_t t0, T* to) {
    const int64_t n = end - t0 < BK ? end - t0 : BK;
    const __amdgpu_buffer_rsrc_t ab = ff_buffer(A + t0 * job.a_stride + m0, ((n - 1) * job.a_stride + job.M - m0) * (int64_t)sizeof(T));
    const __amdgpu_buffer_rsrc_t bb = ff_buffer(B + t0 * job.b_stride + n0, ((n - 1) * job.b_stride + job.N - n0) * (int64_t)sizeof(T));
    const int row = tid / CPR, piece = tid % CPR, c = (sizeof(T) == 2 ? piece ^ (twist(row & 3) << 1) : piece ^ ((row & 4) << 1)) * EPC;
    unsigned char* p = reinterpret_cast<unsigned char*>(to) + __builtin_amdgcn_readfirstlane(wave) * 1024;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int r = row + i * (MM_BLOCK / CPR);
      mm_load_lds(ab, p + i * 4096, m0 + c < job.M ? (unsigned)((r * job.a_stride + c) * sizeof(T)) : FF_OFF);
      mm_load_lds(bb, p + BK * 128 * sizeof(T) + i * 4096, n0 + c < job.N ? (unsigned)((r * job.b_stride + c) * sizeof(T)) : FF_OFF);
    }
  };
  auto operand = [&](const T* arr, int col0, int row0) -> ff_u32x4 {
    if constexpr (sizeof(T) == 2) {  // as op_ld_kappa_tr takes it
      const int L = lane & 15;
      const T* q = arr + (row0 + 4 * hh + (L >> 2)) * 128 + ((col0 / 16 + ((lane >> 4) & 1)) ^ twist(L >> 2)) * 16 + 4 * (L & 3);
      const typename OpVec<T>::x4 lo = op_lds_read_tr4<T>(q), hi = op_lds_read_tr4<T>(q + 8 * 128);
      typename OpVec<T>::x8 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = lo[e]; v[4 + e] = hi[e]; }
      return __builtin_bit_cast(ff_u32x4, v);
    } else {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = arr[(row0 + 4 * hh + e) * 128 + (col0 ^ (32 * hh)) + ln];
      return __builtin_bit_cast(ff_u32x4, v);
    }
  };
  for (int part = 0; part < (jobs.twice ? 2 : 1) && begin < end; ++part) {
    if (part) {
      A += job.a_low;
      B += job.b_low;
      lds_barrier();  // the first part's last rows have been read
    }
    fetch(begin, lds[0][0]);
    int which = 0;
    for (int64_t t0 = begin; t0 < end; t0 += BK, which ^= 1) {
      // this step's rows are there for all waves, and the last step's are free
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();
      // the next step's rows go to `there`, this step's are at `here`: told apart, so that reads do not wait for the loads
      auto step = [&](T* __restrict__ there, const T* __restrict__ here) {
        if (t0 + BK < end) fetch(t0 + BK, there);
        ff_u32x4 fa[2][2], fb[2][2];
        auto read = [&](int ks) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            fa[ks & 1][k] = operand(here, 64 * wm + 32 * k, ks * BK / 4);
            fb[ks & 1][k] = operand(here + BK * 128, 64 * wn + 32 * k, ks * BK / 4);
          }
        };
        read(0);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          if (ks + 1 < 4) read(ks + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int b = 0; b < 2; ++b) acc[m][b] = mm_mac<T>(fb[ks & 1][b], fa[ks & 1][m], acc[m][b]);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      step(lds[which ^ 1][0], lds[which][0]);
    }
  }
  float* out = parts + blockIdx.y * jobs.part_step + job.at;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int row = m0 + 64 * wm + 32 * m + ln;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + 64 * wn + 32 * b + 8 * q + 4 * hh;
        if (row < job.M && n < job.N)
          *reinterpret_cast<f32x4*>(out + (int64_t)row * job.N + n) =
              f32x4{acc[m][b][4 * q], acc[m][b][4 * q + 1], acc[m][b][4 * q + 2], acc[m][b][4 * q + 3]};
      }
  }
}

// ------------------------------------------------------------------------------------------------ small kernels
// The parts of up to three gradients (one behind the other in a part) in order, in one launch.
template <typename T>
struct FfSums {
  T* out[3];
};
template <typename T>
__global__ void __launch_bounds__(256) ff_sums_kernel(const float* __restrict__ parts, int n, int64_t cols, int64_t step, FfSums<T> to) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= cols) return;
  const float* p = parts + blockIdx.y * cols + c;
  f32x4 sum = *reinterpret_cast<const f32x4*>(p);
  for (int r = 1; r < n; ++r) sum += *reinterpret_cast<const f32x4*>(p + r * step);
  ff_store4(to.out[blockIdx.y] + c, sum[0], sum[1], sum[2], sum[3]);
}

// out [cols, rows] = in [rows, cols]^T in tiles of 32 x 32; three matrices side by side in the grid's third dimension.
struct FfTurns {
  const void* in[3];
  void* out[3];
  int rows[3], cols[3];
};
template <typename T>
__global__ void __launch_bounds__(256) ff_turn_kernel(const FfTurns t) {
  __shared__ T tile[32][33];
  const int z = blockIdx.z, rows = t.rows[z], cols = t.cols[z], r0 = blockIdx.y * 32, c0 = blockIdx.x * 32;
  if (r0 >= rows || c0 >= cols) return;
  const T* in = (const T*)t.in[z];
  T* out = (T*)t.out[z];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < 32; k += 8)
    if (r0 + y + k < rows && c0 + x < cols) tile[y + k][x] = in[(int64_t)(r0 + y + k) * cols + c0 + x];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 32; k += 8)
    if (c0 + y + k < cols && r0 + x < rows) out[(int64_t)(c0 + y + k) * rows + r0 + x] = tile[x][y + k];
}

// ------------------------------------------------------------------------------------------------ host
static int64_t ff_size(const lampa_ff_args* a) { return a->dtype == GDR_FP32 ? 4 : 2; }
static int64_t ff_area(int64_t n, int64_t elem) { return lampa_align_up(n * elem, 256); }

// Parts of the weights' gradients: as many as make about two workgroups a CU, of 256 rows or more each.
static int ff_splits(const lampa_ff_args* a) {
  const int64_t tiles = ((a->F + 127) / 128) * (int64_t)((a->D + 127) / 128) * ((a->dw_gate != nullptr) + (a->dw_up != nullptr) + (a->dw_down != nullptr));
  const int64_t want = tiles ? (512 + tiles - 1) / tiles : 1, most = (a->rows + 255) / 256;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

// Rows of a tile (64 times this). 128 where that leaves a workgroup a CU (16 bits: y and dx of 8 192 x 768, 384 tiles, 62 us on average
// against 69; of 4 100 x 1 024, 264 tiles, 53 against 59; hidden of 1 280 rows, 320 tiles, 16 against 17), in fp32, whose products
// take 16 times as long, where it leaves two (gradients of 2 000 rows, D = 512, F = 1024: 67 us with tiles of 128 from one on,
// 63 so); else 64, so that few rows spread over the GPU.
static int ff_row_blocks(const lampa_ff_args* a, int cols, int wide) {
  return (a->rows + 127) / 128 * ((cols + wide - 1) / wide) >= (a->dtype == GDR_FP32 ? 512 : 256) ? 2 : 1;
}
// How a product's contraction is shared out: where its tiles leave CUs idle, over as many workgroups as fill them, of 4 steps or more.
struct FfSplit {
  int mb, n, span;
};
static FfSplit ff_split(const lampa_ff_args* a) {
  FfSplit s;
  s.mb = ff_row_blocks(a, a->D, 128);
  const int64_t tiles = (a->rows + 64 * s.mb - 1) / (64 * s.mb) * ((a->D + 127) / 128);
  const int step = MM_ROW_BYTES / (int)ff_size(a), steps = (a->F + step - 1) / step;
  const int64_t want = tiles ? 256 / tiles : 1;
  int n = (int)(want < steps / 4 ? want : steps / 4);
  if (n < 1) n = 1;
  const int per = (steps + n - 1) / n;
  s.n = (steps + per - 1) / per;
  s.span = per * step;
  return s;
}

// 16-bit hidden values and their gradients as two parts, their rounding and what it left, where the rows are no more than a tile's: what
// outputs are off by would else hang on a handful of roundings (by the norm, over the output's own rounding: one row of 136, 32 hidden
// columns, up to 2.2, 21 rows up to 1.7, 128 rows up to 1.5; 1.41 on average at any number). The last products take twice the operations: at 64 rows x
// 768, 2 048 hidden columns, bf16, 11 us against 9 and the call 22 against 20, at 32 rows 20.6 against 20.1; at 512 27 against 23, not done.
#define FF_TWO_ROWS 64
static bool ff_two(const lampa_ff_args* a) { return a->dtype != GDR_FP32 && a->rows <= FF_TWO_ROWS; }

struct FfAreas {
  int64_t low;  // elements from a hidden value to its second part, 0: none
  int64_t hidden, dg, du, turned, sums, parts, total;  // turned: Wd^T, Wg^T, Wu^T one behind the other
};
static FfAreas ff_areas(const lampa_ff_args* a, int backward) {
  const int64_t e = ff_size(a), one = ff_area(a->rows * a->F, e), h = ff_two(a) ? 2 * one : one, w = ff_area((int64_t)a->D * a->F, e);
  const FfSplit sp = ff_split(a);
  FfAreas l{};
  l.low = ff_two(a) ? one / e : 0;
  l.hidden = 0;
  l.dg = h;
  l.du = l.dg + (backward ? h : 0);
  l.turned = l.du + (backward ? h : 0);
  l.sums = l.turned + (backward ? 3 * w : 0);
  l.parts = l.sums + (sp.n > 1 ? ff_area((int64_t)sp.n * a->rows * a->D, 4) : 0);
  l.total = l.parts + (backward ? ff_area((int64_t)ff_splits(a) * 3 * a->D * a->F, 4) : 0);
  return l;
}
int64_t ff_gemm_workspace(const lampa_ff_args* a, int backward) { return ff_areas(a, backward).total; }

static unsigned ff_tiles(int64_t rows, int mb, int cols, int wide) {
  return (unsigned)((rows + 64 * mb - 1) / (64 * mb) * ((cols + wide - 1) / wide));
}

// Tiles shared out by columns: where Wg and Wu together are more than half an XCD's L2 of 4 MB and there are two tiles or more for
// each (8 192 x 768, F = 2048: hidden 69 us against 72, grads 121 against 130).
static bool ff_by_columns(const lampa_ff_args* a) { return 2 * (int64_t)a->D * a->F * ff_size(a) > 1 << 21 && a->F >= 1024; }
static unsigned ff_column_tiles(int64_t rows, int mb, int F) {
  return (unsigned)(8 * (((F + 63) / 64 + 7) / 8) * ((rows + 64 * mb - 1) / (64 * mb)));
}

#define FF_ROWS(MB, GO) \
  if ((MB) == 1) GO(1); else GO(2);

template <typename T>
static int ff_product_go(const lampa_ff_args* a, const T* a0, const T* b0, const T* a1, const T* b1, int64_t low, T* out, float* sums,
                         hipStream_t s) {
  const FfSplit sp = ff_split(a);
#define FF_GO(MB)                                                                                                                   \
  hipLaunchKernelGGL((ff_product_kernel<T, MB>), dim3(ff_tiles(a->rows, MB, a->D, 128), (unsigned)sp.n), dim3(MM_BLOCK), 0, s, a0, b0, a1, \
                     b1, low, a->rows, a->D, a->F, sp.span, out, sp.n > 1 ? sums : (float*)nullptr)
  FF_ROWS(sp.mb, FF_GO)
#undef FF_GO
  LAMPA_PROF(s, "ff_product_kernel");
  const int rc = lampa_launch_status();
  if (rc != LAMPA_OK || sp.n == 1) return rc;
  return ff_reduce<T>(sums, sp.n, a->rows * a->D, a->rows * a->D, out, s);
}

template <typename T, int ACT>
static int ff_fwd_go(const lampa_ff_args* a, hipStream_t s) {
  const FfAreas l = ff_areas(a, 0);
  T* hidden = (T*)a->workspace;
  const bool columns = ff_by_columns(a);
  LAMPA_PROF(s, "start");
#define FF_GO(MB)                                                                                                                    \
  hipLaunchKernelGGL((ff_hidden_kernel<T, ACT, MB>), dim3(columns ? ff_column_tiles(a->rows, MB, a->F) : ff_tiles(a->rows, MB, a->F, 64)), dim3(MM_BLOCK), 0, s, (const T*)a->x, a->x_stride, \
                     (const T*)a->w_gate, (const T*)a->w_up, a->rows, a->D, a->F, hidden, l.low, columns)
  FF_ROWS(ff_row_blocks(a, a->F, 64), FF_GO)
#undef FF_GO
  LAMPA_PROF(s, "ff_hidden_kernel");
  const int rc = lampa_launch_status();
  if (rc != LAMPA_OK) return rc;
  return ff_product_go<T>(a, hidden, (const T*)a->w_down, nullptr, nullptr, l.low, (T*)a->y, (float*)((char*)a->workspace + l.sums), s);
}

template <typename T, int ACT>
static int ff_bwd_go(const lampa_ff_args* a, hipStream_t s) {
  const FfAreas l = ff_areas(a, 1);
  char* ws = (char*)a->workspace;
  const int64_t w = ff_area((int64_t)a->D * a->F, sizeof(T));
  T *hidden = (T*)(ws + l.hidden), *dg = (T*)(ws + l.dg), *du = (T*)(ws + l.du);
  T *wd_t = (T*)(ws + l.turned), *wg_t = (T*)(ws + l.turned + w), *wu_t = (T*)(ws + l.turned + 2 * w);
  float* parts = (float*)(ws + l.parts);
  const bool weights = a->dw_gate || a->dw_up || a->dw_down, columns = ff_by_columns(a);
  LAMPA_PROF(s, "start");
  const FfTurns turns{{a->w_down, a->w_gate, a->w_up}, {wd_t, wg_t, wu_t}, {a->D, a->F, a->F}, {a->F, a->D, a->D}};
  const int most = a->D > a->F ? a->D : a->F;
  hipLaunchKernelGGL((ff_turn_kernel<T>), dim3((most + 31) / 32, (most + 31) / 32, a->dx ? 3 : 1), dim3(256), 0, s, turns);
  LAMPA_PROF(s, "ff_turn_kernel");
#define FF_GO(MB)                                                                                                                     \
  hipLaunchKernelGGL((ff_grads_kernel<T, ACT, MB>), dim3(columns ? ff_column_tiles(a->rows, MB, a->F) : ff_tiles(a->rows, MB, a->F, 64)), dim3(MM_BLOCK), 0, s, (const T*)a->x, a->x_stride, \
                     (const T*)a->dy, (const T*)a->w_gate, (const T*)a->w_up, (const T*)wd_t, a->rows, a->D, a->F,                          \
                     a->dw_down ? hidden : (T*)nullptr, dg, du, l.low, columns)
  FF_ROWS(ff_row_blocks(a, a->F, 64), FF_GO)
#undef FF_GO
  LAMPA_PROF(s, "ff_grads_kernel");
  int rc = lampa_launch_status();
  if (rc != LAMPA_OK) return rc;
  if (a->dx) {
    rc = ff_product_go<T>(a, dg, wg_t, du, wu_t, l.low, (T*)a->dx, (float*)(ws + l.sums), s);
    if (rc != LAMPA_OK) return rc;
  }
  if (!weights) return LAMPA_OK;
  FfWeightJobs jobs{};
  jobs.splits = ff_splits(a);
  jobs.rows = a->rows;
  jobs.twice = l.low != 0;
  jobs.per = lampa_align_up((a->rows + jobs.splits - 1) / jobs.splits, 64);
  const int64_t size = (int64_t)a->D * a->F;
  FfSums<T> outs{};
  int tiles = 0;
  auto add = [&](void* out, const void* A, int64_t as, int64_t a_low, const void* B, int64_t bs, int64_t b_low, int M, int N) {
    if (!out) return;
    FfWeightJob& j = jobs.job[jobs.n];
    j = FfWeightJob{A, B, as, bs, a_low, b_low, jobs.n * size, M, N, (M + 127) / 128 * ((N + 127) / 128)};
    tiles += j.tiles;
    outs.out[jobs.n++] = (T*)out;
  };
  add(a->dw_gate, dg, a->F, l.low, a->x, a->x_stride, 0, a->F, a->D);
  add(a->dw_up, du, a->F, l.low, a->x, a->x_stride, 0, a->F, a->D);
  add(a->dw_down, a->dy, a->D, 0, hidden, a->F, l.low, a->D, a->F);
  jobs.part_step = jobs.n * size;
  hipLaunchKernelGGL((ff_weights_kernel<T>), dim3((unsigned)tiles, (unsigned)jobs.splits), dim3(MM_BLOCK), 0, s, jobs, parts);
  LAMPA_PROF(s, "ff_weights_kernel");
  hipLaunchKernelGGL((ff_sums_kernel<T>), dim3((unsigned)((size / 4 + 255) / 256), (unsigned)jobs.n), dim3(256), 0, s, parts, jobs.splits,
                     size, jobs.part_step, outs);
  LAMPA_PROF(s, "ff_sums_kernel");
  return lampa_launch_status();
}

#define FF_TYPES(GO)                                                                                               \
  switch (a->dtype * 3 + a->activation) {                                                                          \
    case 0: return GO<__bf16, 0>(a, s);                                                                            \
    case 1: return GO<__bf16, 1>(a, s);                                                                            \
    case 2: return GO<__bf16, 2>(a, s);                                                                            \
    case 3: return GO<_Float16, 0>(a, s);                                                                          \
    case 4: return GO<_Float16, 1>(a, s);                                                                          \
    case 5: return GO<_Float16, 2>(a, s);                                                                          \
    case 6: return GO<float, 0>(a, s);                                                                             \
    case 7: return GO<float, 1>(a, s);                                                                             \
    default: return GO<float, 2>(a, s);                                                                            \
  }
int ff_gemm_fwd(const lampa_ff_args* a, hipStream_t s) { FF_TYPES(ff_fwd_go) }
int ff_gemm_bwd(const lampa_ff_args* a, hipStream_t s) { FF_TYPES(ff_bwd_go) }
