// The gated feed-forward block for 16-bit types and narrow blocks (D <= 128): hidden values never leave the registers
// (ff_common.h has the mathematics).
//   out:      y (or, BACK, dx): a wave keeps 32 rows of x (and dy) as operands and their outputs as sums; the hidden columns pass in
//             chunks of 32, whose weights the workgroup's waves share in LDS (the next chunk under way in registers). Products are
//             formed transposed, hidden columns x rows: the sums of the first products, rounded, are then the operands of the next as
//             they lie in the registers.
//   weights:  a wave keeps 32 hidden columns (their weights as operands, the sums of the three gradients: 16 DB values a lane each)
//             and the rows pass in tiles of 32 in LDS; workgroups share the rows out and leave their sums in fp32.
//   reduce:   the parts of the weights' gradients in order, dWd turned on the way.
// Few rows: the chunks of hidden columns are shared out as well, and the outputs' parts summed in order.
//
// Measured, 60 000 rows x 128, 512 hidden columns, bf16 (a large product of the library reaches 1.3 .. 1.6 PFLOP/s on this card):
// y 31 us (23.6 GFLOP, 0.76 PFLOP/s; its products alone, without operand reads, loads or elementwise part, 17 and reading x and writing y
// 8), dx 49 us (39 GFLOP with the first products again), gradients of the weights 77 us (47 GFLOP) and 9 for their parts' sums (50 MB;
// medians of a kernel trace, calls back to back take 28 us forward).
// With 4 waves a workgroup y takes 34 us, with two blocks of 32 rows a wave and one wave a SIMD 42. The weights' kernel holds 192 sums
// and 96 operands a lane, one wave a SIMD, so its products, its elementwise part and its LDS reads come one after the other; keeping
// another tile's operands to overlap them spills (125 .. 280 us).
// One token: two kernels of 5.4 and 5.1 us behind 16 on the host.
// Built once for each type (ff_fused_bf16.hip, ff_fused_fp16.hip), side by side.
#pragma once
#include "ff_common.h"

#define FU_BLOCK 256
#define FU_WIDE 8   // waves of a workgroup of `out` where the rows fill the GPU
#define FU_AHEAD 2  // steps that operands are read ahead of their products
#define FU_CHUNK 32  // hidden columns of a chunk

template <typename T>
__device__ __forceinline__ typename OpVec<T>::x8 fu_op(ff_u32x4 v) { return __builtin_bit_cast(typename OpVec<T>::x8, v); }

// A row's share of an operand: 16 bytes at column c of a row-major matrix of D columns; zero behind them.
__device__ __forceinline__ ff_u32x4 fu_load(__amdgpu_buffer_rsrc_t buf, unsigned row_bytes, int c, int D) {
  return ff_load16(buf, c < D ? row_bytes + (unsigned)c * 2 : FF_OFF);
}

// v as element i of an operand, and, TWO, what its rounding left as that of another (none where there is no finite rest).
template <bool TWO, typename T>
__device__ __forceinline__ void fu_parts(float v, T& high, T& low, int i) {
  const auto h = (__typeof__(high[0]))v;
  high[i] = h;
  if constexpr (TWO) {
    const float rest = v - (float)h;
    low[i] = (__typeof__(high[0]))(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f);
  }
}

struct FuOut {
  const void *x, *dy, *wg, *wu, *wd;
  void* out;     // [rows, D] of the type, or
  float* parts;  // [splits, rows, D]
  int64_t rows, x_stride;
  int D, F, chunks;  // chunks of a workgroup
};

// Row-major tiles of up to 128 columns that are read both along their rows (16 bytes a lane, 32 rows side by side) and turned (four rows
// of 16 columns for each 16 lanes): the 16-byte pieces of a row are permuted by three bits of the row, piece ^ fu_twist(row), so
// that neither kind of read meets itself in a bank. Rows are a multiple of 128 bytes.
__device__ __forceinline__ int fu_twist(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }
template <typename T, int STRIDE>
__device__ __forceinline__ void fu_put(T* tile, int row, int c, ff_u32x4 v) {
  *reinterpret_cast<ff_u32x4*>(tile + row * STRIDE + ((c >> 3) ^ fu_twist(row)) * 8) = v;
}
// Row `row`, columns c .. c + 7.
template <typename T, int STRIDE>
__device__ __forceinline__ typename OpVec<T>::x8 fu_along(const T* tile, int row, int c) {
  return *reinterpret_cast<const typename OpVec<T>::x8*>(tile + row * STRIDE + ((c >> 3) ^ fu_twist(row)) * 8);
}
// A 16-wide step's operand whose rows are the 32 columns col0 .. of a tile and whose contraction runs over the tile's rows row0 .., in
// slot order (op_ld_kappa_tr of gdr_ops.h on a permuted tile).
template <typename T, int STRIDE>
__device__ __forceinline__ typename OpVec<T>::x8 fu_turned(const T* tile, int col0, int row0, int lane) {
  const int L = lane & 15, blk = (lane >> 4) & 1, hh = lane >> 5, row = row0 + 4 * hh + (L >> 2);
  const int piece = (col0 >> 3) + 2 * blk + ((L & 3) >> 1);
  const T* p = tile + row * STRIDE + (piece ^ fu_twist(row)) * 8 + (L & 1) * 4;
  const typename OpVec<T>::x4 lo = op_lds_read_tr4<T>(p), hi = op_lds_read_tr4<T>(p + 8 * STRIDE);  // 8 rows on: the same twist
  typename OpVec<T>::x8 out;
#pragma unroll
  for (int s = 0; s < 4; ++s) { out[s] = lo[s]; out[4 + s] = hi[s]; }
  return out;
}

// WAVES waves of 32 rows each. With 4, where the GPU has room (fu_share), hidden values enter the last products as two parts, their
// rounding and what it left: what a few outputs are off by would else hang on a handful of roundings (one token of 128 columns: up to
// 1.6 times the output's own rounding). With FU_WIDE, as one: their roundings, as large as the output's own, cost a third of the time.
template <typename T, int ACT, int DB, int WAVES, bool BACK>
__global__ void __launch_bounds__(64 * WAVES, WAVES == 4 ? 1 : 2) ff_out_kernel(const FuOut a) {
  typedef typename OpVec<T>::x8 x8;
  typedef typename OpVec<T>::x4 x4;
  constexpr bool TWO = WAVES == 4;
  constexpr int KS = 2 * DB, WIDE = DB * 32, GS = (DB + 1) / 2 * 64, DS = BACK ? 32 : 40;  // elements between the rows of the tiles
  constexpr int BLOCK = 64 * WAVES, PIECES = 128 * DB, LOADS = (PIECES + BLOCK - 1) / BLOCK;  // 16-byte pieces of each matrix's chunk
  constexpr int STAGE = 2 * FU_CHUNK * GS + WIDE * DS, ROWS = 32 * WAVES;
  // BACK: two chunks; forward: three. At the end 32 rows of outputs for each wave.
  constexpr int LOOP = (BACK ? 2 : 3) * STAGE, OUTS = WAVES * 32 * (WIDE + 8), LDS = LOOP > OUTS ? LOOP : OUTS;
  __shared__ __attribute__((aligned(16))) T lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6;
  const int D = a.D, F = a.F;
  const int64_t r0 = (int64_t)blockIdx.x * ROWS;
  const int64_t left = a.rows - r0;
  const int here = left < ROWS ? (int)left : ROWS;
  const int c0 = blockIdx.y * a.chunks, all = (F + FU_CHUNK - 1) / FU_CHUNK, c1 = c0 + a.chunks < all ? c0 + a.chunks : all;

  ff_u32x4 rg[LOADS], ru[LOADS], rd[LOADS];
  // where this thread's pieces lie in a chunk, and in its tiles
  unsigned from[LOADS], from_down[LOADS];
  int at[LOADS], at_down[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int id = tid + i * BLOCK, row = id / (DB * 4), c = id % (DB * 4) * 8, d = id / 4, f = id % 4 * 8;
    from[i] = c < D ? (unsigned)(row * D + c) * 2 : FF_OFF;
    from_down[i] = d < D ? (unsigned)(d * F + f) * 2 : FF_OFF;
    at[i] = row * GS + ((c >> 3) ^ fu_twist(row)) * 8;
    at_down[i] = 2 * FU_CHUNK * GS + d * DS + (BACK ? f ^ (d & 2 ? 16 : 0) : f);  // BACK: read turned, rows 2, 3 of four the other way round
  }
  auto fetch = [&](int chunk) {
    const int f0 = chunk * FU_CHUNK, n = F - f0 < FU_CHUNK ? F - f0 : FU_CHUNK;
    const __amdgpu_buffer_rsrc_t gb = ff_buffer((const T*)a.wg + (int64_t)f0 * D, (int64_t)n * D * 2);
    const __amdgpu_buffer_rsrc_t ub = ff_buffer((const T*)a.wu + (int64_t)f0 * D, (int64_t)n * D * 2);
    const __amdgpu_buffer_rsrc_t db = ff_buffer((const T*)a.wd + f0, ((int64_t)(D - 1) * F + n) * 2);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if (PIECES % BLOCK && tid + i * BLOCK >= PIECES) break;
      rg[i] = ff_load16(gb, from[i]);
      ru[i] = ff_load16(ub, from[i]);
    }
    if (n == FU_CHUNK) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) rd[i] = ff_load16(db, from_down[i]);
    } else {  // the columns behind the last are the next row's
#pragma unroll
      for (int i = 0; i < LOADS; ++i) rd[i] = ff_load16(db, tid % 4 * 8 < n ? from_down[i] : FF_OFF);
    }
  };
  auto stage = [&](int which) {
    T* p = lds + which * STAGE;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if (PIECES % BLOCK && tid + i * BLOCK >= PIECES) break;
      *reinterpret_cast<ff_u32x4*>(p + at[i]) = rg[i];
      *reinterpret_cast<ff_u32x4*>(p + FU_CHUNK * GS + at[i]) = ru[i];
      *reinterpret_cast<ff_u32x4*>(p + at_down[i]) = rd[i];
    }
  };
  // Wd as the operand whose rows are the chunk's hidden columns, contraction over its rows d0 .. in slot order
  auto down_turned = [&](const T* w, int d0) {
    const int L = lane & 15, blk = (lane >> 4) & 1, row = d0 + 4 * hh + (L >> 2);
    const T* p = w + row * DS + ((16 * blk + 4 * (L & 3)) ^ (row & 2 ? 16 : 0));
    const x4 lo = op_lds_read_tr4<T>(p), hi = op_lds_read_tr4<T>(p + 8 * DS);
    return x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  // Row of a chunk's Wg and Wu that is row ln of the first products: chosen so that the 8 sums a lane holds for a step of the last
  // product are 8 hidden columns in line, as Wd has them (BACK reads Wd and both turned, in the order the sums lie in anyway).
  const int gl = BACK ? ln : (ln & 16) | ((ln & 4) << 1) | ((ln & 8) >> 1) | (ln & 3);
  fetch(c0);
  // this wave's rows
  x8 xo[KS], dyo[BACK ? KS : 1];
  {
    const int row = 32 * wave + ln;
    const __amdgpu_buffer_rsrc_t xb = ff_buffer((const T*)a.x + r0 * a.x_stride, ((here - 1) * a.x_stride + D) * 2);
#pragma unroll
    for (int k = 0; k < KS; ++k)
      xo[k] = fu_op<T>(fu_load(xb, row < here ? (unsigned)(row * a.x_stride) * 2 : FF_OFF, 16 * k + 8 * hh, D));
    if constexpr (BACK) {
      const __amdgpu_buffer_rsrc_t yb = ff_buffer((const T*)a.dy + r0 * D, (int64_t)here * D * 2);
#pragma unroll
      for (int k = 0; k < KS; ++k) {  // in slot order: 4 columns at 16 k + 4 hh, 4 more 8 columns on
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
        const int c = 16 * k + 4 * hh;
        const unsigned at = row < here ? (unsigned)(row * D) * 2 : FF_OFF;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(yb, c < D ? at + c * 2 : FF_OFF, 0, 0));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(yb, c + 8 < D ? at + (c + 8) * 2 : FF_OFF, 0, 0));
        dyo[k] = fu_op<T>(ff_u32x4{lo[0], lo[1], hi[0], hi[1]});
      }
    }
  }
  f32x16 out[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) out[d][r] = 0.0f;
  stage(0);
  ff_loads_done();
  if (c0 + 1 < c1) fetch(c0 + 1);
  lds_barrier();
  if constexpr (!BACK) {
    // Chunk c + 1's first products run while chunk c's elementwise part does, pinned side by side in steps: the matrix cores work
    // through a product while the wave issues what does not depend on it.
    f32x16 Ga, Ua, Gb, Ub;
    auto first = [&](const T* g, f32x16& G, f32x16& U, auto between) {
      const T* u = g + FU_CHUNK * GS;
#pragma unroll
      for (int r = 0; r < 16; ++r) G[r] = U[r] = 0.0f;
      x8 ga[KS], ua[KS];
#pragma unroll
      for (int k = 0; k < KS + FU_AHEAD; ++k) {
        if (k < KS) {
          ga[k] = fu_along<T, GS>(g, gl, 16 * k + 8 * hh);
          ua[k] = fu_along<T, GS>(u, gl, 16 * k + 8 * hh);
        }
        if (k >= FU_AHEAD) {
          const int m = k - FU_AHEAD;
          G = mfma32(ga[m], xo[m], G);
          U = mfma32(ua[m], xo[m], U);
          between(m);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    int slot = 0;  // of the chunk being finished
    auto next_slot = [](int s) { return s == 2 ? 0 : s + 1; };
    auto one = [&](int chunk, f32x16& G, f32x16& U, f32x16& G1, f32x16& U1) {
      const int s1 = next_slot(slot), s2 = next_slot(s1);
      if (chunk + 2 < c1) stage(s2);  // requested a whole chunk ago
      if (chunk + 3 < c1) fetch(chunk + 3);
      const T* w = lds + slot * STAGE + 2 * FU_CHUNK * GS;
      x8 h[2], low[2];
      auto act = [&](int k) {
#pragma unroll
        for (int r = 16 * k / KS; r < 16 * (k + 1) / KS; ++r) fu_parts<TWO>(ff_act<ACT>(G[r]) * U[r], h[r / 8], low[r / 8], r % 8);
      };
      if (chunk + 1 < c1) {
        first(lds + s1 * STAGE, G1, U1, act);
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) act(k);
      }
      x8 da[2 * DB];
#pragma unroll
      for (int m = 0; m < 2 * DB + FU_AHEAD; ++m) {
        if (m < 2 * DB) da[m] = *reinterpret_cast<const x8*>(w + (32 * (m % DB) + ln) * DS + 16 * (m / DB) + 8 * hh);
        if (m >= FU_AHEAD) {
          const int n = m - FU_AHEAD;
          out[n % DB] = mfma32(da[n], h[n / DB], out[n % DB]);
          if constexpr (TWO) out[n % DB] = mfma32(da[n], low[n / DB], out[n % DB]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      lds_barrier();
      slot = s1;
    };
    first(lds, Ga, Ua, [](int) {});
    if (c0 + 1 < c1) stage(1);
    if (c0 + 2 < c1) fetch(c0 + 2);
    lds_barrier();
    for (int chunk = c0; chunk < c1; chunk += 2) {
      one(chunk, Ga, Ua, Gb, Ub);
      if (chunk + 1 < c1) one(chunk + 1, Gb, Ub, Ga, Ua);
    }
  } else {
    for (int chunk = c0; chunk < c1; ++chunk) {
      const int which = (chunk - c0) & 1;
      if (chunk + 1 < c1) stage(which ^ 1);  // requested a whole chunk ago
      if (chunk + 2 < c1) fetch(chunk + 2);
      const T *g = lds + which * STAGE, *u = g + FU_CHUNK * GS, *w = u + FU_CHUNK * GS;
      f32x16 G, U, S;
#pragma unroll
      for (int r = 0; r < 16; ++r) G[r] = U[r] = S[r] = 0.0f;
      // operands are read FU_AHEAD steps ahead of their products, held there by the barriers (left to itself the compiler reads each just
      // before its product and waits)
      x8 ga[KS], ua[KS], wa[KS];
#pragma unroll
      for (int k = 0; k < KS + FU_AHEAD; ++k) {
        if (k < KS) {
          ga[k] = fu_along<T, GS>(g, gl, 16 * k + 8 * hh);
          ua[k] = fu_along<T, GS>(u, gl, 16 * k + 8 * hh);
          wa[k] = down_turned(w, 16 * k);
        }
        if (k >= FU_AHEAD) {
          const int m = k - FU_AHEAD;
          G = mfma32(ga[m], xo[m], G);
          U = mfma32(ua[m], xo[m], U);
          S = mfma32(wa[m], dyo[m], S);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      x8 da[2 * DB], db[2 * DB];
      auto last_operands = [&](int m) {
        da[m] = fu_turned<T, GS>(g, 32 * (m % DB), 16 * (m / DB), lane);
        db[m] = fu_turned<T, GS>(u, 32 * (m % DB), 16 * (m / DB), lane);
      };
#pragma unroll
      for (int m = 0; m < FU_AHEAD && m < 2 * DB; ++m) last_operands(m);
      __builtin_amdgcn_sched_barrier(0);
      x8 dg[2], du[2], dg_low[2], du_low[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float value, slope;
        ff_act_slope<ACT>(G[r], value, slope);
        fu_parts<TWO>(S[r] * U[r] * slope, dg[r / 8], dg_low[r / 8], r % 8);
        fu_parts<TWO>(S[r] * value, du[r / 8], du_low[r / 8], r % 8);
      }
#pragma unroll
      for (int m = 0; m < 2 * DB; ++m) {
        const int s = m / DB, d = m % DB;
        if (m + FU_AHEAD < 2 * DB) last_operands(m + FU_AHEAD);
        out[d] = mfma32(da[m], dg[s], out[d]);
        out[d] = mfma32(db[m], du[s], out[d]);
        if constexpr (TWO) {
          out[d] = mfma32(da[m], dg_low[s], out[d]);
          out[d] = mfma32(db[m], du_low[s], out[d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      lds_barrier();
    }
  }
  if (a.parts) {
    const int row = 32 * wave + ln;
    if (row >= here) return;
    float* p = a.parts + ((int64_t)blockIdx.y * a.rows + r0 + row) * D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = 32 * d + 8 * q + 4 * hh;
        if (c < D) *reinterpret_cast<f32x4*>(p + c) = f32x4{out[d][4 * q], out[d][4 * q + 1], out[d][4 * q + 2], out[d][4 * q + 3]};
      }
    return;
  }
  // through LDS (the tiles have been read), so that a row is written in pieces of 16 bytes side by side
  constexpr int OS = WIDE + 8;
  T* o = lds + wave * 32 * OS;
  const __amdgpu_buffer_rsrc_t ob = ff_buffer((T*)a.out + r0 * D, (int64_t)here * D * 2);
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      ff_store4(o + ln * OS + 32 * d + 8 * q + 4 * hh, out[d][4 * q], out[d][4 * q + 1], out[d][4 * q + 2], out[d][4 * q + 3]);
  lds_fence();
#pragma unroll
  for (int i = 0; i < 2 * DB; ++i) {
    const int id = lane + 64 * i, row = id / (DB * 4), c = id % (DB * 4) * 8;
    const ff_u32x4 v = *reinterpret_cast<const ff_u32x4*>(o + row * OS + c);
    __builtin_amdgcn_raw_buffer_store_b128(v, ob, c < D ? (unsigned)((32 * wave + row) * D + c) * 2 : FF_OFF, 0, 0);
  }
}

// ------------------------------------------------------------------------------------------------ weights' gradients
struct FuWeights {
  const void *x, *dy, *wg, *wu, *wd;
  float* parts;  // [splits, 3, F, D]: dWg, dWu, dWd^T
  int64_t rows, x_stride, per;  // rows of a workgroup, a multiple of 32
  int D, F;
};

// Up to FU_TWO_ROWS rows the hidden values and their gradients enter as two parts, as in `out`: sums of few rows hang on a handful of
// roundings (with one part, bf16, 1 row of 80 columns: 1.56 times the output's own rounding; 1.4 over many). The more rows
// a sum runs over, the nearer it keeps to their average, and the more the second part costs: x 128, 512 hidden columns, 4 096 rows 24 us
// against 21, 8 192 29 against 26, 60 000 91 against 70.
#define FU_TWO_ROWS 4096
template <typename T, int ACT, int DB, bool TWO>
__global__ void __launch_bounds__(FU_BLOCK, 1) ff_fused_weights_kernel(const FuWeights a) {
  typedef typename OpVec<T>::x8 x8;
  constexpr int KS = 2 * DB, XS = (DB + 1) / 2 * 64, TILE = 32 * XS;
  constexpr int PIECES = 128 * DB, LOADS = (PIECES + FU_BLOCK - 1) / FU_BLOCK;
  __shared__ __attribute__((aligned(16))) T lds[2][2 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6;
  const int D = a.D, F = a.F, f0 = blockIdx.x * 128 + 32 * wave, f = f0 + ln;
  const int64_t begin = (int64_t)blockIdx.y * a.per, end = begin + a.per < a.rows ? begin + a.per : a.rows;
  const int tiles = end > begin ? (int)((end - begin + 31) / 32) : 0;

  ff_u32x4 rx[LOADS], ry[LOADS];
  auto fetch = [&](int tile) {
    const int64_t t0 = begin + 32 * (int64_t)tile;
    const int n = end - t0 < 32 ? (int)(end - t0) : 32;
    const __amdgpu_buffer_rsrc_t xb = ff_buffer((const T*)a.x + t0 * a.x_stride, ((n - 1) * a.x_stride + D) * 2);
    const __amdgpu_buffer_rsrc_t yb = ff_buffer((const T*)a.dy + t0 * D, (int64_t)n * D * 2);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int id = tid + i * FU_BLOCK;
      if (PIECES % FU_BLOCK && id >= PIECES) break;
      const int row = id / (DB * 4), c = id % (DB * 4) * 8;
      rx[i] = fu_load(xb, row < n ? (unsigned)(row * a.x_stride) * 2 : FF_OFF, c, D);
      ry[i] = fu_load(yb, row < n ? (unsigned)(row * D) * 2 : FF_OFF, c, D);
    }
  };
  auto stage = [&](int which) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int id = tid + i * FU_BLOCK;
      if (PIECES % FU_BLOCK && id >= PIECES) break;
      const int row = id / (DB * 4), c = id % (DB * 4) * 8;
      fu_put<T, XS>(lds[which], row, c, rx[i]);
      fu_put<T, XS>(lds[which] + TILE, row, c, ry[i]);
    }
  };
  if (tiles) fetch(0);
  x8 wg[KS], wu[KS], wd[KS];
  {
    const __amdgpu_buffer_rsrc_t gb = ff_buffer(a.wg, (int64_t)F * D * 2), ub = ff_buffer(a.wu, (int64_t)F * D * 2);
    const __amdgpu_buffer_rsrc_t db = ff_buffer(a.wd, (int64_t)F * D * 2);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = 16 * k + 8 * hh;
      const unsigned at = f < F ? (unsigned)(f * D) * 2 : FF_OFF;
      wg[k] = fu_op<T>(fu_load(gb, at, c, D));
      wu[k] = fu_op<T>(fu_load(ub, at, c, D));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        wd[k][e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(db, f < F && c < D ? (unsigned)((c + e) * F + f) * 2 : FF_OFF, 0, 0));
    }
  }
  f32x16 dwg[DB], dwu[DB], dwd[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dwg[d][r] = dwu[d][r] = dwd[d][r] = 0.0f;
  if (tiles) {
    stage(0);
    ff_loads_done();
    if (tiles > 1) fetch(1);
    lds_barrier();
    for (int tile = 0; tile < tiles; ++tile) {
      const int which = tile & 1;
      if (tile + 1 < tiles) stage(which ^ 1);  // requested a whole tile ago
      if (tile + 2 < tiles) fetch(tile + 2);
      const T *x = lds[which], *y = x + TILE;
      f32x16 G, U, S;
#pragma unroll
      for (int r = 0; r < 16; ++r) G[r] = U[r] = S[r] = 0.0f;
      // operands are read FU_AHEAD steps ahead of their products, held there by the barriers (left to itself the compiler reads each
      // just before its product and waits)
      x8 xa[KS], ya[KS];
#pragma unroll
      for (int k = 0; k < KS + FU_AHEAD; ++k) {
        if (k < KS) {
          xa[k] = fu_along<T, XS>(x, ln, 16 * k + 8 * hh);
          ya[k] = fu_along<T, XS>(y, ln, 16 * k + 8 * hh);
        }
        if (k >= FU_AHEAD) {
          const int m = k - FU_AHEAD;
          G = mfma32(xa[m], wg[m], G);
          U = mfma32(xa[m], wu[m], U);
          S = mfma32(ya[m], wd[m], S);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      x8 xt[2 * DB], yt[2 * DB];
#pragma unroll
      for (int m = 0; m < FU_AHEAD && m < 2 * DB; ++m) {
        xt[m] = fu_turned<T, XS>(x, 32 * (m % DB), 16 * (m / DB), lane);
        yt[m] = fu_turned<T, XS>(y, 32 * (m % DB), 16 * (m / DB), lane);
      }
      __builtin_amdgcn_sched_barrier(0);
      x8 dg[2], du[2], h[2], dg_low[2], du_low[2], low[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float value, slope;
        ff_act_slope<ACT>(G[r], value, slope);
        fu_parts<TWO>(value * U[r], h[r / 8], low[r / 8], r % 8);
        fu_parts<TWO>(S[r] * value, du[r / 8], du_low[r / 8], r % 8);
        fu_parts<TWO>(S[r] * U[r] * slope, dg[r / 8], dg_low[r / 8], r % 8);
      }
#pragma unroll
      for (int m = 0; m < 2 * DB; ++m) {
        const int s = m / DB, d = m % DB, n = m + FU_AHEAD;
        if (n < 2 * DB) {
          xt[n] = fu_turned<T, XS>(x, 32 * (n % DB), 16 * (n / DB), lane);
          yt[n] = fu_turned<T, XS>(y, 32 * (n % DB), 16 * (n / DB), lane);
        }
        dwg[d] = mfma32(xt[m], dg[s], dwg[d]);
        dwu[d] = mfma32(xt[m], du[s], dwu[d]);
        dwd[d] = mfma32(yt[m], h[s], dwd[d]);
        if constexpr (TWO) {
          dwg[d] = mfma32(xt[m], dg_low[s], dwg[d]);
          dwu[d] = mfma32(xt[m], du_low[s], dwu[d]);
          dwd[d] = mfma32(yt[m], low[s], dwd[d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      lds_barrier();
    }
  }
  if (f >= F) return;
  float* p = a.parts + (int64_t)blockIdx.y * 3 * F * D + (int64_t)f * D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * d + 8 * q + 4 * hh;
      if (c >= D) continue;
      *reinterpret_cast<f32x4*>(p + c) = f32x4{dwg[d][4 * q], dwg[d][4 * q + 1], dwg[d][4 * q + 2], dwg[d][4 * q + 3]};
      *reinterpret_cast<f32x4*>(p + (int64_t)F * D + c) = f32x4{dwu[d][4 * q], dwu[d][4 * q + 1], dwu[d][4 * q + 2], dwu[d][4 * q + 3]};
      *reinterpret_cast<f32x4*>(p + 2 * (int64_t)F * D + c) = f32x4{dwd[d][4 * q], dwd[d][4 * q + 1], dwd[d][4 * q + 2], dwd[d][4 * q + 3]};
    }
}

// Sums of the parts in order, 32 x 32 of one gradient a workgroup; z = 2 is turned into [D, F].
template <typename T>
__global__ void __launch_bounds__(256) ff_fused_reduce_kernel(const float* __restrict__ parts, int n, int D, int F, T* dwg, T* dwu, T* dwd) {
  __shared__ float tile[32][33];
  const int z = blockIdx.z, f = blockIdx.y * 32 + threadIdx.x / 8, c = blockIdx.x * 32 + threadIdx.x % 8 * 4;
  T* out = z == 0 ? dwg : z == 1 ? dwu : dwd;
  if (!out) return;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (f < F && c < D) {
    const float* p = parts + ((int64_t)z * F + f) * D + c;
    const int64_t step = 3 * (int64_t)F * D;
    int i = 0;
    for (; i + 8 <= n; i += 8) {
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const f32x4*>(p + (i + k) * step);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[k];
    }
    for (; i < n; ++i) sum += *reinterpret_cast<const f32x4*>(p + i * step);
  }
  if (z < 2) {
    if (f < F && c < D) ff_store4(out + (int64_t)f * D + c, sum[0], sum[1], sum[2], sum[3]);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) tile[threadIdx.x % 8 * 4 + k][threadIdx.x / 8] = sum[k];
  __syncthreads();
  const int d = blockIdx.x * 32 + threadIdx.x / 8, f4 = blockIdx.y * 32 + threadIdx.x % 8 * 4;
  const float* t = &tile[threadIdx.x / 8][threadIdx.x % 8 * 4];
  if (d < D && f4 < F) ff_store4(out + (int64_t)d * F + f4, t[0], t[1], t[2], t[3]);
}

// ------------------------------------------------------------------------------------------------ host
// Rows: workgroups of 4 waves while those of 4 leave no CU with two (up to 32 768 rows), of 8 beyond (60 000 x 128: 29 us against 34: the
// weights of a chunk are staged for twice the rows). How the chunks of hidden columns are shared out: over one workgroup where the
// rows alone fill half the GPU (every further share writes and reads the outputs' fp32 parts), else over as many as make one
// workgroup a CU.
struct FuShare {
  int splits, chunks, waves;
};
static FuShare fu_share(const lampa_ff_args* a) {
  const int waves = a->rows > 128 * 256 ? FU_WIDE : 4;
  const int64_t tiles = (a->rows + 32 * waves - 1) / (32 * waves);
  const int all = (a->F + FU_CHUNK - 1) / FU_CHUNK;
  const int64_t want = tiles < 1 ? 1 : 256 / tiles;
  const int n = want < 1 || waves > 4 ? 1 : (want < all ? (int)want : all);
  const int chunks = (all + n - 1) / n;
  return {(all + chunks - 1) / chunks, chunks, waves};
}
// The rows of the weights' gradients: one workgroup of 128 hidden columns a CU.
static int fu_weight_splits(const lampa_ff_args* a) {
  const int64_t cols = (a->F + 127) / 128, want = (256 + cols - 1) / cols, most = (a->rows + 31) / 32;
  return (int)(want < 1 ? 1 : (want < most ? want : (most < 1 ? 1 : most)));
}

static int64_t fu_workspace(const lampa_ff_args* a, int backward) {
  const FuShare sh = fu_share(a);
  const int64_t outs = sh.splits > 1 ? lampa_align_up((int64_t)sh.splits * a->rows * a->D * 4, 256) : 0;
  return outs + (backward ? (int64_t)fu_weight_splits(a) * 3 * a->D * a->F * 4 : 0);
}

template <typename T, int ACT, bool BACK>
static int fu_out(const lampa_ff_args* a, hipStream_t s) {
  const FuShare sh = fu_share(a);
  T* out = (T*)(BACK ? a->dx : a->y);
  FuOut k{a->x, a->dy, a->w_gate, a->w_up, a->w_down, out, sh.splits > 1 ? (float*)a->workspace : nullptr, a->rows, a->x_stride, a->D, a->F, sh.chunks};
  const int rows = 32 * sh.waves;
  const dim3 grid((unsigned)((a->rows + rows - 1) / rows), (unsigned)sh.splits), block(64 * sh.waves);
#define FU_GO(DB)                                                                                       \
  if (sh.waves == 4) hipLaunchKernelGGL((ff_out_kernel<T, ACT, DB, 4, BACK>), grid, block, 0, s, k);          \
  else hipLaunchKernelGGL((ff_out_kernel<T, ACT, DB, FU_WIDE, BACK>), grid, block, 0, s, k);                  \
  break;
  switch ((a->D + 31) / 32) {
    case 1: FU_GO(1)
    case 2: FU_GO(2)
    case 3: FU_GO(3)
    default: FU_GO(4)
  }
#undef FU_GO
  LAMPA_PROF(s, BACK ? "ff_out_kernel_back" : "ff_out_kernel");
  const int rc = lampa_launch_status();
  if (rc != LAMPA_OK || sh.splits == 1) return rc;
  return ff_reduce<T>(k.parts, sh.splits, a->rows * a->D, a->rows * a->D, out, s);
}

template <typename T, int ACT>
static int fu_fwd_go(const lampa_ff_args* a, hipStream_t s) {
  LAMPA_PROF(s, "start");
  return fu_out<T, ACT, false>(a, s);
}
template <typename T, int ACT>
static int fu_bwd_go(const lampa_ff_args* a, hipStream_t s) {
  LAMPA_PROF(s, "start");
  if (a->dx) {
    const int rc = fu_out<T, ACT, true>(a, s);
    if (rc != LAMPA_OK) return rc;
  }
  if (!a->dw_gate && !a->dw_up && !a->dw_down) return LAMPA_OK;
  const FuShare sh = fu_share(a);
  const int64_t outs = sh.splits > 1 ? lampa_align_up((int64_t)sh.splits * a->rows * a->D * 4, 256) : 0;
  const int n = fu_weight_splits(a);
  FuWeights k{a->x, a->dy, a->w_gate, a->w_up, a->w_down, (float*)((char*)a->workspace + outs), a->rows, a->x_stride,
              lampa_align_up((a->rows + n - 1) / n, 32), a->D, a->F};
  const dim3 grid((unsigned)((a->F + 127) / 128), (unsigned)n), block(FU_BLOCK);
#define FU_GO(DB)                                                                                                   \
  if (a->rows <= FU_TWO_ROWS) hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, DB, true>), grid, block, 0, s, k); \
  else hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, DB, false>), grid, block, 0, s, k);                       \
  break;
  switch ((a->D + 31) / 32) {
    case 1: FU_GO(1)
    case 2: FU_GO(2)
    case 3: FU_GO(3)
    default: FU_GO(4)
  }
#undef FU_GO
  LAMPA_PROF(s, "ff_fused_weights_kernel");
  hipLaunchKernelGGL((ff_fused_reduce_kernel<T>), dim3((a->D + 31) / 32, (a->F + 31) / 32, 3), dim3(256), 0, s, k.parts, n, a->D, a->F,
                     (T*)a->dw_gate, (T*)a->dw_up, (T*)a->dw_down);
  LAMPA_PROF(s, "ff_fused_reduce_kernel");
  return lampa_launch_status();
}

template <typename T>
static int fu_fwd(const lampa_ff_args* a, hipStream_t s) {
  switch (a->activation) {
    case FF_ACT_NONE: return fu_fwd_go<T, FF_ACT_NONE>(a, s);
    case FF_ACT_SILU: return fu_fwd_go<T, FF_ACT_SILU>(a, s);
    default: return fu_fwd_go<T, FF_ACT_SIGMOID>(a, s);
  }
}
template <typename T>
static int fu_bwd(const lampa_ff_args* a, hipStream_t s) {
  switch (a->activation) {
    case FF_ACT_NONE: return fu_bwd_go<T, FF_ACT_NONE>(a, s);
    case FF_ACT_SILU: return fu_bwd_go<T, FF_ACT_SILU>(a, s);
    default: return fu_bwd_go<T, FF_ACT_SIGMOID>(a, s);
  }
}
