// The gated feed-forward block for 16-bit types and narrow blocks (D <= 128): hidden values never leave the registers
// (ff_common.h has the mathematics).
//   out:      y (or, BACK, dx): a wave keeps 32 rows of x (and dy) as operands and their outputs as sums; the hidden columns pass in
//             chunks of 32, whose weights the workgroup's 4 waves share in LDS (double buffered, the next chunk under way in
//             registers). Products are formed transposed, hidden columns x rows: the sums of the first products, rounded, are
//             then the operands of the next as they lie in the registers.
//   weights:  a wave keeps 32 hidden columns (their weights as operands, the sums of the three gradients: 16 DB values a lane each)
//             and the rows pass in tiles of 32 in LDS; workgroups share the rows out and leave their sums in fp32.
//   reduce:   the parts of the weights' gradients in order, dWd turned on the way.
// Few rows: the chunks of hidden columns are shared out as well, and the outputs' parts summed in order.
#include "ff_common.h"

#define FU_BLOCK 256
#define FU_ROWS 128  // rows of a workgroup of `out`
#define FU_CHUNK 32  // hidden columns of a chunk

template <typename T>
__device__ __forceinline__ typename OpVec<T>::x8 fu_op(ff_u32x4 v) { return __builtin_bit_cast(typename OpVec<T>::x8, v); }

// A row's share of an operand: 16 bytes at column c of a row-major matrix of D columns; zero behind them.
__device__ __forceinline__ ff_u32x4 fu_load(__amdgpu_buffer_rsrc_t buf, unsigned row_bytes, int c, int D) {
  return ff_load16(buf, c < D ? row_bytes + (unsigned)c * 2 : FF_OFF);
}

struct FuOut {
  const void *x, *dy, *wg, *wu, *wd;
  void* out;     // [rows, D] of the type, or
  float* parts;  // [splits, rows, D]
  int64_t rows, x_stride;
  int D, F, chunks;  // chunks of a workgroup
};

// A 16-wide step's operand whose rows are the 32 columns col0 .. of a tile and whose contraction runs over the tile's rows.
template <typename T, int STRIDE>
__device__ __forceinline__ typename OpVec<T>::x8 fu_turned(const T* tile, int col0, int row0, int lane) {
  return op_ld_kappa_tr<T>(tile, STRIDE, col0, row0, lane);
}

template <typename T, int ACT, int DB, bool BACK>
__global__ void __launch_bounds__(FU_BLOCK, 2) ff_out_kernel(const FuOut a) {
  typedef typename OpVec<T>::x8 x8;
  typedef typename OpVec<T>::x4 x4;
  constexpr int KS = 2 * DB, WIDE = DB * 32, GS = WIDE + 8, DS = 40;       // elements between the rows of the tiles
  constexpr int PIECES = 128 * DB, LOADS = (PIECES + FU_BLOCK - 1) / FU_BLOCK;  // 16-byte pieces of each matrix's chunk
  constexpr int STAGE = 2 * FU_CHUNK * GS + WIDE * DS;
  __shared__ __attribute__((aligned(16))) T lds[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6;
  const int D = a.D, F = a.F;
  const int64_t r0 = (int64_t)blockIdx.x * FU_ROWS;
  const int64_t left = a.rows - r0;
  const int here = left < FU_ROWS ? (int)left : FU_ROWS;
  const int c0 = blockIdx.y * a.chunks, all = (F + FU_CHUNK - 1) / FU_CHUNK, c1 = c0 + a.chunks < all ? c0 + a.chunks : all;

  ff_u32x4 rg[LOADS], ru[LOADS], rd[LOADS];
  auto fetch = [&](int chunk) {
    const int f0 = chunk * FU_CHUNK, n = F - f0 < FU_CHUNK ? F - f0 : FU_CHUNK;
    const __amdgpu_buffer_rsrc_t gb = ff_buffer((const T*)a.wg + (int64_t)f0 * D, (int64_t)n * D * 2);
    const __amdgpu_buffer_rsrc_t ub = ff_buffer((const T*)a.wu + (int64_t)f0 * D, (int64_t)n * D * 2);
    const __amdgpu_buffer_rsrc_t db = ff_buffer((const T*)a.wd + f0, ((int64_t)(D - 1) * F + n) * 2);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int id = tid + i * FU_BLOCK;
      if (PIECES % FU_BLOCK && id >= PIECES) break;
      const int row = id / (DB * 4), c = id % (DB * 4) * 8;
      rg[i] = fu_load(gb, (unsigned)(row * D) * 2, c, D);
      ru[i] = fu_load(ub, (unsigned)(row * D) * 2, c, D);
      const int d = id / 4, f = id % 4 * 8;
      rd[i] = ff_load16(db, f < n && d < D ? (unsigned)(d * F + f) * 2 : FF_OFF);
    }
  };
  auto stage = [&](int which) {
    T *g = lds + which * STAGE, *u = g + FU_CHUNK * GS, *w = u + FU_CHUNK * GS;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int id = tid + i * FU_BLOCK;
      if (PIECES % FU_BLOCK && id >= PIECES) break;
      const int row = id / (DB * 4), c = id % (DB * 4) * 8;
      *reinterpret_cast<ff_u32x4*>(g + row * GS + c) = rg[i];
      *reinterpret_cast<ff_u32x4*>(u + row * GS + c) = ru[i];
      const int d = id / 4, f = id % 4 * 8;
      if constexpr (BACK) {
        *reinterpret_cast<ff_u32x4*>(w + d * DS + f) = rd[i];
      } else {  // groups of four in slot order within each 16 columns: the share of a step is then one 16-byte piece
        const x8 v = fu_op<T>(rd[i]);
        T* p = w + d * DS + (f & 16) + (f & 8 ? 4 : 0);
        *reinterpret_cast<x4*>(p) = x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<x4*>(p + 8) = x4{v[4], v[5], v[6], v[7]};
      }
    }
  };

  fetch(c0);
  // this wave's 32 rows
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
  __syncthreads();
  for (int chunk = c0; chunk < c1; ++chunk) {
    if (chunk + 1 < c1) fetch(chunk + 1);
    const int which = (chunk - c0) & 1;
    const T *g = lds + which * STAGE, *u = g + FU_CHUNK * GS, *w = u + FU_CHUNK * GS;
    f32x16 G, U, S;
#pragma unroll
    for (int r = 0; r < 16; ++r) G[r] = U[r] = S[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      G = mfma32(*reinterpret_cast<const x8*>(g + ln * GS + 16 * k + 8 * hh), xo[k], G);
      U = mfma32(*reinterpret_cast<const x8*>(u + ln * GS + 16 * k + 8 * hh), xo[k], U);
      if constexpr (BACK) S = mfma32(fu_turned<T, DS>(w, 0, 16 * k, lane), dyo[k], S);
    }
    if constexpr (!BACK) {
#pragma unroll
      for (int r = 0; r < 16; ++r) G[r] = ff_act<ACT>(G[r]) * U[r];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const x8 h = acc_to_op<T>(G, 8 * s);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          out[d] = mfma32(*reinterpret_cast<const x8*>(w + (32 * d + ln) * DS + 16 * s + 8 * hh), h, out[d]);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float value, slope;
        ff_act_slope<ACT>(G[r], value, slope);
        G[r] = S[r] * U[r] * slope;
        U[r] = S[r] * value;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const x8 dg = acc_to_op<T>(G, 8 * s), du = acc_to_op<T>(U, 8 * s);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          out[d] = mfma32(fu_turned<T, GS>(g, 32 * d, 16 * s, lane), dg, out[d]);
          out[d] = mfma32(fu_turned<T, GS>(u, 32 * d, 16 * s, lane), du, out[d]);
        }
      }
    }
    if (chunk + 1 < c1) stage(which ^ 1);
    __syncthreads();
  }
  const int row = 32 * wave + ln;
  if (row >= here) return;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * d + 8 * q + 4 * hh;
      if (c >= D) continue;
      if (a.parts)
        *reinterpret_cast<f32x4*>(a.parts + ((int64_t)blockIdx.y * a.rows + r0 + row) * D + c) =
            f32x4{out[d][4 * q], out[d][4 * q + 1], out[d][4 * q + 2], out[d][4 * q + 3]};
      else
        ff_store4((T*)a.out + (r0 + row) * D + c, out[d][4 * q], out[d][4 * q + 1], out[d][4 * q + 2], out[d][4 * q + 3]);
    }
}

// ------------------------------------------------------------------------------------------------ weights' gradients
struct FuWeights {
  const void *x, *dy, *wg, *wu, *wd;
  float* parts;  // [splits, 3, F, D]: dWg, dWu, dWd^T
  int64_t rows, x_stride, per;  // rows of a workgroup, a multiple of 32
  int D, F;
};

template <typename T, int ACT, int DB>
__global__ void __launch_bounds__(FU_BLOCK, 1) ff_fused_weights_kernel(const FuWeights a) {
  typedef typename OpVec<T>::x8 x8;
  constexpr int KS = 2 * DB, WIDE = DB * 32, XS = WIDE + 8, TILE = 32 * XS;
  constexpr int PIECES = 128 * DB, LOADS = (PIECES + FU_BLOCK - 1) / FU_BLOCK;
  __shared__ __attribute__((aligned(16))) T lds[2][2 * TILE];
  const int tid = threadIdx.x, lane = tid & 63, ln = lane & 31, hh = lane >> 5, wave = tid >> 6;
  const int D = a.D, F = a.F, f0 = blockIdx.x * 128 + 32 * wave, f = f0 + ln;
  const int64_t begin = (int64_t)blockIdx.y * a.per, end = begin + a.per < a.rows ? begin + a.per : a.rows;

  ff_u32x4 rx[LOADS], ry[LOADS];
  auto fetch = [&](int64_t t0) {
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
      *reinterpret_cast<ff_u32x4*>(&lds[which][row * XS + c]) = rx[i];
      *reinterpret_cast<ff_u32x4*>(&lds[which][TILE + row * XS + c]) = ry[i];
    }
  };
  if (begin < end) fetch(begin);
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
  if (begin < end) {
    stage(0);
    __syncthreads();
    int which = 0;
    for (int64_t t0 = begin; t0 < end; t0 += 32, which ^= 1) {
      const bool more = t0 + 32 < end;
      if (more) fetch(t0 + 32);
      const T *x = lds[which], *y = x + TILE;
      f32x16 G, U, S;
#pragma unroll
      for (int r = 0; r < 16; ++r) G[r] = U[r] = S[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const x8 xa = *reinterpret_cast<const x8*>(x + ln * XS + 16 * k + 8 * hh), ya = *reinterpret_cast<const x8*>(y + ln * XS + 16 * k + 8 * hh);
        G = mfma32(xa, wg[k], G);
        U = mfma32(xa, wu[k], U);
        S = mfma32(ya, wd[k], S);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float value, slope;
        ff_act_slope<ACT>(G[r], value, slope);
        const float s = S[r], up = U[r];
        S[r] = value * up;
        U[r] = s * value;
        G[r] = s * up * slope;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const x8 dg = acc_to_op<T>(G, 8 * s), du = acc_to_op<T>(U, 8 * s), h = acc_to_op<T>(S, 8 * s);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const x8 xt = fu_turned<T, XS>(x, 32 * d, 16 * s, lane), yt = fu_turned<T, XS>(y, 32 * d, 16 * s, lane);
          dwg[d] = mfma32(xt, dg, dwg[d]);
          dwu[d] = mfma32(xt, du, dwu[d]);
          dwd[d] = mfma32(yt, h, dwd[d]);
        }
      }
      if (more) stage(which ^ 1);
      __syncthreads();
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
bool ff_fused_takes(const lampa_ff_args* a) { return a->dtype != GDR_FP32 && a->D <= 128; }

// How the chunks of hidden columns are shared out: over one workgroup where the rows alone fill half the GPU (every further share
// writes and reads the outputs' fp32 parts), else over as many as make one workgroup a CU.
struct FuShare {
  int splits, chunks;
};
static FuShare fu_share(const lampa_ff_args* a) {
  const int64_t tiles = (a->rows + FU_ROWS - 1) / FU_ROWS;
  const int all = (a->F + FU_CHUNK - 1) / FU_CHUNK;
  const int64_t want = tiles < 1 ? 1 : 256 / tiles;
  const int n = want < 1 ? 1 : (want < all ? (int)want : all);
  const int chunks = (all + n - 1) / n;
  return {(all + chunks - 1) / chunks, chunks};
}
// The rows of the weights' gradients: one workgroup of 128 hidden columns a CU.
static int fu_weight_splits(const lampa_ff_args* a) {
  const int64_t cols = (a->F + 127) / 128, want = (256 + cols - 1) / cols, most = (a->rows + 31) / 32;
  return (int)(want < 1 ? 1 : (want < most ? want : (most < 1 ? 1 : most)));
}

int64_t ff_fused_workspace(const lampa_ff_args* a, int backward) {
  const FuShare sh = fu_share(a);
  const int64_t outs = sh.splits > 1 ? lampa_align_up((int64_t)sh.splits * a->rows * a->D * 4, 256) : 0;
  return outs + (backward ? (int64_t)fu_weight_splits(a) * 3 * a->D * a->F * 4 : 0);
}

template <typename T, int ACT, bool BACK>
static int fu_out(const lampa_ff_args* a, hipStream_t s) {
  const FuShare sh = fu_share(a);
  T* out = (T*)(BACK ? a->dx : a->y);
  FuOut k{a->x, a->dy, a->w_gate, a->w_up, a->w_down, out, sh.splits > 1 ? (float*)a->workspace : nullptr, a->rows, a->x_stride, a->D, a->F, sh.chunks};
  const dim3 grid((unsigned)((a->rows + FU_ROWS - 1) / FU_ROWS), (unsigned)sh.splits), block(FU_BLOCK);
  switch ((a->D + 31) / 32) {
    case 1: hipLaunchKernelGGL((ff_out_kernel<T, ACT, 1, BACK>), grid, block, 0, s, k); break;
    case 2: hipLaunchKernelGGL((ff_out_kernel<T, ACT, 2, BACK>), grid, block, 0, s, k); break;
    case 3: hipLaunchKernelGGL((ff_out_kernel<T, ACT, 3, BACK>), grid, block, 0, s, k); break;
    default: hipLaunchKernelGGL((ff_out_kernel<T, ACT, 4, BACK>), grid, block, 0, s, k); break;
  }
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
  switch ((a->D + 31) / 32) {
    case 1: hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, 1>), grid, block, 0, s, k); break;
    case 2: hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, 2>), grid, block, 0, s, k); break;
    case 3: hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, 3>), grid, block, 0, s, k); break;
    default: hipLaunchKernelGGL((ff_fused_weights_kernel<T, ACT, 4>), grid, block, 0, s, k); break;
  }
  LAMPA_PROF(s, "ff_fused_weights_kernel");
  hipLaunchKernelGGL((ff_fused_reduce_kernel<T>), dim3((a->D + 31) / 32, (a->F + 31) / 32, 3), dim3(256), 0, s, k.parts, n, a->D, a->F,
                     (T*)a->dw_gate, (T*)a->dw_up, (T*)a->dw_down);
  LAMPA_PROF(s, "ff_fused_reduce_kernel");
  return lampa_launch_status();
}

#define FU_TYPES(GO)                                   \
  switch (a->dtype * 3 + a->activation) {              \
    case 0: return GO<__bf16, 0>(a, s);                \
    case 1: return GO<__bf16, 1>(a, s);                \
    case 2: return GO<__bf16, 2>(a, s);                \
    case 3: return GO<_Float16, 0>(a, s);              \
    case 4: return GO<_Float16, 1>(a, s);              \
    default: return GO<_Float16, 2>(a, s);             \
  }
int ff_fused_fwd(const lampa_ff_args* a, hipStream_t s) { FU_TYPES(fu_fwd_go) }
int ff_fused_bwd(const lampa_ff_args* a, hipStream_t s) { FU_TYPES(fu_bwd_go) }
