// The border between two blocks of a pre-norm stack, in one pass over the rows (gfx950): the norm behind a block, its gate, the
// scaled residual add and the norm in front of the next block,
//   a = x  or  x / rms(x) * post_weight,   m = scale * act(gate) * a,   r = residual + m,   y = r / rms(r) * weight,
// with rms(v) = sqrt(mean(v^2) + eps) over the last dimension, and its gradients. Every factor and the residual are optional.
// Bound by bytes: each input is read once, each output written once; sums and everything between load and store are fp32 (y
// comes from the unrounded r). The gradients recompute a, r and both rms from the inputs, which costs the bytes of x and the
// residual instead of those of kept intermediates, and is exact where a kept r would be rounded to the residual's type.
//
// LPR lanes (or, at 256, a whole workgroup) share a row, each holding 8 consecutive channels in each of STEPS strides.
//
// Measured, 60 000 x 512 in bf16 beside an fp32 residual, post-norm, a gate for each token, a scale: forward 81 us (430 MB, 5.3
// TB/s), gradients 167 us (676 MB, 4.1 TB/s; 147 at best) with the next row's operands under way (190 us without) and 9 us for the
// sums over the workgroups' rows.
#include "gdr_common.h"
#include "row_sums.h"

#define RN_BLOCK 256
enum { RN_GATE_NONE = 0, RN_GATE_TOKEN = 1, RN_GATE_SEQ = 2 };
enum { RN_ACT_NONE = 0, RN_ACT_SILU = 1, RN_ACT_SIGMOID = 2 };

struct RnArgs {
  const void *x, *residual, *gate;
  const float *weight, *post_weight, *scale;
  void *y, *res_out;
  int64_t rows, seq_rows;  // rows in all; rows that share one row of a sequence's gate
  int D, gate_kind, act;
  float eps;
  // gradients
  const void *dy, *dres;
  void *dx, *dresidual, *dgate;
  float* parts;            // [workgroups, sums, D]
  int n_sums;              // weight, post_weight, scale, sequence gate, as far as they are wanted
  int at_weight, at_post, at_scale, at_gate;  // places of the sums, -1: not wanted
};

template <typename T>
__device__ __forceinline__ void rn_store8(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    vec8 o;
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = GdrElem<T>::from_float(v[c]);
    *reinterpret_cast<vec8*>(p) = o;
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// 8 consecutive elements as loaded.
template <typename T>
struct RnRaw {
  typedef T vec __attribute__((ext_vector_type(sizeof(T) == 2 ? 8 : 4)));
  vec v[sizeof(T) == 2 ? 1 : 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int k = 0; k < (sizeof(T) == 2 ? 1 : 2); ++k) v[k] = reinterpret_cast<const vec*>(p)[k];
  }
  __device__ __forceinline__ void get(float* out) const {
#pragma unroll
    for (int c = 0; c < 8; ++c) out[c] = GdrElem<T>::to_float(sizeof(T) == 2 ? v[0][c] : v[c / 4 < (sizeof(T) == 2 ? 1 : 2) ? c / 4 : 0][c % 4]);
  }
};

// Sum over the lanes of a row (every lane gets it). `part`: LDS of 2 x 4 floats for rows of a whole workgroup; `turn`
// alternates, so that one barrier a sum is enough.
template <int LPR>
__device__ __forceinline__ float rn_row_sum(float v, float (*part)[4], int& turn) {
#pragma unroll
  for (int off = 1; off < (LPR < 64 ? LPR : 64); off <<= 1) v += __shfl_xor(v, off);
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = (part[turn][0] + part[turn][1]) + (part[turn][2] + part[turn][3]);
    turn ^= 1;
  }
  return v;
}

__device__ __forceinline__ float rn_act(float g, int act, float& slope) {
  if (act == RN_ACT_NONE) { slope = 1.0f; return g; }
  const float s = 1.0f / (1.0f + expf(-g));
  if (act == RN_ACT_SIGMOID) { slope = s * (1.0f - s); return s; }
  slope = s * __builtin_fmaf(g, 1.0f - s, 1.0f);
  return g * s;
}

template <typename T, typename RT, int LPR, int STEPS, bool GRAD>
__global__ void __launch_bounds__(RN_BLOCK) rn_kernel(RnArgs a) {
  constexpr int ROWS = RN_BLOCK / LPR;  // rows a workgroup has under way
  __shared__ float part[2][4];
  int turn = 0;
  const int sub = threadIdx.x % LPR, slot = threadIdx.x / LPR;
  const float inv_d = 1.0f / (float)a.D;
  // a workgroup stays within one sequence where a gate's gradient is summed over it: blockIdx.y counts sequences then
  const int64_t row_base = GRAD ? (int64_t)blockIdx.y * a.seq_rows : 0;
  const int64_t n_rows = GRAD ? a.seq_rows : a.rows;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  float dw[GRAD ? STEPS : 1][8], dpw[GRAD ? STEPS : 1][8], dsc[GRAD ? STEPS : 1][8], dga[GRAD ? STEPS : 1][8];
  if constexpr (GRAD) {
#pragma unroll
    for (int st = 0; st < STEPS; ++st)
#pragma unroll
      for (int c = 0; c < 8; ++c) dw[st][c] = dpw[st][c] = dsc[st][c] = dga[st][c] = 0.0f;
  }
  // The next row's operands are requested while this one is worked on, where they fit the registers (one stride a row).
  constexpr bool AHEAD = GRAD && STEPS == 1;
  RnRaw<T> nx, ng, ndy;
  RnRaw<RT> nh, ndr;
  auto request = [&](int64_t r0) {
    const int c0 = sub * 8;
    if (!(r0 + slot < n_rows && c0 < a.D)) return;
    const int64_t row = row_base + r0 + slot, at = row * a.D + c0;
    nx.load((const T*)a.x + at);
    if (a.residual) nh.load((const RT*)a.residual + at);
    if (a.gate_kind) ng.load((const T*)a.gate + (a.gate_kind == RN_GATE_SEQ ? row / a.seq_rows : row) * a.D + c0);
    if (a.dy) ndy.load((const T*)a.dy + at);
    if (a.dres) ndr.load((const RT*)a.dres + at);
  };
  if (AHEAD) request((int64_t)blockIdx.x * ROWS);
  // every thread makes the same number of turns: rows past the end are worked on as zeros, with a norm of zero (eps may be 0),
  // and not stored
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < n_rows; r0 += stride) {
    const bool live = r0 + slot < n_rows;
    const int64_t row = row_base + r0 + slot;
    const RnRaw<T> cx = nx, cg = ng, cdy = ndy;
    const RnRaw<RT> ch = nh, cdr = ndr;
    if (AHEAD) request(r0 + stride);
    float x[STEPS][8], h[STEPS][8], sq = 0.0f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int c0 = (st * LPR + sub) * 8;
      const bool on = live && c0 < a.D;
#pragma unroll
      for (int c = 0; c < 8; ++c) x[st][c] = h[st][c] = 0.0f;
      if (on) {
        if constexpr (AHEAD) {
          cx.get(x[st]);
          if (a.residual) ch.get(h[st]);
        } else {
          load8((const T*)a.x + row * a.D + c0, x[st]);
          if (a.residual) load8((const RT*)a.residual + row * a.D + c0, h[st]);
        }
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) sq = __builtin_fmaf(x[st][c], x[st][c], sq);
    }
    float i1 = 1.0f;
    if (a.post_weight) {
      const float mean = rn_row_sum<LPR>(sq, part, turn) * inv_d;
      i1 = live ? 1.0f / sqrtf(mean + a.eps) : 0.0f;
    }
    const int64_t gate_row = a.gate_kind == RN_GATE_SEQ ? row / a.seq_rows : row;
    float am[GRAD ? STEPS : 1][8], act[GRAD ? STEPS : 1][8], slope[GRAD ? STEPS : 1][8];  // a; act(gate); its derivative
    float sq2 = 0.0f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int c0 = (st * LPR + sub) * 8;
      const bool on = live && c0 < a.D;
      float pw[8], g[8], sc[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) { pw[c] = 1.0f; g[c] = 1.0f; sc[c] = 1.0f; }
      if (on && a.post_weight) load8(a.post_weight + c0, pw);
      if (on && a.gate_kind) {
        if constexpr (AHEAD) cg.get(g);
        else load8((const T*)a.gate + gate_row * a.D + c0, g);
      }
      if (on && a.scale) load8(a.scale + c0, sc);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float v = a.post_weight ? x[st][c] * i1 * pw[c] : x[st][c];
        float sl = 0.0f, ac = 1.0f;
        if (a.gate_kind) ac = rn_act(g[c], a.act, sl);
        if constexpr (GRAD) { am[st][c] = v; act[st][c] = ac; slope[st][c] = sl; }
        h[st][c] = __builtin_fmaf(sc[c], ac * v, h[st][c]);
        if (!on) h[st][c] = 0.0f;
        sq2 = __builtin_fmaf(h[st][c], h[st][c], sq2);
      }
      if constexpr (!GRAD)
        if (on && a.res_out) rn_store8((RT*)a.res_out + row * a.D + c0, h[st]);
    }
    const float mean2 = rn_row_sum<LPR>(sq2, part, turn) * inv_d;
    const float i2 = live ? 1.0f / sqrtf(mean2 + a.eps) : 0.0f;
    if constexpr (!GRAD) {
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int c0 = (st * LPR + sub) * 8;
        if (!(live && c0 < a.D)) continue;
        float w[8], o[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] = 1.0f;
        if (a.weight) load8(a.weight + c0, w);
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] = h[st][c] * i2 * w[c];
        rn_store8((T*)a.y + row * a.D + c0, o);
      }
    } else {
      // dr = dres + i2 (dy w) - r i2^3 mean(dy w r);  da = dr scale act;  dx likewise through the first norm
      float dh[STEPS][8], dot = 0.0f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int c0 = (st * LPR + sub) * 8;
        const bool on = live && c0 < a.D;
        float w[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) { dh[st][c] = 0.0f; w[c] = 1.0f; }
        if (on && a.dy) {
          if constexpr (AHEAD) cdy.get(dh[st]);
          else load8((const T*)a.dy + row * a.D + c0, dh[st]);
        }
        if (on && a.weight) load8(a.weight + c0, w);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          dw[st][c] = __builtin_fmaf(dh[st][c], h[st][c] * i2, dw[st][c]);
          dh[st][c] *= w[c];
          dot = __builtin_fmaf(dh[st][c], h[st][c], dot);
        }
      }
      dot = rn_row_sum<LPR>(dot, part, turn);
      const float k2 = dot * inv_d * i2 * i2 * i2;
      float dot1 = 0.0f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int c0 = (st * LPR + sub) * 8;
        const bool on = live && c0 < a.D;
        float dr[8], sc[8], pw[8], dg[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) { dr[c] = 0.0f; sc[c] = 1.0f; pw[c] = 1.0f; }
        if (on && a.dres) {
          if constexpr (AHEAD) cdr.get(dr);
          else load8((const RT*)a.dres + row * a.D + c0, dr);
        }
        if (on && a.scale) load8(a.scale + c0, sc);
        if (on && a.post_weight) load8(a.post_weight + c0, pw);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          dr[c] += i2 * dh[st][c] - h[st][c] * k2;
          const float ds = dr[c] * act[st][c];
          dsc[st][c] = __builtin_fmaf(ds, am[st][c], dsc[st][c]);
          dg[c] = dr[c] * sc[c] * am[st][c] * slope[st][c];
          if (a.gate_kind == RN_GATE_SEQ) dga[st][c] += dg[c];
          float da = ds * sc[c];
          if (a.post_weight) {
            dpw[st][c] = __builtin_fmaf(da, x[st][c] * i1, dpw[st][c]);
            da *= pw[c];
            dot1 = __builtin_fmaf(da, x[st][c], dot1);
          }
          dh[st][c] = da;
        }
        if (on) {
          if (a.dresidual) rn_store8((RT*)a.dresidual + row * a.D + c0, dr);
          if (a.gate_kind == RN_GATE_TOKEN && a.dgate) rn_store8((T*)a.dgate + row * a.D + c0, dg);
        }
      }
      float k1 = 0.0f;
      if (a.post_weight) k1 = rn_row_sum<LPR>(dot1, part, turn) * inv_d * i1 * i1 * i1;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const int c0 = (st * LPR + sub) * 8;
        if (!(live && c0 < a.D)) continue;
        float o[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] = a.post_weight ? i1 * dh[st][c] - x[st][c] * k1 : dh[st][c];
        rn_store8((T*)a.dx + row * a.D + c0, o);
      }
    }
  }
  if constexpr (GRAD) {
    // over the rows of the workgroup: across the lanes of a wave that hold the same channels, then across the waves
    __shared__ float red[LPR < 64 ? RN_BLOCK / 64 : 1][LPR < 64 ? LPR * 8 : 1];
    float* out = a.parts + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.n_sums * a.D;
    auto leave = [&](float (*v)[8], int at) {
      if (at < 0) return;
      if constexpr (LPR >= 256) {
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          const int c0 = (st * LPR + sub) * 8;
          if (c0 < a.D) rn_store8(out + (int64_t)at * a.D + c0, v[st]);
        }
      } else {
        __shared__ float wide[LPR == 64 ? 4 : 1][LPR == 64 ? 64 * 8 : 1];
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          __syncthreads();
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float s = v[st][c];
#pragma unroll
            for (int off = LPR; off < 64; off <<= 1) s += __shfl_xor(s, off);
            if constexpr (LPR < 64) {
              if ((threadIdx.x & 63) < LPR) red[threadIdx.x >> 6][sub * 8 + c] = s;
            } else {
              wide[threadIdx.x >> 6][sub * 8 + c] = s;
            }
          }
          __syncthreads();
          for (int i = threadIdx.x; i < LPR * 8; i += RN_BLOCK) {
            const int ch = st * LPR * 8 + i;
            float s;
            if constexpr (LPR < 64) s = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
            else s = (wide[0][i] + wide[1][i]) + (wide[2][i] + wide[3][i]);
            if (ch < a.D) out[(int64_t)at * a.D + ch] = s;
          }
        }
      }
    };
    leave(dw, a.at_weight);
    leave(dpw, a.at_post);
    leave(dsc, a.at_scale);
    leave(dga, a.at_gate);
  }
}

// Lanes and strides of a row. 513 to 1024 channels: two strides of a wave without gradients, half a workgroup with them (they would
// take 280 registers); 30 000 rows of 768 / 1024 in bf16 beside an fp32 residual, a wave against a workgroup: forward 59 / 70
// against 74 / 75 us, gradients 214 / 224 against 178 / 183 us.
static int rn_shape(int D, bool grad, int* lpr, int* steps) {
  if (D <= 512) {
    *lpr = 8;
    while (*lpr * 8 < D) *lpr <<= 1;
    *steps = 1;
  } else if (D <= 1024 && !grad) {
    *lpr = 64;
    *steps = 2;
  } else if (D <= 8192) {
    *lpr = 256;
    *steps = D <= 2048 ? 1 : (D <= 4096 ? 2 : 4);
  } else {
    return LAMPA_ERR_UNSUPPORTED;
  }
  return LAMPA_OK;
}

// Workgroups of the gradients for each sequence: each leaves one row of sums, so no more than a few a CU.
static int64_t rn_grad_blocks(int64_t seq_rows, int64_t n_seq, int lpr) {
  const int64_t per = RN_BLOCK / lpr, need = (seq_rows + per - 1) / per;
  int64_t most = (1024 + n_seq - 1) / n_seq;
  return need < most ? (need < 1 ? 1 : need) : most;
}

template <typename T, typename RT, bool GRAD>
static int rn_launch(const RnArgs& a, int lpr, int steps, dim3 grid, hipStream_t s) {
  LAMPA_PROF(s, "start");
#define RN_GO(L, S) hipLaunchKernelGGL((rn_kernel<T, RT, L, S, GRAD>), grid, dim3(RN_BLOCK), 0, s, a)
  switch (lpr) {
    case 8: RN_GO(8, 1); break;
    case 16: RN_GO(16, 1); break;
    case 32: RN_GO(32, 1); break;
    case 64:
      if constexpr (GRAD) RN_GO(64, 1);
      else if (steps == 1) RN_GO(64, 1);
      else RN_GO(64, 2);
      break;
    default: if (steps == 1) RN_GO(256, 1); else if (steps == 2) RN_GO(256, 2); else RN_GO(256, 4); break;
  }
#undef RN_GO
  LAMPA_PROF(s, GRAD ? "rn_kernel<grad>" : "rn_kernel");
  return lampa_launch_status();
}

template <bool GRAD>
static int rn_types(const RnArgs& a, int dtype, int res_dtype, int lpr, int steps, dim3 grid, hipStream_t s) {
  if (dtype == GDR_FP32) return rn_launch<float, float, GRAD>(a, lpr, steps, grid, s);
  if (dtype == GDR_BF16)
    return res_dtype == GDR_FP32 ? rn_launch<__bf16, float, GRAD>(a, lpr, steps, grid, s)
                                 : rn_launch<__bf16, __bf16, GRAD>(a, lpr, steps, grid, s);
  return res_dtype == GDR_FP32 ? rn_launch<_Float16, float, GRAD>(a, lpr, steps, grid, s)
                               : rn_launch<_Float16, _Float16, GRAD>(a, lpr, steps, grid, s);
}

static int rn_check(const void* x, const void* residual, const void* gate, int gate_kind, int act, int64_t rows, int64_t seq_rows,
                    int D, int dtype, int res_dtype) {
  if (rows < 0 || D < 1 || dtype < 0 || dtype > 2 || (res_dtype != dtype && res_dtype != GDR_FP32) || act < 0 || act > 2 ||
      gate_kind < 0 || gate_kind > 2 || (rows && (!x || (gate_kind && !gate))) || seq_rows < 1 || rows % seq_rows)
    return LAMPA_ERR_INVALID;
  if (D % 8 || D > 8192 || ((uintptr_t)x | (uintptr_t)residual | (uintptr_t)gate) % 16) return LAMPA_ERR_UNSUPPORTED;
  return LAMPA_OK;
}

extern "C" int lampa_residual_norm_fwd(const void* x, const void* residual, const float* weight, const float* post_weight,
                                       const void* gate, int gate_kind, int activation, const float* scale, int64_t rows,
                                       int64_t seq_rows, int D, float eps, int dtype, int res_dtype, void* y, void* residual_out,
                                       void* stream) {
  int lpr, steps, rc = rn_check(x, residual, gate, gate_kind, activation, rows, seq_rows, D, dtype, res_dtype);
  if (rc == LAMPA_OK) rc = rn_shape(D, false, &lpr, &steps);
  if (rc != LAMPA_OK) return rc;
  if (rows == 0) return LAMPA_OK;
  if (!y || (residual && !residual_out)) return LAMPA_ERR_INVALID;
  if (((uintptr_t)y | (uintptr_t)residual_out) % 16) return LAMPA_ERR_UNSUPPORTED;
  RnArgs a = {};
  a.x = x; a.residual = residual; a.gate = gate; a.weight = weight; a.post_weight = post_weight; a.scale = scale;
  a.y = y; a.res_out = residual_out; a.rows = rows; a.seq_rows = seq_rows; a.D = D; a.gate_kind = gate_kind;
  a.act = activation; a.eps = eps;
  const int64_t blocks = (rows + RN_BLOCK / lpr - 1) / (RN_BLOCK / lpr);
  if (blocks > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  return rn_types<false>(a, dtype, res_dtype, lpr, steps, dim3((unsigned)blocks), (hipStream_t)stream);
}

extern "C" int64_t lampa_residual_norm_bwd_workspace_bytes(int64_t rows, int64_t seq_rows, int D) {
  int lpr, steps;
  if (rows < 0 || seq_rows < 1 || rows % seq_rows || D < 1 || D % 8) return LAMPA_ERR_INVALID;
  if (rn_shape(D, true, &lpr, &steps) != LAMPA_OK) return LAMPA_ERR_UNSUPPORTED;
  const int64_t n_seq = rows / seq_rows;
  return n_seq * rn_grad_blocks(seq_rows, n_seq ? n_seq : 1, lpr) * 4 * D * 4;
}

extern "C" int lampa_residual_norm_bwd(const void* x, const void* residual, const float* weight, const float* post_weight,
                                       const void* gate, int gate_kind, int activation, const float* scale, const void* dy,
                                       const void* dres, int64_t rows, int64_t seq_rows, int D, float eps, int dtype, int res_dtype,
                                       void* dx, void* dresidual, void* dgate, float* dweight, float* dpost_weight, float* dscale,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  int lpr, steps, rc = rn_check(x, residual, gate, gate_kind, activation, rows, seq_rows, D, dtype, res_dtype);
  if (rc == LAMPA_OK) rc = rn_shape(D, true, &lpr, &steps);
  if (rc != LAMPA_OK) return rc;
  const int64_t n_seq = rows / seq_rows;
  if (rows == 0) return LAMPA_OK;  // nothing to sum: the caller's zeros stand
  if (!dx || (residual && !dresidual) || (!weight && dweight) || (!post_weight && dpost_weight) || (!scale && dscale) || (!gate_kind && dgate))
    return LAMPA_ERR_INVALID;
  if (((uintptr_t)dx | (uintptr_t)dresidual | (uintptr_t)dgate | (uintptr_t)dy | (uintptr_t)dres) % 16) return LAMPA_ERR_UNSUPPORTED;
  if (n_seq > 65535) return LAMPA_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < lampa_residual_norm_bwd_workspace_bytes(rows, seq_rows, D)) return LAMPA_ERR_WORKSPACE;
  RnArgs a = {};
  a.x = x; a.residual = residual; a.gate = gate; a.weight = weight; a.post_weight = post_weight; a.scale = scale;
  a.rows = rows; a.seq_rows = seq_rows; a.D = D; a.gate_kind = gate_kind; a.act = activation; a.eps = eps;
  a.dy = dy; a.dres = dres; a.dx = dx; a.dresidual = dresidual; a.dgate = dgate; a.parts = (float*)workspace;
  a.at_weight = dweight ? a.n_sums++ : -1;
  a.at_post = dpost_weight ? a.n_sums++ : -1;
  a.at_scale = dscale ? a.n_sums++ : -1;
  a.at_gate = gate_kind == RN_GATE_SEQ && dgate ? a.n_sums++ : -1;
  const int64_t per_seq = rn_grad_blocks(seq_rows, n_seq, lpr);
  hipStream_t s = (hipStream_t)stream;
  rc = rn_types<true>(a, dtype, res_dtype, lpr, steps, dim3((unsigned)per_seq, (unsigned)n_seq), s);
  // [n_seq, per_seq, n_sums, D]: a weight's sums are columns of rows of n_sums * D, the weights' ones side by side
  const int64_t width = (int64_t)a.n_sums * D;
  RowSumsOut<float> to = {{nullptr, nullptr, nullptr}, 0};
  int sets = 0;
  for (float* out : {dweight, dpost_weight, dscale})
    if (out) to.out[sets++] = out;
  if (rc == LAMPA_OK && sets) rc = row_sums_launch<float>(a.parts, n_seq * per_seq, D, width, D, sets, to, s);
  if (rc == LAMPA_OK && a.at_gate >= 0) {
    const float* src = a.parts + (int64_t)a.at_gate * D;
    const int64_t set = per_seq * width;
    if (dtype == GDR_BF16) rc = row_sums_launch<__bf16>(src, per_seq, D, width, set, (int)n_seq, RowSumsOut<__bf16>{{(__bf16*)dgate, nullptr, nullptr}, D}, s);
    else if (dtype == GDR_FP16) rc = row_sums_launch<_Float16>(src, per_seq, D, width, set, (int)n_seq, RowSumsOut<_Float16>{{(_Float16*)dgate, nullptr, nullptr}, D}, s);
    else rc = row_sums_launch<float>(src, per_seq, D, width, set, (int)n_seq, RowSumsOut<float>{{(float*)dgate, nullptr, nullptr}, D}, s);
  }
  return rc;
}
