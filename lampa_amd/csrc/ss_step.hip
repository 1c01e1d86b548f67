// One token of the state-space operator for each of n sequences, on a kept state (gfx950):
//   S <- exp(delta A) S + delta B x^T,   y = S^T C + D x      per sequence and head, S [N, P] fp32.
// Bound by the state's bytes, read once and written once. A workgroup takes PB columns (all N rows) of one head's state:
// PB / VW lanes side by side over the columns, the rest of the 256 threads over the rows, so that every load of the state
// can be under way at once; y is then summed over the rows' threads.
//
// Measured, bf16, 8 heads of 64: 250 sequences at N = 128 26 us (139 MB, 5.3 TB/s), one sequence at N = 64 6.5 us.
#include "ss_common.h"

#define SP_BLOCK 256
#define SP_ROWS 8  // rows of a thread under way at once

template <typename T, int PB, int VW>
__global__ void __launch_bounds__(SP_BLOCK) ss_step_kernel(const T* __restrict__ x, int64_t x_stride, const void* __restrict__ dt,
                                                           int dt_dtype, int64_t dt_stride, const T* __restrict__ Bm, int64_t B_stride,
                                                           const T* __restrict__ Cm, int64_t C_stride,
                                                           const float* __restrict__ A, const float* __restrict__ D,
                                                           const float* __restrict__ dt_bias, const float* state,
                                                           float* new_state, T* __restrict__ y, int H, int P, int G, int N,
                                                           int softplus) {
  constexpr int LANES = PB / VW, GROUPS = SP_BLOCK / LANES;
  typedef float vec __attribute__((ext_vector_type(VW)));
  const int pblocks = (P + PB - 1) / PB;
  const int pb = blockIdx.x % pblocks, h = blockIdx.x / pblocks % H;
  const int64_t b = blockIdx.x / pblocks / H;
  const int pl = threadIdx.x % LANES, rg = threadIdx.x / LANES;
  const int p0 = pb * PB + pl * VW;
  const bool on = p0 < P;  // VW divides P where it is not 1
  const int grp = h / (H / G);
  const T* Br = Bm + b * B_stride + (int64_t)grp * N;
  const T* Cr = Cm + b * C_stride + (int64_t)grp * N;
  const int64_t base = (b * H + h) * (int64_t)N * P + p0;
  const float delta = ss_delta(ss_load_dt<T>(dt, dt_dtype, b * dt_stride + h), dt_bias ? dt_bias[h] : 0.0f, softplus);
  const float decay = expf(delta * A[h]);
  float xv[VW], acc[VW];
#pragma unroll
  for (int i = 0; i < VW; ++i) {
    xv[i] = on ? GdrElem<T>::to_float(x[b * x_stride + (int64_t)h * P + p0 + i]) : 0.0f;
    acc[i] = 0.0f;
  }
  for (int n0 = rg; n0 < N; n0 += GROUPS * SP_ROWS) {
    vec s[SP_ROWS];
    float bn[SP_ROWS], cn[SP_ROWS];
#pragma unroll
    for (int k = 0; k < SP_ROWS; ++k) {
      const int n = n0 + k * GROUPS;
      if (n < N && on) {
        if constexpr (VW == 1) s[k][0] = state[base + (int64_t)n * P];
        else s[k] = *reinterpret_cast<const vec*>(state + base + (int64_t)n * P);
      }
      if (n < N) {
        bn[k] = GdrElem<T>::to_float(Br[n]);
        cn[k] = GdrElem<T>::to_float(Cr[n]);
      }
    }
#pragma unroll
    for (int k = 0; k < SP_ROWS; ++k) {
      const int n = n0 + k * GROUPS;
      if (n >= N || !on) continue;
      const float u = delta * bn[k];
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        s[k][i] = __builtin_fmaf(u, xv[i], decay * s[k][i]);
        acc[i] = __builtin_fmaf(cn[k], s[k][i], acc[i]);
      }
      if constexpr (VW == 1) new_state[base + (int64_t)n * P] = s[k][0];
      else *reinterpret_cast<vec*>(new_state + base + (int64_t)n * P) = s[k];
    }
  }
  __shared__ float part[SP_BLOCK / 64][PB];
#pragma unroll
  for (int i = 0; i < VW; ++i) {
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1) acc[i] += __shfl_xor(acc[i], off);
    if ((threadIdx.x & 63) < LANES) part[threadIdx.x >> 6][pl * VW + i] = acc[i];
  }
  __syncthreads();
  const int p = pb * PB + threadIdx.x;
  if (threadIdx.x < PB && p < P) {
    float out = 0.0f;
#pragma unroll
    for (int w = 0; w < SP_BLOCK / 64; ++w) out += part[w][threadIdx.x];
    const int64_t at = (int64_t)h * P + p;
    if (D) out = __builtin_fmaf(D[h], GdrElem<T>::to_float(x[b * x_stride + at]), out);
    y[b * H * P + at] = GdrElem<T>::from_float(out);
  }
}

template <typename T>
static int ss_step_launch(const void* x, int64_t xs, const void* dt, int dt_dtype, int64_t dts, const void* B, int64_t bs, const void* C,
                          int64_t cs, const float* A, const float* D, const float* dt_bias, const float* state,
                          float* new_state, void* y, int n, int H, int P, int G, int N, int softplus, hipStream_t s) {
  const bool vec = P % 4 == 0 && ((uintptr_t)state | (uintptr_t)new_state) % 16 == 0;
  const int64_t wide = (int64_t)n * H * ((P + 63) / 64), narrow = (int64_t)n * H * ((P + 15) / 16);
  // Fewer workgroups than CUs: narrower ones. 16 against 64 columns a workgroup, us, sequences x N (8 heads of 64): 1 x 128 6.7 / 8.0,
  // 16 x 128 7.4 / 8.7, 32 x 64 8.2 / 7.6, 64 x 128 16.7 / 10.6, 250 x 128 42.8 / 26.0.
  const bool few = wide < 256;
  if ((few ? narrow : wide) > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  LAMPA_PROF(s, "start");
#define SP_GO(PB, VW)                                                                                                     \
  hipLaunchKernelGGL((ss_step_kernel<T, PB, VW>), dim3((unsigned)(PB == 64 ? wide : narrow)), dim3(SP_BLOCK), 0, s, (const T*)x, \
                     xs, dt, dt_dtype, dts, (const T*)B, bs, (const T*)C, cs, A, D, dt_bias, state, new_state, (T*)y, H, P, G,  \
                     N, softplus)
  if (few) { if (vec) SP_GO(16, 4); else SP_GO(16, 1); }
  else { if (vec) SP_GO(64, 4); else SP_GO(64, 1); }
#undef SP_GO
  LAMPA_PROF(s, "ss_step_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_ss_step(const void* x, int64_t x_stride, const void* dt, int64_t dt_stride, const void* B, int64_t B_stride,
                             const void* C, int64_t C_stride, const float* A, const float* D, const float* dt_bias,
                             const float* state, float* new_state, void* y, int n, int H, int P, int G, int N, int dtype,
                             int dt_dtype, int softplus, void* stream) {
  if (!x || !dt || !B || !C || !A || !state || !new_state || !y || n < 0 || H < 1 || P < 1 || G < 1 || N < 1 || H % G ||
      (dt_dtype != dtype && dt_dtype != GDR_FP32))
    return LAMPA_ERR_INVALID;
  if (x_stride < (int64_t)H * P || dt_stride < H || B_stride < (int64_t)G * N || C_stride < (int64_t)G * N) return LAMPA_ERR_INVALID;
  if (n == 0) return LAMPA_OK;
  hipStream_t s = (hipStream_t)stream;
#define SP_ARGS x, x_stride, dt, dt_dtype, dt_stride, B, B_stride, C, C_stride, A, D, dt_bias, state, new_state, y, n, H, P, G, N, softplus, s
  switch (dtype) {
    case GDR_BF16: return ss_step_launch<__bf16>(SP_ARGS);
    case GDR_FP16: return ss_step_launch<_Float16>(SP_ARGS);
    case GDR_FP32: return ss_step_launch<float>(SP_ARGS);
    default: return LAMPA_ERR_INVALID;
  }
#undef SP_ARGS
}
