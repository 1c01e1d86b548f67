// Shared by the kernels of the gated feed-forward block (gfx950).
//   forward:    G = x Wg^T,  U = x Wu^T,  S = act(G) * U,  y = S Wd^T
//   gradients:  dS = dy Wd,  dG = dS * U * act'(G),  dU = dS * act(G),
//               dx = dG Wg + dU Wu,  dWg = dG^T x,  dWu = dU^T x,  dWd = dy^T S.
// Products run on the matrix cores with fp32 sums (16-bit inputs on the 16-bit instructions, fp32 inputs on the fp32 ones).
// S, dG and dU are operands of further products. For 16-bit inputs they are rounded to the input type, half a step of each, which comes to as
// much as the outputs' own rounding; where the rows are few they enter as two parts, the rounding and what it left, so that outputs do not
// hang on a handful of roundings (each form states its rule). act and act' are taken from the unrounded fp32 sums in both passes.
#pragma once
#include "../../include/lampa_amd.h"
#include "gdr_ops.h"

enum { FF_ACT_NONE = 0, FF_ACT_SILU = 1, FF_ACT_SIGMOID = 2 };
#define FF_OFF 0x80000000u  // byte offset past the end of every buffer

__device__ __forceinline__ float ff_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
template <int ACT>
__device__ __forceinline__ float ff_act(float g) {
  if constexpr (ACT == FF_ACT_NONE) return g;
  const float s = ff_sigmoid(g);
  return ACT == FF_ACT_SILU ? g * s : s;
}
// (act(g), act'(g))
template <int ACT>
__device__ __forceinline__ void ff_act_slope(float g, float& value, float& slope) {
  if constexpr (ACT == FF_ACT_NONE) {
    value = g;
    slope = 1.0f;
  } else {
    const float s = ff_sigmoid(g);
    value = ACT == FF_ACT_SILU ? g * s : s;
    slope = ACT == FF_ACT_SILU ? __builtin_fmaf(value, 1.0f - s, s) : s * (1.0f - s);
  }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t ff_buffer(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes > 0 ? (unsigned)bytes : 0u, 0x00020000);
}
typedef unsigned ff_u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ ff_u32x4 ff_load16(__amdgpu_buffer_rsrc_t buf, unsigned offset) {
  return __builtin_bit_cast(ff_u32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, offset, 0, 0));
}

// Everything that this wave has asked memory for has come. Before a loop with loads of its own: a register loaded in front of the loop
// would otherwise be waited for inside it, and the loop's own loads, which are counted in order, with it.
__device__ __forceinline__ void ff_loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// Four consecutive values, rounded to T.
template <typename T>
__device__ __forceinline__ void ff_store4(T* p, float a, float b, float c, float d) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<vec4*>(p) = vec4{GdrElem<T>::from_float(a), GdrElem<T>::from_float(b), GdrElem<T>::from_float(c), GdrElem<T>::from_float(d)};
}

// What v's rounding to T leaves (none where there is no finite rest): v as two parts of T is off by half a step of half a step.
template <typename T>
__device__ __forceinline__ float ff_rest(float v) {
  const float rest = v - GdrElem<T>::to_float(GdrElem<T>::from_float(v));
  return __builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f;
}

// out[c] = sum over n rows, `step` values apart, of rows[c], in order; cols a multiple of 4.
template <typename T>
static __global__ void __launch_bounds__(256) ff_reduce_kernel(const float* __restrict__ rows, int n, int64_t cols, int64_t step, T* __restrict__ out) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= cols) return;
  f32x4 sum = *reinterpret_cast<const f32x4*>(rows + c);
  for (int r = 1; r < n; ++r) sum += *reinterpret_cast<const f32x4*>(rows + r * step + c);
  ff_store4(out + c, sum[0], sum[1], sum[2], sum[3]);
}
template <typename T>
static int ff_reduce(const float* rows, int n, int64_t cols, int64_t step, T* out, hipStream_t s) {
  hipLaunchKernelGGL((ff_reduce_kernel<T>), dim3((unsigned)((cols / 4 + 255) / 256)), dim3(256), 0, s, rows, n, cols, step, out);
  LAMPA_PROF(s, "ff_reduce_kernel");
  return lampa_launch_status();
}

// The general form (ff_gemm.hip): hidden values through memory.
int64_t ff_gemm_workspace(const lampa_ff_args* a, int backward);
int ff_gemm_fwd(const lampa_ff_args* a, hipStream_t s);
int ff_gemm_bwd(const lampa_ff_args* a, hipStream_t s);
// 16-bit types and D <= 128 (ff_fused.h): hidden values in registers (60 000 x 128, 512 hidden columns, bf16: forward 28 us, training
// step 146; the general form 55 and 263). Wider blocks' sums and operands do not fit a wave's registers.
static inline bool ff_fused_takes(const lampa_ff_args* a) { return a->dtype != GDR_FP32 && a->D <= 128; }
int64_t ff_fused_workspace(const lampa_ff_args* a, int backward);
int ff_fused_fwd_bf16(const lampa_ff_args* a, hipStream_t s);
int ff_fused_bwd_bf16(const lampa_ff_args* a, hipStream_t s);
int ff_fused_fwd_fp16(const lampa_ff_args* a, hipStream_t s);
int ff_fused_bwd_fp16(const lampa_ff_args* a, hipStream_t s);
