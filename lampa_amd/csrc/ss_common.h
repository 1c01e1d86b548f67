// Arguments, segment tables and small device helpers shared by the state-space scan kernels (gfx950).
//
// The operator, for one head of one sequence (state S [N, P], fp32):
//   delta_t = softplus(dt_t + bias)            (or dt_t + bias as it is)
//   S_t = exp(delta_t A) S_{t-1} + delta_t B_t x_t^T,      y_t = S_t^T C_t + D x_t.
// Its gradients run the adjoint R from the end, R_t = C_t dy_t^T + exp(delta_{t+1} A) R_{t+1}:
//   dC_t = S_t dy_t,   dB_t = delta_t R_t x_t,   dx_t = delta_t R_t^T B_t + D dy_t,
//   dg_t = <R_t, exp(g_t) S_{t-1}> = dg_{t+1} + dy_t.(S_t^T C_t) - delta_t x_t.(R_t^T B_t)     (g_t = delta_t A),
//   d delta_t = A dg_t + x_t.(R_t^T B_t).
//
// A sequence is cut into segments of seg_tokens tokens. A segment's effect on the state is affine with one scalar,
// S -> exp(sum g) S + S_local, so the segments' local states are computed in parallel, joined by a scan over the segments
// (element by element of the state), and the outputs are then computed in parallel from every segment's initial state.
#pragma once
#include "../../include/lampa_amd.h"
#include "gdr_ops.h"

// Decay exponents below this leave nothing of an fp32 value (exp(-104) is below the smallest denormal): clamped there, a sum over the
// 64 tokens of a chunk stays within 9 600 (as an exponent of 2) however strongly tokens cut the past off. The chunk kernels sum in
// 64 bits; a pair's weight takes the difference of two such sums rounded to fp32, each off by half a step: 2^-16 each behind two
// clamped tokens of a chunk, 2^-11 each (7e-4 of the weight) behind 63.
#define SS_MIN_LOG_DECAY (-104.0f)

struct SsSegment {
  int64_t t0, t1;   // tokens of this segment
  int seq, index;   // sequence, place of the segment in it
  int64_t begin;    // first token of the sequence
  bool live;        // false: this slot holds no segment
  bool outside;     // rows behind the last sequence: their outputs are zero
};

// Boundary i of the sequences; boundaries read from the device are held inside the tensors.
__device__ __forceinline__ int64_t ss_bound(const lampa_ss_args& a, int i) {
  if (!a.cu_seqlens) return (int64_t)i * a.seq_len;
  if (i == 0) return 0;
  if (i > a.n_seq) return a.n_tokens;
  const int64_t c = a.cu_seqlens[i];
  return c < 0 ? 0 : (c > a.n_tokens ? a.n_tokens : c);
}
// First slot of sequence i. Packed sequences take floor(begin / S) + i: room for every sequence's ceil(length / S) segments
// (at least one, so that an empty sequence has a slot) without knowing the lengths on the host.
__device__ __forceinline__ int64_t ss_first_slot(const lampa_ss_args& a, int i) {
  if (!a.cu_seqlens) return (int64_t)i * ((a.seq_len + a.seg_tokens - 1) / a.seg_tokens);
  return ss_bound(a, i) / a.seg_tokens + i;
}
__device__ __forceinline__ SsSegment ss_segment(const lampa_ss_args& a, int64_t slot) {
  SsSegment s;
  int64_t b, e;
  if (!a.cu_seqlens) {
    const int64_t per = (a.seq_len + a.seg_tokens - 1) / a.seg_tokens;
    s.seq = (int)(slot / per);
    s.index = (int)(slot % per);
    s.live = s.seq < a.n_seq;
    s.outside = false;
    b = (int64_t)s.seq * a.seq_len;
    e = b + a.seq_len;
  } else {
    int lo = 0, hi = a.n_seq;  // the rows behind the last sequence count as sequence n_seq
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ss_bound(a, mid) / a.seg_tokens + mid <= slot) lo = mid; else hi = mid - 1;
    }
    s.seq = lo;
    b = ss_bound(a, lo);
    e = ss_bound(a, lo + 1);
    const int64_t index = slot - (b / a.seg_tokens + lo);
    s.index = (int)index;
    s.outside = lo == a.n_seq;
    s.live = index >= 0 && (index == 0 || b + index * a.seg_tokens < e);
  }
  s.t0 = b + (int64_t)s.index * a.seg_tokens;
  s.t1 = s.t0 + a.seg_tokens < e ? s.t0 + a.seg_tokens : e;
  if (s.t1 < s.t0) s.t1 = s.t0;
  s.begin = b;
  return s;
}

// Element i of dt (a row of it, from its head's column), which is of the other tensors' type or fp32.
template <typename T>
__device__ __forceinline__ float ss_load_dt(const void* dt, int dt_dtype, int64_t i) {
  return dt_dtype == GDR_FP32 ? ((const float*)dt)[i] : GdrElem<T>::to_float(((const T*)dt)[i]);
}
// Row of a segment's first tokens in a table with one row for every `every` tokens of a sequence (a divisor of 64): sequence i
// takes its rows from floor(begin / every) + i on, as it takes its slots.
__device__ __forceinline__ int64_t ss_row_of(const SsSegment& s, int every) { return s.begin / every + s.seq + (s.t0 - s.begin) / every; }

__device__ __forceinline__ float ss_delta(float raw, float bias, int softplus) {
  const float x = raw + bias;
  return softplus ? (x > 20.0f ? x : log1pf(expf(x))) : x;
}
__device__ __forceinline__ float ss_log_decay(float delta, float A) {
  const float g = delta * A;
  return g < SS_MIN_LOG_DECAY ? SS_MIN_LOG_DECAY : g;  // a NaN stays one
}

// Sum over the 64 lanes of a wave, in every lane (the last lane of a prefix sum has it; no LDS round trips).
__device__ __forceinline__ float ss_wave_sum(float x) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_inclusive_scan(x)), 63));
}

static inline int ss_blocks64(int n) { return (n + 63) / 64; }

// Slots of a call (what the launchers size their grids and tables by).
static inline int64_t ss_slots(const lampa_ss_args* a) {
  if (!a->cu_seqlens) return (int64_t)a->n_seq * ((a->seq_len + a->seg_tokens - 1) / a->seg_tokens);
  return a->n_tokens / a->seg_tokens + a->n_seq + 1;
}
static inline int64_t ss_rows(const lampa_ss_args* a, int every) { return a->n_tokens / every + a->n_seq + 1; }  // of ss_row_of's tables
// One segment holds any sequence: no scan over segments, the walks start from h0 and leave the final states themselves.
static inline bool ss_single(const lampa_ss_args* a) {
  return (a->cu_seqlens ? a->n_tokens : a->seq_len) <= a->seg_tokens;
}
