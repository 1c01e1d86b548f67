// The state-space scan's entry points on gfx950: checks, the scan over segments, the join of the gradients' parts.
//
// Replaces the selective scan behind Mamba2.forward (reference chengjiang123/Lampa: models/baselines/full_mamba2.py:221-430,
// models/baselines/hmamba.py:356-460), whose kernels the reference imports from a package it does not hold.
#include "ss_kernels.h"

#define SS_BLOCK 256

// S (or, from the end, R) across the segments of one sequence, one thread an element of the state: every slot's local state
// is replaced by the state its segment starts from, and what is left after the last one goes to `out`. A thread reads
// SS_AHEAD slots before it needs the first.
#define SS_AHEAD 16
template <bool REV>
__global__ void __launch_bounds__(SS_BLOCK) ss_join_kernel(lampa_ss_args a, float* __restrict__ states,
                                                           const float* __restrict__ init, float* __restrict__ out) {
  const int64_t per_h = (int64_t)a.N * a.P;
  const int64_t blocks = (per_h + SS_BLOCK - 1) / SS_BLOCK;
  const int64_t e = (int64_t)(blockIdx.x % blocks) * SS_BLOCK + threadIdx.x;
  const int h = (int)(blockIdx.x / blocks % a.H), seq = (int)(blockIdx.x / blocks / a.H);
  if (e >= per_h) return;
  const int64_t slot0 = a.n_tokens ? ss_first_slot(a, seq) : 0, len = ss_bound(a, seq + 1) - ss_bound(a, seq);
  const int64_t n = a.n_tokens && len > 0 ? (len + a.seg_tokens - 1) / a.seg_tokens : (a.n_tokens ? 1 : 0);
  const int64_t own = ((int64_t)seq * a.H + h) * per_h + e;
  float S = init ? init[own] : 0.0f;
  for (int64_t j0 = 0; j0 < n; j0 += SS_AHEAD) {
    float local[SS_AHEAD], decay[SS_AHEAD];
#pragma unroll
    for (int i = 0; i < SS_AHEAD; ++i) {
      const int64_t j = j0 + i, slot = slot0 + (REV ? n - 1 - j : j);
      local[i] = j < n ? states[(slot * a.H + h) * per_h + e] : 0.0f;
      decay[i] = j < n ? a.slot_decay[slot * a.H + h] : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < SS_AHEAD; ++i) {
      const int64_t j = j0 + i, slot = slot0 + (REV ? n - 1 - j : j);
      if (j < n) states[(slot * a.H + h) * per_h + e] = S;
      S = __builtin_fmaf(S, decay[i], local[i]);
    }
  }
  if (out) out[own] = S;
}

template <bool REV>
static int ss_join(const lampa_ss_args& a, float* states, const float* init, float* out, hipStream_t s) {
  const int64_t blocks = ((int64_t)a.N * a.P + SS_BLOCK - 1) / SS_BLOCK * a.H * a.n_seq;
  if (blocks > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  LAMPA_PROF(s, "start");
  hipLaunchKernelGGL((ss_join_kernel<REV>), dim3((unsigned)blocks), dim3(SS_BLOCK), 0, s, a, states, init, out);
  LAMPA_PROF(s, "ss_join_kernel");
  return lampa_launch_status();
}

// From the gradient of the decays to those of dt, A and dt_bias. One workgroup takes 256 tokens of a segment and head,
// a wave 64, a lane one. Where dg has not been summed up yet (fp32), it is here, SS_DOT tokens at a time from their end:
// dg_t = dg_{t+1} + read_t - delta_t behind_t, behind the last of them <R, S>: what ends at t minus what begins there. What a token
// passes to its own output is in neither. It does not cross a token; where decays are fast it is most of both, e^|g| of dg, and its
// rounding stayed in dg (ddt off by 22 half-steps at g = -3, now 4; 48 883 tokens at g = -1.2: dA 2.5e-6, now 2.5e-7). Starting anew
// that often keeps rounding errors of the sum, which pass on to every earlier token of it, from adding up (dA off by 2.5e-5 over
// segments of 256 tokens, 6e-6 over 64).
template <typename T>
__global__ void __launch_bounds__(SS_BLOCK) ss_decay_grad_kernel(lampa_ss_args a, SsGrad w, bool summed) {
  const SsSegment seg = ss_segment(a, blockIdx.x);
  const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t part_row = ((int64_t)blockIdx.x * gridDim.z + blockIdx.z) * a.H + h;
  const int npb = (a.P + 63) / 64, reads = summed ? npb : npb * ((a.N + 63) / 64);
  const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  float dA = 0.0f, dbias = 0.0f;
  const int64_t t0 = seg.t0 + (int64_t)SS_BLOCK * blockIdx.z + 64 * wave;
  if (seg.live && t0 < seg.t1) {
    const int64_t tok = t0 + lane;
    const bool on = tok < seg.t1 && !seg.outside;
    float raw = 0.0f, delta = 0.0f, dg = 0.0f, reach = 0.0f;
    if (on) {
      raw = ss_load_dt<T>(a.dt, a.dt_dtype, tok * a.dt_stride + h) + bias;
      delta = ss_delta(raw, 0.0f, a.softplus);
      for (int i = 0; i < reads; ++i) dg += w.dg[(tok * a.H + h) * reads + i];
      if (summed) {
        for (int i = 0; i < npb; ++i) reach += w.reach[(tok * a.H + h) * npb + i];
      } else {
        const float* pair = w.pair + (tok * a.H + h) * (1 + npb);
        float behind = 0.0f, own = 0.0f;
        for (int i = 0; i < npb; ++i) {
          behind += w.behind[(tok * a.H + h) * npb + i];
          own += pair[1 + i];
        }
        dg -= delta * behind;
        reach = __builtin_fmaf(pair[0], own, behind);
      }
    }
    if (!summed && !seg.outside) {
#pragma unroll
      for (int off = 1; off < SS_DOT; off <<= 1) {
        const float later = __shfl_down(dg, off);
        if (lane % SS_DOT + off < SS_DOT) dg += later;
      }
      const int64_t row = (ss_row_of(seg, SS_DOT) + (tok - seg.t0) / SS_DOT) * a.H + h;
      for (int i = 0; on && i < npb; ++i) dg += w.chunk_dots[row * npb + i];
    }
    if (tok < seg.t1) {
      float d = on ? __builtin_fmaf(A, dg, reach) : 0.0f;
      // the derivative of log(1 + e^x), which is used as x above 20
      if (on && a.softplus) d *= raw > 20.0f ? 1.0f : 1.0f / (1.0f + expf(-raw));
      if (a.dt_dtype == GDR_FP32) ((float*)a.ddt)[tok * a.H + h] = d;
      else ((T*)a.ddt)[tok * a.H + h] = GdrElem<T>::from_float(d);
      if (on) {
        dbias += d;
        dA = __builtin_fmaf(delta, dg, dA);
      }
    }
  }
  dA = ss_wave_sum(dA);
  dbias = ss_wave_sum(dbias);
  __shared__ float part[2][4];
  if (lane == 0) {
    part[0][wave] = dA;
    part[1][wave] = dbias;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const float* v = part[threadIdx.x];
    w.param_part[part_row * 2 + threadIdx.x] = (v[0] + v[1]) + (v[2] + v[3]);
  }
}

// The parts of dB and dC, one for each head and block of columns, added up over the heads of a group in their order. VW: columns
// a thread takes (4 where N allows: a wave then reads 1 KiB at a time).
template <typename T, int VW>
__global__ void __launch_bounds__(SS_BLOCK) ss_group_sum_kernel(const float* __restrict__ dB_part, const float* __restrict__ dC_part,
                                                                T* __restrict__ dB, T* __restrict__ dC, int64_t n, int N, int parts) {
  typedef float vec __attribute__((ext_vector_type(VW)));
  typedef T out_vec __attribute__((ext_vector_type(VW)));
  const int64_t i = ((int64_t)blockIdx.x * SS_BLOCK + threadIdx.x) * VW;
  if (i >= n) return;
  const int64_t row = i / N;
  const float* src = (blockIdx.y ? dC_part : dB_part) + row * parts * N + (i - row * N);
  vec sum = *reinterpret_cast<const vec*>(src);
#pragma unroll 4
  for (int j = 1; j < parts; ++j) sum += *reinterpret_cast<const vec*>(src + (int64_t)j * N);
  out_vec o;
#pragma unroll
  for (int e = 0; e < VW; ++e) o[e] = GdrElem<T>::from_float(sum[e]);
  *reinterpret_cast<out_vec*>((blockIdx.y ? dC : dB) + i) = o;
}

// dA, d dt_bias and dD of a head: its segments' shares in their order.
__global__ void __launch_bounds__(SS_BLOCK) ss_param_sum_kernel(lampa_ss_args a, SsGrad w, int64_t slots, int64_t pieces) {
  const int h = blockIdx.x, which = blockIdx.y, npb = (a.P + 63) / 64;
  float* out = which == 0 ? a.dA : which == 1 ? a.ddt_bias : a.dD;
  if (!out) return;
  float sum = 0.0f;
  if (which < 2) {
    for (int64_t row = threadIdx.x; row < slots * pieces; row += SS_BLOCK) sum += w.param_part[(row * a.H + h) * 2 + which];
  } else {
    for (int64_t slot = threadIdx.x; slot < slots; slot += SS_BLOCK)
      if (ss_segment(a, slot).live)
        for (int i = 0; i < npb; ++i) sum += w.dD_part[(slot * a.H + h) * npb + i];
  }
  __shared__ float part[4];
  sum = ss_wave_sum(sum);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) out[h] = (part[0] + part[1]) + (part[2] + part[3]);
}

static int ss_check(const lampa_ss_args* a) {
  if (!a || !a->A || a->n_tokens < 0 || (a->n_tokens && (!a->x || !a->dt || !a->B || !a->C)) || a->n_seq < 1 || a->H < 1 || a->P < 1 || a->G < 1 ||
      a->N < 1 || a->H % a->G || a->seg_tokens < 64 || a->seg_tokens % 64 || a->dtype < 0 || a->dtype > 2 ||
      (a->dt_dtype != a->dtype && a->dt_dtype != GDR_FP32))
    return LAMPA_ERR_INVALID;
  if (!a->cu_seqlens && (a->seq_len < 0 || a->seq_len * a->n_seq != a->n_tokens)) return LAMPA_ERR_INVALID;
  if (a->x_stride < (int64_t)a->H * a->P || a->dt_stride < a->H || a->B_stride < (int64_t)a->G * a->N ||
      a->C_stride < (int64_t)a->G * a->N)
    return LAMPA_ERR_INVALID;
  if (a->N > 128) return LAMPA_ERR_UNSUPPORTED;
  // a lane's offset within 64 rows is formed in 32 bits
  if (a->x_stride >= 1 << 24 || a->B_stride >= 1 << 24 || a->C_stride >= 1 << 24 || a->y_stride >= 1 << 24 ||
      (int64_t)a->H * (a->P + 63) * a->N >= 1 << 28)
    return LAMPA_ERR_UNSUPPORTED;
  // the grids' limits: slots along x, heads and blocks along y
  if (ss_slots(a) > 0x7fffffff || a->seg_tokens > (int64_t)65535 * SS_BLOCK || (int64_t)a->H * ss_blocks64(a->P) * 2 > 65535) return LAMPA_ERR_UNSUPPORTED;
  return LAMPA_OK;
}

extern "C" int64_t lampa_ss_slots(const lampa_ss_args* a) { return ss_check(a) == LAMPA_OK ? ss_slots(a) : ss_check(a); }

extern "C" int lampa_ss_scan_fwd(const lampa_ss_args* args, void* stream) {
  const int rc = ss_check(args);
  if (rc != LAMPA_OK) return rc;
  const lampa_ss_args& a = *args;
  hipStream_t s = (hipStream_t)stream;
  if (!a.n_tokens) return a.ht ? ss_join<false>(a, nullptr, a.h0, a.ht, s) : LAMPA_OK;
  if (!a.y || a.y_stride < (int64_t)a.H * a.P) return LAMPA_ERR_INVALID;
  if (!ss_single(&a)) {
    if (!a.slot_states || !a.slot_decay) return LAMPA_ERR_WORKSPACE;
    int e = a.dtype == GDR_FP32 ? ss_serial_maps(a, nullptr, s) : ss_chunk_maps(a, nullptr, s);
    if (e == LAMPA_OK) e = ss_join<false>(a, a.slot_states, a.h0, a.ht, s);
    if (e != LAMPA_OK) return e;
  }
  return a.dtype == GDR_FP32 ? ss_serial_walk(a, SS_Y, SsGrad{}, s) : ss_chunk_out(a, s);
}

// Workgroups of 256 tokens a segment takes.
static int64_t ss_pieces(const lampa_ss_args& a) {
  const int64_t most = a.cu_seqlens ? a.n_tokens : a.seq_len, longest = a.seg_tokens < most ? a.seg_tokens : most;
  return longest < 1 ? 1 : (longest + SS_BLOCK - 1) / SS_BLOCK;
}

static int64_t ss_grad_layout(const lampa_ss_args& a, char* base, SsGrad* w) {
  const int64_t slots = ss_slots(&a), npb = ss_blocks64(a.P), nnb = ss_blocks64(a.N);
  int64_t at = 0;
  auto take = [&](float*& p, int64_t n) {
    p = base ? (float*)(base + at) : nullptr;
    at += lampa_align_up(n * 4, 256);
  };
  SsGrad g;
  take(g.adjoints, ss_single(&a) ? 0 : slots * a.H * a.N * a.P);
  take(g.dB_part, a.n_tokens * a.H * npb * a.N);
  take(g.dC_part, a.n_tokens * a.H * npb * a.N);
  const bool serial = a.dtype == GDR_FP32;
  take(g.dg, a.n_tokens * a.H * npb * (serial ? nnb : 1));
  take(g.reach, serial ? 0 : a.n_tokens * a.H * npb);
  take(g.behind, serial ? a.n_tokens * a.H * npb : 0);
  take(g.pair, serial ? a.n_tokens * a.H * (1 + npb) : 0);
  take(g.chunk_states, ss_rows(&a, serial ? SS_DOT : 64) * a.H * (serial ? (int64_t)a.N * a.P : npb * ss_chunk_n(a.N) * 64));
  take(g.chunk_dots, serial ? ss_rows(&a, SS_DOT) * a.H * npb : 0);
  take(g.param_part, slots * ss_pieces(a) * a.H * 2);
  take(g.dD_part, slots * a.H * npb);
  if (w) *w = g;
  return at;
}

extern "C" int64_t lampa_ss_bwd_workspace_bytes(const lampa_ss_args* a) {
  const int rc = ss_check(a);
  return rc == LAMPA_OK ? ss_grad_layout(*a, nullptr, nullptr) : rc;
}

extern "C" int lampa_ss_scan_bwd(const lampa_ss_args* args, void* stream) {
  const int rc = ss_check(args);
  if (rc != LAMPA_OK) return rc;
  const lampa_ss_args& a = *args;
  if (!a.dA) return LAMPA_ERR_INVALID;
  if (a.n_tokens && (!a.dy || !a.dx || !a.ddt || !a.dB || !a.dC)) return LAMPA_ERR_INVALID;
  const int64_t need = ss_grad_layout(a, nullptr, nullptr);
  if (need && (!a.workspace || a.workspace_bytes < need)) return LAMPA_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  SsGrad w;
  ss_grad_layout(a, (char*)a.workspace, &w);
  const int64_t slots = a.n_tokens ? ss_slots(&a) : 0;
  const bool serial = a.dtype == GDR_FP32;
  int e = LAMPA_OK;
  if (!a.n_tokens) {
    if (a.dh0) e = ss_join<true>(a, nullptr, a.dht, a.dh0, s);
  } else {
    const bool single = ss_single(&a);
    if (!single && (!a.slot_states || !a.slot_decay)) return LAMPA_ERR_WORKSPACE;
    if (!serial) e = ss_chunk_maps(a, &w, s);
    else if (!single) e = ss_serial_maps(a, &w, s);
    if (e == LAMPA_OK && !single) e = ss_join<true>(a, w.adjoints, a.dht, a.dh0, s);
    if (serial) {
      for (int kind : {SS_DC, SS_DX, SS_DB})
        if (e == LAMPA_OK) e = ss_serial_walk(a, kind, w, s);
    } else if (e == LAMPA_OK) {
      e = ss_chunk_grad(a, w, s);
    }
    if (e != LAMPA_OK) return e;
    const int64_t n = a.n_tokens * a.G * a.N;
    const bool wide = a.N % 4 == 0 && ((uintptr_t)a.dB | (uintptr_t)a.dC) % 16 == 0;
    const int64_t per = SS_BLOCK * (wide ? 4 : 1);
    const dim3 sums((unsigned)((n + per - 1) / per), 2), segs((unsigned)slots, (unsigned)a.H, (unsigned)ss_pieces(a));
    const int parts = a.H / a.G * ss_blocks64(a.P);
#define SS_TAIL(T)                                                                                                          \
  hipLaunchKernelGGL((ss_decay_grad_kernel<T>), segs, dim3(SS_BLOCK), 0, s, a, w, !serial);                                          \
  LAMPA_PROF(s, "ss_decay_grad_kernel");                                                                                    \
  if (wide)                                                                                                                 \
    hipLaunchKernelGGL((ss_group_sum_kernel<T, 4>), sums, dim3(SS_BLOCK), 0, s, w.dB_part, w.dC_part, (T*)a.dB, (T*)a.dC, n, a.N, parts); \
  else                                                                                                                      \
    hipLaunchKernelGGL((ss_group_sum_kernel<T, 1>), sums, dim3(SS_BLOCK), 0, s, w.dB_part, w.dC_part, (T*)a.dB, (T*)a.dC, n, a.N, parts); \
  LAMPA_PROF(s, "ss_group_sum_kernel");
    if (n > (int64_t)0x7fffffff * SS_BLOCK) return LAMPA_ERR_UNSUPPORTED;
    LAMPA_PROF(s, "start");
    switch (a.dtype) {
      case GDR_BF16: SS_TAIL(__bf16) break;
      case GDR_FP16: SS_TAIL(_Float16) break;
      default: SS_TAIL(float) break;
    }
#undef SS_TAIL
  }
  if (e != LAMPA_OK) return e;
  hipLaunchKernelGGL(ss_param_sum_kernel, dim3((unsigned)a.H, 3), dim3(SS_BLOCK), 0, s, a, w, slots, ss_pieces(a));
  LAMPA_PROF(s, "ss_param_sum_kernel");
  return lampa_launch_status();
}
