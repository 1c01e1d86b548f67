// The causal short convolution with what precedes and follows a call, on gfx950 (its plain forward is in layer_ops.hip):
//   * forward on top of the inputs before the first token (a cache of the last W inputs), the last W inputs handed on;
//   * one token for each sequence, the cache moved on;
//   * gradients of x, the taps and the bias.
//   pre[t] = bias + sum_{j < W} w[j] x[t - (W-1) + j],  y = pre or pre sigmoid(pre)
//   dpre[t] = dy[t] y'(pre[t]),  dx[s] = sum_j w[j] dpre[s + W-1 - j],  dw[j] = sum_t dpre[t] x[t - (W-1) + j],  dbias = sum_t dpre[t]
// Bound by bytes: every row of x (and dy) is read once, plus W - 1 (and 2 (W - 1)) rows of history for every run of tokens,
// which hit in L2. Arithmetic is fp32, results are rounded once.
//
// Measured: gradients of 60 000 x 640 in bf16 65 us (230 MB, 3.5 TB/s) and 10 us for the sums over the workgroups' rows (the
// vector instructions, about 30 a value, are what is left: 40 us of it); forward with state, 24 packed sequences of 15 000 x 224 in fp16
// 19 us, one sequence of 60 000 x 640 in bf16 / fp32 44 / 80 us with the host (153 / 307 MB).
#include "gdr_common.h"
#include "row_sums.h"

#define CC_BLOCK 256
#define CC_MAX_W 8

__device__ __forceinline__ float cc_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

struct CcSeq {
  const int64_t* cu;  // device [n_seq + 1] or null: dense sequences of len tokens
  int n_seq;
  int64_t len, n_tokens;
};
__device__ __forceinline__ int64_t cc_bound(const CcSeq& q, int i) {
  if (!q.cu) return i * q.len;
  if (i == 0) return 0;
  if (i > q.n_seq) return q.n_tokens;
  const int64_t c = q.cu[i];
  return c < 0 ? 0 : (c > q.n_tokens ? q.n_tokens : c);
}
// Sequence of token t; n_seq for the rows behind the last one.
__device__ __forceinline__ int cc_seq_of(const CcSeq& q, int64_t t) {
  if (!q.cu) return (int)(t / q.len);
  int lo = 0, hi = q.n_seq;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cc_bound(q, mid) <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ void cc_store8(T* dst, const float* v) {
  if constexpr (sizeof(T) == 2) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    vec8 o;
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = GdrElem<T>::from_float(v[c]);
    *reinterpret_cast<vec8*>(dst) = o;
  } else {
    *reinterpret_cast<f32x4*>(dst) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(dst + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// ------------------------------------------------------------------------------------------------ forward with state
// One thread: 8 channels x CF_TOKENS tokens, its W - 1 rows of history in registers. The workgroups behind the tokens' ones
// write the caches. Rows behind the last sequence come back as zero.
#define CF_TOKENS 8

template <typename T, int W>
__global__ void __launch_bounds__(CC_BLOCK) cc_fwd_kernel(const T* __restrict__ x, int64_t x_stride, int D, CcSeq q,
                                                          const float* __restrict__ weight, const float* __restrict__ bias,
                                                          const T* __restrict__ past, int act, T* __restrict__ y,
                                                          T* __restrict__ last, int64_t token_blocks) {
  const int groups = D / 8;
  if ((int64_t)blockIdx.x >= token_blocks) {
    const int64_t i = ((int64_t)blockIdx.x - token_blocks) * CC_BLOCK + threadIdx.x;
    if (i >= (int64_t)q.n_seq * D) return;
    const int seq = (int)(i / D), d = (int)(i % D);
    const int64_t b = cc_bound(q, seq), e = cc_bound(q, seq + 1), n = e > b ? e - b : 0;
    T keep[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (n - W + w >= 0) keep[w] = x[(b + n - W + w) * x_stride + d];
      else keep[w] = past ? past[i * W + n + w] : (T)0.0f;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) last[i * W + w] = keep[w];
    return;
  }
  const int64_t item = (int64_t)blockIdx.x * CC_BLOCK + threadIdx.x;
  const int c0 = (int)(item % groups) * 8;
  const int64_t t0 = item / groups * CF_TOKENS;
  if (t0 >= q.n_tokens) return;
  float rows[CF_TOKENS + W - 1][8];
#pragma unroll
  for (int r = 0; r < CF_TOKENS + W - 1; ++r) {
    const int64_t t = t0 - (W - 1) + r;
    load8(x + (t < 0 ? 0 : (t < q.n_tokens ? t : q.n_tokens - 1)) * x_stride + c0, rows[r]);
  }
  float w[W][8], bv[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    bv[c] = bias ? bias[c0 + c] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][c] = weight[(int64_t)(c0 + c) * W + j];
  }
  int seq = cc_seq_of(q, t0);
  int64_t b = cc_bound(q, seq), e = cc_bound(q, seq + 1);
#pragma unroll
  for (int i = 0; i < CF_TOKENS; ++i) {
    const int64_t t = t0 + i;
    if (t >= q.n_tokens) break;
    if (t >= e) {
      seq = cc_seq_of(q, t);
      b = cc_bound(q, seq);
      e = cc_bound(q, seq + 1);
    }
    float out[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float v = 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int64_t from = t - (W - 1) + j;
        float xv = rows[i + j][c];
        if (from < b)
          xv = past && seq < q.n_seq ? GdrElem<T>::to_float(past[((int64_t)seq * D + c0 + c) * W + W + (from - b)]) : 0.0f;
        v = __builtin_fmaf(xv, w[j][c], v);
      }
      v += bv[c];
      if (act) v *= cc_sigmoid(v);
      out[c] = seq < q.n_seq ? v : 0.0f;
    }
    cc_store8(y + t * D + c0, out);
  }
}

// ------------------------------------------------------------------------------------------------------- one token
template <typename T, int W>
__global__ void __launch_bounds__(CC_BLOCK) cc_step_kernel(const T* __restrict__ x, int64_t x_stride, const T* cache,
                                                           T* new_cache, const float* __restrict__ weight,
                                                           const float* __restrict__ bias, int act, T* __restrict__ y, int64_t n,
                                                           int D) {
  const int64_t i = (int64_t)blockIdx.x * CC_BLOCK + threadIdx.x;
  if (i >= n * D) return;
  const int64_t b = i / D;
  const int d = (int)(i % D);
  T keep[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) keep[j] = cache[i * W + j + 1];
  keep[W - 1] = x[b * x_stride + d];
  float v = 0.0f;
#pragma unroll
  for (int j = 0; j < W; ++j) v = __builtin_fmaf(GdrElem<T>::to_float(keep[j]), weight[(int64_t)d * W + j], v);
  v += bias ? bias[d] : 0.0f;
  if (act) v *= cc_sigmoid(v);
  y[i] = GdrElem<T>::from_float(v);
#pragma unroll
  for (int j = 0; j < W; ++j) new_cache[i * W + j] = keep[j];
}

// ------------------------------------------------------------------------------------------------------- gradients
// A workgroup takes 32 groups of 4 channels and, side by side, 8 runs of CB_TOKENS tokens; it goes over the tokens in strides of
// the whole grid and leaves one share of dw and dbias, added up over its runs in a fixed order. Rows are requested four at a
// time, one four ahead. (Eight channels a thread, or all rows of a run requested at once, take over 200 registers: 138 and
// 151 us at 60 000 x 640 in bf16.)
#define CB_CH 4
#define CB_TOKENS 16
#define CB_LANES 32
#define CB_RUNS (CC_BLOCK / CB_LANES)

template <typename T>
struct CbRaw { typedef T vec __attribute__((ext_vector_type(CB_CH))); };

// One run of tokens of one thread. EDGE: a sequence may begin or end among the rows that are looked at (t0 - (W-1) .. t0 +
// CB_TOKENS + W-2); without, no row is masked.
template <typename T, int W, bool EDGE>
__device__ __forceinline__ void cc_bwd_run(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy, int D, const CcSeq& q,
                                           const float (&w)[W][CB_CH], const float (&bv)[CB_CH], const T* __restrict__ past, int act,
                                           T* __restrict__ dx, int64_t t0, int c0, int seq, int64_t b, int64_t e,
                                           float (&dw)[W][CB_CH], float (&db)[CB_CH]) {
  typedef typename CbRaw<T>::vec raw;
  constexpr int ROWS = CB_TOKENS + W - 1, GROUPS = (ROWS + 3) / 4;
  float win[W][CB_CH], dpre[W][CB_CH];  // x of the last W rows; dpre of the last W tokens
  int64_t begins[W];                    // where the sequences of the last W tokens begin
#pragma unroll
  for (int r = 0; r < W; ++r) {
    begins[r] = 0;
#pragma unroll
    for (int c = 0; c < CB_CH; ++c) win[r][c] = dpre[r][c] = 0.0f;
  }
  raw rx[2][4], ry[2][4];
  auto fetch = [&](int group) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 4 * group + k;
      if (i >= ROWS) continue;
      int64_t t = t0 + i;
      if (EDGE && t >= q.n_tokens) t = q.n_tokens - 1;  // not used
      rx[group & 1][k] = *reinterpret_cast<const raw*>(x + t * x_stride + c0);
      ry[group & 1][k] = *reinterpret_cast<const raw*>(dy + t * D + c0);
    }
  };
  fetch(0);
#pragma unroll
  for (int r = 0; r < W - 1; ++r) {
    const int64_t t = t0 - (W - 1) + r;
    if (!EDGE || t >= 0) {
      const raw v = *reinterpret_cast<const raw*>(x + t * x_stride + c0);
#pragma unroll
      for (int c = 0; c < CB_CH; ++c) win[r + 1][c] = GdrElem<T>::to_float(v[c]);
    }
  }
#pragma unroll
  for (int group = 0; group < GROUPS; ++group) {
    if (group + 1 < GROUPS) fetch(group + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 4 * group + k;
      if (i >= ROWS) continue;
      const int64_t t = t0 + i;
#pragma unroll
      for (int r = 0; r + 1 < W; ++r) {
        begins[r] = begins[r + 1];
#pragma unroll
        for (int c = 0; c < CB_CH; ++c) { win[r][c] = win[r + 1][c]; dpre[r][c] = dpre[r + 1][c]; }
      }
      if (!EDGE || t < q.n_tokens) {
        if (EDGE && t >= e) {
          seq = cc_seq_of(q, t);
          b = cc_bound(q, seq);
          e = cc_bound(q, seq + 1);
        }
        begins[W - 1] = b;
        const bool inside = !EDGE || seq < q.n_seq;  // rows behind the last sequence may hold anything: no share in any sum
#pragma unroll
        for (int c = 0; c < CB_CH; ++c) {
          win[W - 1][c] = GdrElem<T>::to_float(rx[group & 1][k][c]);
          float taps[W], pre = 0.0f;
#pragma unroll
          for (int j = 0; j < W; ++j) {
            const int64_t src = t - (W - 1) + j;
            taps[j] = win[j][c];
            if (EDGE && src < b)
              taps[j] = past && inside ? GdrElem<T>::to_float(past[((int64_t)seq * D + c0 + c) * W + W + (src - b)]) : 0.0f;
            if (EDGE && !inside) taps[j] = 0.0f;
            pre = __builtin_fmaf(taps[j], w[j][c], pre);
          }
          pre += bv[c];
          float d = GdrElem<T>::to_float(ry[group & 1][k][c]);
          if (act) {
            const float s = cc_sigmoid(pre);
            d *= s * __builtin_fmaf(pre, 1.0f - s, 1.0f);
          }
          if (EDGE && !inside) d = 0.0f;
          dpre[W - 1][c] = d;
          if (i < CB_TOKENS) {
            db[c] += d;
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j][c] = __builtin_fmaf(d, taps[j], dw[j][c]);
          }
        }
      } else {
        begins[W - 1] = INT64_MAX;
#pragma unroll
        for (int c = 0; c < CB_CH; ++c) win[W - 1][c] = dpre[W - 1][c] = 0.0f;
      }
      const int64_t s = t - (W - 1);
      if (i >= W - 1 && (!EDGE || s < q.n_tokens)) {  // dx of token s: dpre[r] belongs to token s + r
        raw out;
#pragma unroll
        for (int c = 0; c < CB_CH; ++c) {
          float v = 0.0f;
#pragma unroll
          for (int r = 0; r < W; ++r) v = __builtin_fmaf(!EDGE || begins[r] <= s ? dpre[r][c] : 0.0f, w[W - 1 - r][c], v);
          out[c] = GdrElem<T>::from_float(v);
        }
        *reinterpret_cast<raw*>(dx + s * D + c0) = out;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(CC_BLOCK) cc_bwd_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ dy,
                                                          int D, CcSeq q, const float* __restrict__ weight,
                                                          const float* __restrict__ bias, const T* __restrict__ past, int act,
                                                          T* __restrict__ dx, float* __restrict__ parts) {
  constexpr int ROWS = CB_TOKENS + W - 1;
  const int groups = D / CB_CH, cl = threadIdx.x % CB_LANES, run = threadIdx.x / CB_LANES;
  const int cg = blockIdx.x * CB_LANES + cl, c0 = cg * CB_CH;
  const bool on = cg < groups;
  float w[W][CB_CH], bv[CB_CH], dw[W][CB_CH], db[CB_CH];
#pragma unroll
  for (int c = 0; c < CB_CH; ++c) {
    bv[c] = on && bias ? bias[c0 + c] : 0.0f;
    db[c] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      w[j][c] = on ? weight[(int64_t)(c0 + c) * W + j] : 0.0f;
      dw[j][c] = 0.0f;
    }
  }
  for (int64_t t0 = ((int64_t)blockIdx.y * CB_RUNS + run) * CB_TOKENS; t0 < q.n_tokens && on;
       t0 += (int64_t)gridDim.y * CB_RUNS * CB_TOKENS) {
    const int seq = cc_seq_of(q, t0);
    const int64_t b = cc_bound(q, seq), e = cc_bound(q, seq + 1);
    if (__all(seq < q.n_seq && t0 - (W - 1) >= b && t0 + ROWS <= e))
      cc_bwd_run<T, W, false>(x, x_stride, dy, D, q, w, bv, past, act, dx, t0, c0, seq, b, e, dw, db);
    else
      cc_bwd_run<T, W, true>(x, x_stride, dy, D, q, w, bv, past, act, dx, t0, c0, seq, b, e, dw, db);
  }
  // over the 8 runs: 2 in a wave, then the 4 waves
  __shared__ float red[4][CB_LANES][CB_CH * (W + 1)];
#pragma unroll
  for (int c = 0; c < CB_CH; ++c)
#pragma unroll
    for (int j = 0; j <= W; ++j) {
      float v = j < W ? dw[j < W ? j : 0][c] : db[c];
      v += __shfl_xor(v, CB_LANES);
      if ((threadIdx.x & 63) < CB_LANES) red[threadIdx.x >> 6][cl][c * (W + 1) + j] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < CB_LANES * CB_CH * (W + 1); i += CC_BLOCK) {
    const int g = i / (CB_CH * (W + 1)), k = i % (CB_CH * (W + 1));
    if (blockIdx.x * CB_LANES + g < groups)
      parts[((int64_t)blockIdx.y * D + (blockIdx.x * CB_LANES + g) * CB_CH) * (W + 1) + k] =
          (red[0][g][k] + red[1][g][k]) + (red[2][g][k] + red[3][g][k]);
  }
}

// Workgroups along the tokens: eight a CU over the whole call where there are tokens enough (each leaves a row of sums).
static int cc_bwd_runs(int64_t n_tokens, int D) {
  const int64_t need = (n_tokens + CB_RUNS * CB_TOKENS - 1) / (CB_RUNS * CB_TOKENS);
  const int64_t most = 2048 / ((D / CB_CH + CB_LANES - 1) / CB_LANES) + 1;
  return (int)(need < 1 ? 1 : (need < most ? need : most));
}

static int cc_check(const void* x, int64_t x_stride, int64_t n_tokens, int D, int W, const float* weight, const int64_t* cu, int n_seq,
                    int64_t seq_len, int act, int dtype) {
  if ((n_tokens && !x) || !weight || n_tokens < 0 || D < 1 || W < 1 || x_stride < D || n_seq < 1 || act < 0 || act > 1 || dtype < 0 || dtype > 2)
    return LAMPA_ERR_INVALID;
  if (!cu && (seq_len < 0 || seq_len * n_seq != n_tokens)) return LAMPA_ERR_INVALID;
  if (W > CC_MAX_W || D % 8 || x_stride % 8 || (uintptr_t)x % 16) return LAMPA_ERR_UNSUPPORTED;
  return LAMPA_OK;
}

#define CC_WIDTHS(GO) \
  switch (W) { GO(1) GO(2) GO(3) GO(4) GO(5) GO(6) GO(7) GO(8) default: return LAMPA_ERR_UNSUPPORTED; }

template <typename T>
static int cc_fwd_launch(const void* x, int64_t x_stride, int D, int W, CcSeq q, const float* weight, const float* bias,
                         const void* past, int act, void* y, void* last, hipStream_t s) {
  const int64_t items = (int64_t)(D / 8) * ((q.n_tokens + CF_TOKENS - 1) / CF_TOKENS);
  const int64_t tb = (items + CC_BLOCK - 1) / CC_BLOCK, lb = last ? ((int64_t)q.n_seq * D + CC_BLOCK - 1) / CC_BLOCK : 0;
  if (tb + lb == 0) return LAMPA_OK;
  if (tb + lb > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  LAMPA_PROF(s, "start");
#define CC_GO(WW)                                                                                                             \
  case WW:                                                                                                                    \
    hipLaunchKernelGGL((cc_fwd_kernel<T, WW>), dim3((unsigned)(tb + lb)), dim3(CC_BLOCK), 0, s, (const T*)x, x_stride, D, q, weight, \
                       bias, (const T*)past, act, (T*)y, (T*)last, tb);                                                       \
    break;
  CC_WIDTHS(CC_GO)
#undef CC_GO
  LAMPA_PROF(s, "cc_fwd_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_causal_conv1d_state_fwd(const void* x, int64_t x_stride, int64_t n_tokens, int D, int W, const float* weight,
                                             const float* bias, const void* past, const int64_t* cu_seqlens, int n_seq,
                                             int64_t seq_len, int activation, int dtype, void* y, void* last, void* stream) {
  const int rc = cc_check(x, x_stride, n_tokens, D, W, weight, cu_seqlens, n_seq, seq_len, activation, dtype);
  if (rc != LAMPA_OK) return rc;
  if (n_tokens && (!y || (uintptr_t)y % 16)) return LAMPA_ERR_INVALID;
  const CcSeq q{cu_seqlens, n_seq, seq_len, n_tokens};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case GDR_BF16: return cc_fwd_launch<__bf16>(x, x_stride, D, W, q, weight, bias, past, activation, y, last, s);
    case GDR_FP16: return cc_fwd_launch<_Float16>(x, x_stride, D, W, q, weight, bias, past, activation, y, last, s);
    default: return cc_fwd_launch<float>(x, x_stride, D, W, q, weight, bias, past, activation, y, last, s);
  }
}

template <typename T>
static int cc_step_launch(const void* x, int64_t x_stride, const void* cache, void* new_cache, const float* weight, const float* bias,
                          int act, void* y, int64_t n, int D, int W, hipStream_t s) {
  const int64_t blocks = (n * D + CC_BLOCK - 1) / CC_BLOCK;
  if (blocks > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  LAMPA_PROF(s, "start");
#define CC_GO(WW)                                                                                                                \
  case WW:                                                                                                                       \
    hipLaunchKernelGGL((cc_step_kernel<T, WW>), dim3((unsigned)blocks), dim3(CC_BLOCK), 0, s, (const T*)x, x_stride, (const T*)cache, \
                       (T*)new_cache, weight, bias, act, (T*)y, n, D);                                                           \
    break;
  CC_WIDTHS(CC_GO)
#undef CC_GO
  LAMPA_PROF(s, "cc_step_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_causal_conv1d_step(const void* x, int64_t x_stride, const void* cache, void* new_cache, const float* weight,
                                        const float* bias, int activation, int dtype, void* y, int64_t n, int D, int W,
                                        void* stream) {
  if (!x || !cache || !new_cache || !weight || !y || n < 0 || D < 1 || W < 1 || x_stride < D || activation < 0 || activation > 1)
    return LAMPA_ERR_INVALID;
  if (W > CC_MAX_W) return LAMPA_ERR_UNSUPPORTED;
  if (n == 0) return LAMPA_OK;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case GDR_BF16: return cc_step_launch<__bf16>(x, x_stride, cache, new_cache, weight, bias, activation, y, n, D, W, s);
    case GDR_FP16: return cc_step_launch<_Float16>(x, x_stride, cache, new_cache, weight, bias, activation, y, n, D, W, s);
    case GDR_FP32: return cc_step_launch<float>(x, x_stride, cache, new_cache, weight, bias, activation, y, n, D, W, s);
    default: return LAMPA_ERR_INVALID;
  }
}

extern "C" int64_t lampa_causal_conv1d_bwd_workspace_bytes(int64_t n_tokens, int D, int W, int dtype) {
  if (n_tokens < 0 || D < 8 || D % 8 || W < 1 || W > CC_MAX_W || dtype < 0 || dtype > 2) return LAMPA_ERR_INVALID;
  return (int64_t)cc_bwd_runs(n_tokens, D) * D * (W + 1) * 4;
}

template <typename T>
static int cc_bwd_launch(const void* x, int64_t x_stride, const void* dy, int D, int W, CcSeq q, const float* weight,
                         const float* bias, const void* past, int act, void* dx, float* parts, int runs, hipStream_t s) {
  const dim3 grid((unsigned)((D / CB_CH + CB_LANES - 1) / CB_LANES), (unsigned)runs);
  LAMPA_PROF(s, "start");
#define CC_GO(WW)                                                                                                            \
  case WW:                                                                                                                   \
    hipLaunchKernelGGL((cc_bwd_kernel<T, WW>), grid, dim3(CC_BLOCK), 0, s, (const T*)x, x_stride, (const T*)dy, D, q, weight, bias, \
                       (const T*)past, act, (T*)dx, parts);                                                                  \
    break;
  CC_WIDTHS(CC_GO)
#undef CC_GO
  LAMPA_PROF(s, "cc_bwd_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_causal_conv1d_bwd(const void* x, int64_t x_stride, const void* dy, int64_t n_tokens, int D, int W,
                                       const float* weight, const float* bias, const void* past, const int64_t* cu_seqlens, int n_seq,
                                       int64_t seq_len, int activation, int dtype, void* dx, float* dweight_bias, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  const int rc = cc_check(x, x_stride, n_tokens, D, W, weight, cu_seqlens, n_seq, seq_len, activation, dtype);
  if (rc != LAMPA_OK) return rc;
  if (!dweight_bias || (n_tokens && (!dy || !dx || ((uintptr_t)dy | (uintptr_t)dx) % 16))) return LAMPA_ERR_INVALID;
  if (!workspace || workspace_bytes < lampa_causal_conv1d_bwd_workspace_bytes(n_tokens, D, W, dtype)) return LAMPA_ERR_WORKSPACE;
  const CcSeq q{cu_seqlens, n_seq, seq_len, n_tokens};
  const int runs = cc_bwd_runs(n_tokens, D);
  float* parts = (float*)workspace;
  hipStream_t s = (hipStream_t)stream;
  int e;
  switch (dtype) {
    case GDR_BF16: e = cc_bwd_launch<__bf16>(x, x_stride, dy, D, W, q, weight, bias, past, activation, dx, parts, runs, s); break;
    case GDR_FP16: e = cc_bwd_launch<_Float16>(x, x_stride, dy, D, W, q, weight, bias, past, activation, dx, parts, runs, s); break;
    default: e = cc_bwd_launch<float>(x, x_stride, dy, D, W, q, weight, bias, past, activation, dx, parts, runs, s); break;
  }
  if (e != LAMPA_OK) return e;
  const int64_t cols = (int64_t)D * (W + 1);
  return row_sums_launch<float>(parts, runs, cols, cols, 0, 1, RowSumsOut<float>{{dweight_bias, nullptr, nullptr}, 0}, s);
}
