// Chunked forward of the state-space scan on the matrix cores: the segments' local states, and the outputs (see ss_chunk.h).
#include "ss_chunk.h"

// A segment's local state, or (REV) local adjoint: sum over its tokens of B_s (delta_s e^{gamma_end - gamma_s} x_s)^T, or of
// C_t (e^{gamma_t} dy_t)^T with gamma counted from the segment's start. Reads x and B (dy and C) once.
// KEEP: the walk starts from the segment's initial state and leaves the state in front of every chunk in w.chunk_states, in the
// order in which the gradients' lanes read it (sc_kept_at).
template <typename T, int NP>
struct ScMapTiles {
  static const int KS = NP + 8, VS = 64 + 8;
  __align__(16) T k[64 * KS], v[64 * VS];
  __align__(16) ScDecay dec;
};
template <typename T, int NP, bool REV, bool KEEP, bool VEC, int PARTS>
__device__ __forceinline__ void sc_map(const lampa_ss_args& a, const SsGrad& w, ScMapTiles<T, NP>& tiles) {
  constexpr int NT = NP / 16, KS = NP + 8, VS = 64 + 8;
  const SsSegment seg = ss_segment(a, blockIdx.x);
  if (!seg.live) return;
  const int npb = (a.P + 63) / 64, pb = blockIdx.y % npb, h = blockIdx.y / npb, grp = h / (a.H / a.G);
  const int lane0 = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = a.P - 64 * pb < 64 ? a.P - 64 * pb : 64;
  T *tk = tiles.k, *tv = tiles.v;
  ScDecay& dec = tiles.dec;
  const T* kb = (REV ? (const T*)a.C : (const T*)a.B) + (int64_t)grp * a.N;
  const T* vb = (REV ? (const T*)a.dy : (const T*)a.x) + (int64_t)h * a.P + 64 * pb;
  const int64_t ks = REV ? a.C_stride : a.B_stride, vs = REV ? (int64_t)a.H * a.P : a.x_stride;
  const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  const int64_t chunks = seg.outside ? 0 : (seg.t1 - seg.t0 + 63) / 64;

  f32x4 S[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int p = 64 * pb + 16 * wave + (lane0 & 15);
  if (KEEP) {
    const bool single = (a.cu_seqlens ? a.n_tokens : a.seq_len) <= a.seg_tokens;
    const float* init = single ? a.h0 : a.slot_states;
    if (init) init += ((single ? (int64_t)seg.seq : (int64_t)blockIdx.x) * a.H + h) * a.N * a.P;
    if (init && !seg.outside)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[nt][r] = sc_state_at(init, 16 * nt + 4 * (lane0 >> 4) + r, p, a.N, a.P);
  }
  ScTile<T, NP> pk;
  ScTile<T, 64> pv;
  float pdt = 0.0f, sum = 0.0f, sign = 1.0f;  // sign (REV): of S, and of dy in this chunk
  auto fetch = [&](int64_t c) {
    const int64_t t0 = seg.t0 + 64 * (REV ? chunks - 1 - c : c);
    const int n = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    pk.template fetch<VEC>(kb + t0 * ks, ks, n, a.N);
    pv.template fetch<VEC>(vb + t0 * vs, vs, n, cols);
    if (wave == 0 && lane0 < n) pdt = ss_load_dt<T>(a.dt, a.dt_dtype, (t0 + lane0) * a.dt_stride + h);
  };
  if (chunks) fetch(0);
  for (int64_t c = 0; c < chunks; ++c) {
    const int lane = sc_fresh(lane0), g = lane >> 4, i = lane & 15;
    const int64_t t0 = seg.t0 + 64 * (REV ? chunks - 1 - c : c);
    const int n = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    if (KEEP) {
      float* keep = w.chunk_states + ((ss_row_of(seg, 64) + c) * a.H * npb + blockIdx.y) * (NP * 64);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) keep[sc_kept_at(nt, wave, 4 * g + r, i)] = S[nt][r];
    }
    if (REV) {
      sign = -sign;
      pv.flip(sc_flip_bits(sign));
    }
    pk.put(tk, KS);
    pv.put(tv, VS);
    if (wave == 0) sc_decays(dec, nullptr, pdt, n, bias, A, a.softplus);
    lds_barrier();
    if (c + 1 < chunks) fetch(c + 1);
    const float end = REV ? -dec.end : dec.end;
    sum += dec.sum;
    sc_x8<T> v[2];
    sc_columns<T>(tv, VS, 16 * wave, lane, v);
    float wt[2][8];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if constexpr (REV) {
        sc_row_weights(dec.grow, kk, lane, wt[kk]);
      } else {
        float d[8];
        sc_row_weights(dec.left, kk, lane, wt[kk]);
        sc_row_weights(dec.delta, kk, lane, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) wt[kk][e] *= d[e];
      }
    }
    sc_update<T, NT, PARTS>(tk, KS, lane, v, wt, end, S);
    lds_barrier();
  }
  if (KEEP) return;
  float* local = (REV ? w.adjoints : a.slot_states) + ((int64_t)blockIdx.x * a.H + h) * a.N * a.P;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = 16 * nt + 4 * (lane0 >> 4) + r;
      if (n < a.N && p < a.P) local[(int64_t)n * a.P + p] = REV ? sign * S[nt][r] : S[nt][r];
    }
  if (!REV && threadIdx.x == 0 && pb == 0) a.slot_decay[(int64_t)blockIdx.x * a.H + h] = __builtin_amdgcn_exp2f(sum);
}

// Waves a SIMD that fit (element-by-element loads and fp16's scales take more registers; of all variants one, bf16 element by element
// at N = 64 with three parts, spills two).
template <typename T, int NP, bool VEC>
constexpr int sc_map_waves() { return !VEC ? (NP <= 64 && __is_same(T, __bf16) ? 3 : 2) : NP <= 32 ? 5 : NP <= 64 ? 4 : (__is_same(T, __bf16) ? 3 : 2); }

// PARTS: all of them where the states go to the caller or into gradients, two where they only go into outputs.
template <typename T, int NP, bool VEC, int PARTS>
__global__ void __launch_bounds__(SC_BLOCK, (sc_map_waves<T, NP, VEC>())) sc_map_kernel(lampa_ss_args a, SsGrad w) {
  __shared__ ScMapTiles<T, NP> tiles;
  sc_map<T, NP, false, false, VEC, PARTS>(a, w, tiles);
}
// Before the gradients: the states in front of the chunks (first half of the grid) and the local adjoints, which do not depend on
// each other, side by side: neither fills the chip by itself (60 000 tokens x 8 heads, N = 128: 62 and 120 us in turn).
template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(SC_BLOCK, (sc_map_waves<T, NP, VEC>())) sc_prepare_kernel(lampa_ss_args a, SsGrad w) {
  __shared__ ScMapTiles<T, NP> tiles;
  if (blockIdx.z == 0) sc_map<T, NP, false, true, VEC, ScParts<T>::n>(a, w, tiles);
  else sc_map<T, NP, true, false, VEC, ScParts<T>::n>(a, w, tiles);
}

// Outputs of a segment from the state it starts from.
template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(SC_BLOCK, 2) sc_out_kernel(lampa_ss_args a) {
  constexpr int NT = NP / 16, KK = NP / 32, KS = NP + 8, VS = 64 + 8, MS = 64 + 8;
  const SsSegment seg = ss_segment(a, blockIdx.x);
  if (!seg.live) return;
  const int npb = (a.P + 63) / 64, pb = blockIdx.y % npb, h = blockIdx.y / npb, grp = h / (a.H / a.G);
  const int lane0 = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = a.P - 64 * pb < 64 ? a.P - 64 * pb : 64;
  T* yb = (T*)a.y + (int64_t)h * a.P + 64 * pb;
  if (seg.outside) {
    for (int64_t e = threadIdx.x; e < (seg.t1 - seg.t0) * cols; e += SC_BLOCK) yb[(seg.t0 + e / cols) * a.y_stride + e % cols] = (T)0.0f;
    return;
  }
  __shared__ __align__(16) T tb[64 * KS], tc[64 * KS], tx[64 * VS], tm[64 * MS];
  __shared__ __align__(16) ScDecay dec;
  __shared__ float mback[__is_same(T, _Float16) ? 64 : 1];  // fp16: what the rows of the pair weights were scaled down by
  __shared__ int first_bad;
  const T* bb = (const T*)a.B + (int64_t)grp * a.N;
  const T* cb = (const T*)a.C + (int64_t)grp * a.N;
  const T* xb = (const T*)a.x + (int64_t)h * a.P + 64 * pb;
  const float A = a.A[h], D = a.D ? a.D[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  const bool single = (a.cu_seqlens ? a.n_tokens : a.seq_len) <= a.seg_tokens;
  const bool handed_on = single && a.ht;
  const int p = 64 * pb + 16 * wave + (lane0 & 15);

  f32x4 S[NT];
  const float* init = single ? a.h0 : a.slot_states;
  if (init) init += ((single ? (int64_t)seg.seq : (int64_t)blockIdx.x) * a.H + h) * a.N * a.P;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (init)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[nt][r] = sc_state_at(init, 16 * nt + 4 * (lane0 >> 4) + r, p, a.N, a.P);

  ScTile<T, NP> pB, pC;
  ScTile<T, 64> pX;
  float pdt = 0.0f;
  auto fetch = [&](int64_t t0) {
    const int n = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    pB.template fetch<VEC>(bb + t0 * a.B_stride, a.B_stride, n, a.N);
    pC.template fetch<VEC>(cb + t0 * a.C_stride, a.C_stride, n, a.N);
    pX.template fetch<VEC>(xb + t0 * a.x_stride, a.x_stride, n, cols);
    if (wave == 0 && lane0 < n) pdt = ss_load_dt<T>(a.dt, a.dt_dtype, (t0 + lane0) * a.dt_stride + h);
  };
  if (threadIdx.x == 0) first_bad = 64;
  if (seg.t0 < seg.t1) fetch(seg.t0);
  lds_barrier();
  for (int64_t t0 = seg.t0; t0 < seg.t1;) {
    const int lane = sc_fresh(lane0), g = lane >> 4, i = lane & 15;
    int n = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    pB.put(tb, KS);
    pC.put(tc, KS);
    pX.put(tx, VS);
    {
      const int bad = pX.first_bad();
      if (bad < 64) atomicMin(&first_bad, bad);
    }
    if (wave == 0) sc_decays(dec, nullptr, pdt, n, bias, A, a.softplus);
    lds_barrier();
    // An x that is not finite times a weight of zero would reach earlier tokens: such a token begins a chunk of its own.
    const int bad = first_bad;
    if (bad < n) {
      n = bad ? bad : 1;
      lds_barrier();
      for (int e = threadIdx.x; e < (64 - n) * KS; e += SC_BLOCK) tb[n * KS + e] = (T)0.0f;
      for (int e = threadIdx.x; e < (64 - n) * VS; e += SC_BLOCK) tx[n * VS + e] = (T)0.0f;
      if (wave == 0) sc_decays(dec, nullptr, pdt, n, bias, A, a.softplus);
      if (threadIdx.x == 0) first_bad = 64;
      lds_barrier();
    }
    if (t0 + n < seg.t1) fetch(t0 + n);

    // Pair weights of tokens t = 16 wave + i with s = 0 .. t, as the operand of the products over s.
    {
      const float gt = dec.gamma[16 * wave + i];
      sc_x8<T> q[KK];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) q[kk] = *reinterpret_cast<const sc_x8<T>*>(tc + (16 * wave + i) * KS + 32 * kk + 8 * g);
      f32x4 m[4];
      float big = 0.0f;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        m[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (st > wave) continue;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          m[st] = mfma16(*reinterpret_cast<const sc_x8<T>*>(tb + (16 * st + i) * KS + 32 * kk + 8 * g), q[kk], m[st]);
        const f32x4 gs = *reinterpret_cast<const f32x4*>(dec.gamma + 16 * st + 4 * g);
        const f32x4 ds = *reinterpret_cast<const f32x4*>(dec.delta + 16 * st + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = m[st][r] * ds[r] * __builtin_amdgcn_exp2f(gt - gs[r]);
          m[st][r] = st < wave || 4 * g + r <= i ? v : 0.0f;
          if (__is_same(T, _Float16)) big = fmaxf(big, fabsf(m[st][r]));
        }
      }
      if constexpr (__is_same(T, _Float16)) {
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        const float s = sc_scale_for<T>(big);
#pragma unroll
        for (int st = 0; st < 4; ++st) m[st] *= s;
        if (g == 0) mback[16 * wave + i] = sc_inverse(s);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        if (2 * kk <= wave)
          *reinterpret_cast<sc_x8<T>*>(tm + (16 * wave + i) * MS + 32 * kk + 8 * g) = acc2_to_op<T>(m[2 * kk], m[2 * kk + 1]);
    }
    lds_barrier();

    // y^T of this wave's 16 columns: lane = token 16 tt + i, registers = columns 4 g .. + 3
    f32x4 y[4];
    f32x4 sback;
    {
      float s = 1.0f;
      if constexpr (__is_same(T, _Float16)) {
        float big = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 4; ++r) big = sc_larger(big, S[nt][r]);
        s = sc_column_scale<T>(big, lane, sback);
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) y[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        sc_x8<T> st[2];
        sc_state_operand<T, 2>(S[2 * kk], S[2 * kk + 1], s, st);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const sc_x8<T> q = *reinterpret_cast<const sc_x8<T>*>(tc + (16 * tt + i) * KS + 32 * kk + 8 * g);
          y[tt] = sc_mfma_right(st, q, y[tt]);
        }
      }
    }
    sc_x8<T> v[2];
    sc_columns<T>(tx, VS, 16 * wave, lane, v);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const int t = 16 * tt + i;
      const float back = __is_same(T, _Float16) ? mback[t] : 1.0f;
      if constexpr (__is_same(T, _Float16)) y[tt] *= sback * (dec.grow[t] * sc_inverse(back));
      else y[tt] *= dec.grow[t];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        if (2 * kk <= tt) y[tt] = mfma16(v[kk], *reinterpret_cast<const sc_x8<T>*>(tm + t * MS + 32 * kk + 8 * g), y[tt]);
      if (t < n) {
        const sc_x4<T> xv = *reinterpret_cast<const sc_x4<T>*>(tx + t * VS + op_perm32_col(16 * wave + 4 * g));
        sc_x4<T> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float out = __is_same(T, _Float16) ? y[tt][r] * back : y[tt][r];
          o[r] = (T)__builtin_fmaf(D, (float)xv[r], out);
        }
        const int c = 16 * wave + 4 * g;
        T* dst = reinterpret_cast<T*>(reinterpret_cast<char*>(yb + (t0 + 16 * tt) * a.y_stride) + (unsigned)(i * (int)a.y_stride + c) * (unsigned)sizeof(T));
        if constexpr (VEC) {
          if (c < cols) *reinterpret_cast<sc_x4<T>*>(dst) = o;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c + r < cols) dst[r] = o[r];
        }
      }
    }
    // the state behind the chunk
    {
      float wt[2][8];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float d[8];
        sc_row_weights(dec.left, kk, lane, wt[kk]);
        sc_row_weights(dec.delta, kk, lane, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) wt[kk][e] *= d[e];
      }
      if (handed_on) sc_update<T, NT, ScParts<T>::n>(tb, KS, lane, v, wt, dec.end, S);
      else sc_update<T, NT, 2>(tb, KS, lane, v, wt, dec.end, S);
    }
    t0 += n;
    lds_barrier();
  }
  if (single && a.ht) {
    float* out = a.ht + ((int64_t)seg.seq * a.H + h) * a.N * a.P;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = 16 * nt + 4 * (lane0 >> 4) + r;
        if (n < a.N && p < a.P) out[(int64_t)n * a.P + p] = S[nt][r];
      }
  }
}

template <typename T, bool VEC>
static int sc_maps_launch(const lampa_ss_args& a, const SsGrad* grad, hipStream_t s) {
  dim3 grid = sc_grid(a);
  if (grad) grid.z = ss_single(&a) ? 1 : 2;  // a sequence of one segment starts from dht: no local adjoints
  LAMPA_PROF(s, "start");
#define SC_GO(NP)                                                                                           \
  if (grad) hipLaunchKernelGGL((sc_prepare_kernel<T, NP, VEC>), grid, dim3(SC_BLOCK), 0, s, a, *grad);      \
  else if (a.ht || a.for_grad) hipLaunchKernelGGL((sc_map_kernel<T, NP, VEC, ScParts<T>::n>), grid, dim3(SC_BLOCK), 0, s, a, SsGrad{}); \
  else hipLaunchKernelGGL((sc_map_kernel<T, NP, VEC, 2>), grid, dim3(SC_BLOCK), 0, s, a, SsGrad{})
  if (a.N <= 32) { SC_GO(32); } else if (a.N <= 64) { SC_GO(64); } else { SC_GO(128); }
#undef SC_GO
  LAMPA_PROF(s, grad ? "sc_prepare_kernel" : "sc_map_kernel");
  return lampa_launch_status();
}
// The segments' local states, or, with `grad`, what the gradients start from.
int ss_chunk_maps(const lampa_ss_args& a, const SsGrad* grad, hipStream_t s) {
  if (a.dtype == GDR_BF16) return sc_vectors(a) ? sc_maps_launch<__bf16, true>(a, grad, s) : sc_maps_launch<__bf16, false>(a, grad, s);
  return sc_vectors(a) ? sc_maps_launch<_Float16, true>(a, grad, s) : sc_maps_launch<_Float16, false>(a, grad, s);
}

template <typename T, bool VEC>
static int sc_out_launch(const lampa_ss_args& a, hipStream_t s) {
  LAMPA_PROF(s, "start");
  if (a.N <= 32) hipLaunchKernelGGL((sc_out_kernel<T, 32, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a);
  else if (a.N <= 64) hipLaunchKernelGGL((sc_out_kernel<T, 64, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a);
  else hipLaunchKernelGGL((sc_out_kernel<T, 128, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a);
  LAMPA_PROF(s, "sc_out_kernel");
  return lampa_launch_status();
}
int ss_chunk_out(const lampa_ss_args& a, hipStream_t s) {
  if (a.dtype == GDR_BF16) return sc_vectors(a) ? sc_out_launch<__bf16, true>(a, s) : sc_out_launch<__bf16, false>(a, s);
  return sc_vectors(a) ? sc_out_launch<_Float16, true>(a, s) : sc_out_launch<_Float16, false>(a, s);
}
