// Chunked gradients of the state-space scan on the matrix cores (see ss_chunk.h for the forward's form and its roundings).
//
// From the end of a segment, with R the adjoint behind a chunk, S the state in front of it, L[t, s] = e^{gamma_t - gamma_s} for
// s <= t and G[t, s] = C_t . B_s, H[t, s] = dy_t . x_s:
//   dx_s = delta_s ( sum_t L G [t, s] dy_t + e^{gamma_end - gamma_s} R^T B_s ) + D dy_s
//   dB_s = delta_s ( sum_t L H [t, s] C_t  + e^{gamma_end - gamma_s} R x_s )
//   dC_t = sum_s delta_s L H [t, s] B_s + e^{gamma_t} S dy_t
//   R   <- e^{gamma_end} R + sum_t e^{gamma_t} C_t dy_t^T
// The decay's gradient dg_t = <R_t, e^{g_t} S_{t-1}> is everything that passes from before token t to t or later:
//   pairs s < t <= i of tokens of the chunk:  a prefix sum of the column sums minus the row sums of delta_s L G H (strictly below
//     the diagonal), formed in fp32 from G and H as they leave the matrix cores;
//   from S to tokens of the chunk, e^{gamma_i} C_i . (S dy_i) over i >= t;  from tokens of the chunk to R, delta_s e^{gamma_end - gamma_s}
//     x_s . (R^T B_s) over s < t;  and from S to R, e^{gamma_end} <R, S>.
// All four are sums of what really passes. The shorter form dg_t = dg_{t+1} + read_t - written_t over a whole segment subtracts
// much larger numbers from each other, and its errors stay in every earlier token: dA came out wrong by 2e-5 to 5e-5.
//
// S in front of every chunk is recomputed from the segments' initial states by a forward walk and kept (fp32). R is held twice,
// as [n, p] with 16 of the columns p a wave and as [p, n] with a share of the columns n, because dx reads it out over n and dB
// over p; summing it up twice costs fewer cycles than passing it through LDS.
#include "ss_chunk.h"

template <typename T, int NP, bool VEC>
__global__ void __launch_bounds__(SC_BLOCK, 2) sc_grad_kernel(lampa_ss_args a, SsGrad w) {
  constexpr int NT = NP / 16, KK = NP / 32, KS = NP + 8, VS = 64 + 8, MS = 64 + 8;
  constexpr int NW = NP == 128 ? 2 : 1;  // tiles of 16 columns n a wave has of dB, dC and the transposed R
  constexpr bool F16 = __is_same(T, _Float16);
  typedef sc_x8<T> x8;
  typedef sc_x4<T> x4;
  constexpr int PARTS = ScParts<T>::n;
  const SsSegment seg = ss_segment(a, blockIdx.x);
  if (!seg.live) return;
  const int npb = (a.P + 63) / 64, pb = blockIdx.y % npb, h = blockIdx.y / npb, grp = h / (a.H / a.G);
  const int lane0 = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = a.P - 64 * pb < 64 ? a.P - 64 * pb : 64;
  const int64_t row_p = (int64_t)a.H * a.P, parts = (int64_t)a.H * npb;
  T* dxb = (T*)a.dx + (int64_t)h * a.P + 64 * pb;
  if (seg.outside) {
    const int64_t n = seg.t1 - seg.t0;
    for (int64_t e = threadIdx.x; e < n * cols; e += SC_BLOCK) dxb[(seg.t0 + e / cols) * row_p + e % cols] = (T)0.0f;
    for (int64_t e = threadIdx.x; e < n * a.N; e += SC_BLOCK) {
      const int64_t at = ((seg.t0 + e / a.N) * parts + blockIdx.y) * a.N + e % a.N;
      w.dB_part[at] = w.dC_part[at] = 0.0f;
    }
    if (threadIdx.x == 0) w.dD_part[(int64_t)blockIdx.x * parts + blockIdx.y] = 0.0f;
    return;
  }
  __shared__ __align__(16) T tb[64 * KS], tc[64 * KS], tx[64 * VS], ty[64 * VS], m1[64 * MS], m2[64 * MS];
  __shared__ __align__(16) ScDecay dec;
  __shared__ __align__(16) float row_part[4][64], col_sum[64], diag[64], left_part[4][64], read_part[4][64], dot_part[4];
  __shared__ __align__(16) float rest2[64];
  __shared__ float back1[64], back2[64];  // fp16: what the rows of m1 and m2 were scaled down by
  const T* bb = (const T*)a.B + (int64_t)grp * a.N;
  const T* cb = (const T*)a.C + (int64_t)grp * a.N;
  const T* xb = (const T*)a.x + (int64_t)h * a.P + 64 * pb;
  const T* yb = (const T*)a.dy + (int64_t)h * a.P + 64 * pb;
  const float A = a.A[h], D = a.D ? a.D[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;
  const bool single = (a.cu_seqlens ? a.n_tokens : a.seq_len) <= a.seg_tokens;
  const int nt0 = NW * wave;        // this wave's tiles of columns n
  const bool has_n = nt0 < NT;      // (a state of 32 has two of them only)

  f32x4 R[NT], RT[4][NW];
  {
  const int lane = lane0, g = lane >> 4, i = lane & 15, p = 64 * pb + 16 * wave + i;
  const float* init = single ? a.dht : w.adjoints;
  if (init) init += ((single ? (int64_t)seg.seq : (int64_t)blockIdx.x) * a.H + h) * a.N * a.P;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) R[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int pt = 0; pt < 4; ++pt)
#pragma unroll
    for (int j = 0; j < NW; ++j) RT[pt][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (init) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) R[nt][r] = sc_state_at(init, 16 * nt + 4 * g + r, p, a.N, a.P);
#pragma unroll
    for (int pt = 0; pt < 4; ++pt)
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) RT[pt][j][r] = sc_state_at(init, 16 * (nt0 + j) + i, 64 * pb + 16 * pt + 4 * g + r, a.N, a.P);
  }
  }
  ScTile<T, NP> pB, pC;
  ScTile<T, 64> pX, pY;
  float pdt = 0.0f, dD = 0.0f, sign = -1.0f;  // sign: of R, of dy in this chunk, and of all that is made from them
  const int64_t chunks = (seg.t1 - seg.t0 + 63) / 64;
  auto fetch = [&](int64_t c) {
    const int64_t t0 = seg.t0 + 64 * c;
    const int n = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    pB.template fetch<VEC>(bb + t0 * a.B_stride, a.B_stride, n, a.N);
    pC.template fetch<VEC>(cb + t0 * a.C_stride, a.C_stride, n, a.N);
    pX.template fetch<VEC>(xb + t0 * a.x_stride, a.x_stride, n, cols);
    pY.template fetch<VEC>(yb + t0 * row_p, row_p, n, cols);
    if (wave == 0 && lane0 < n) pdt = ss_load_dt<T>(a.dt, a.dt_dtype, (t0 + lane0) * a.dt_stride + h);
  };
  // A wide state leaves no registers for the next chunk's tiles: they are fetched when they are due, and the other workgroup of
  // the CU works meanwhile.
  constexpr bool AHEAD = NP <= 64;
  if (AHEAD && chunks) fetch(chunks - 1);
  for (int64_t c = chunks - 1; c >= 0; --c) {
    const int lane = sc_fresh(lane0), g = lane >> 4, i = lane & 15;
    const int64_t t0 = seg.t0 + 64 * c;
    const int n_tok = (int)(seg.t1 - t0 < 64 ? seg.t1 - t0 : 64);
    if (!AHEAD) fetch(c);
    sign = -sign;
    pY.flip(sc_flip_bits(sign));
    pB.put(tb, KS);
    pC.put(tc, KS);
    pX.put(tx, VS);
    pY.put(ty, VS);
    if (wave == 0) sc_decays(dec, rest2, pdt, n_tok, bias, A, a.softplus);
    lds_barrier();
    if (AHEAD && c > 0) fetch(c - 1);
    // Pair weights of tokens s = 16 wave + i with t = s ..: rows of m1 (L G) and m2 (delta_s L H), and the sums of their product.
    {
      const int s = 16 * wave + i;
      // The exponents' rounding (2^rest) matters to the sums only: theirs of t goes in element by element, that of s at the end.
      const float gs = dec.gamma[s], ds = dec.delta[s], rest_s = 1.0f / rest2[s], ds_rest = ds * rest_s;
      x8 qb[KK], qx[2];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qb[kk] = *reinterpret_cast<const x8*>(tb + s * KS + 32 * kk + 8 * g);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) qx[kk] = *reinterpret_cast<const x8*>(tx + s * VS + 32 * kk + 8 * g);
      f32x4 lg[4], lh[4];
      float sum = 0.0f, own = 0.0f, big1 = 0.0f, big2 = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        sc_fence();
        lg[tt] = lh[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        f32x4 rows = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (tt >= wave) {
          f32x4 G = rows, Hm = rows;
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) G = mfma16(*reinterpret_cast<const x8*>(tc + (16 * tt + i) * KS + 32 * kk + 8 * g), qb[kk], G);
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) Hm = mfma16(*reinterpret_cast<const x8*>(ty + (16 * tt + i) * VS + 32 * kk + 8 * g), qx[kk], Hm);
          const f32x4 gt = *reinterpret_cast<const f32x4*>(dec.gamma + 16 * tt + 4 * g);
          const f32x4 rest = *reinterpret_cast<const f32x4*>(rest2 + 16 * tt + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = 16 * tt + 4 * g + r;
            const float l = __builtin_amdgcn_exp2f(gt[r] - gs);
            const bool on = tt > wave || t >= s;
            const float vg = on ? l * G[r] : 0.0f, both = on ? vg * Hm[r] * rest[r] : 0.0f;
            lg[tt][r] = vg;
            lh[tt][r] = on ? ds * l * Hm[r] : 0.0f;
            const bool self = tt == wave && t == s;
            if (self) own = both; else sum += both;
            rows[r] = sc_row16_sum(self ? 0.0f : ds_rest * both);
            if (F16) { big1 = fmaxf(big1, fabsf(vg)); big2 = fmaxf(big2, fabsf(lh[tt][r])); }
          }
        }
        if (i == 0) *reinterpret_cast<f32x4*>(&row_part[wave][16 * tt + 4 * g]) = rows;
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      own += __shfl_xor(own, 16);  // one lane of the four has it
      own += __shfl_xor(own, 32);
      if (g == 0) { col_sum[s] = sum * rest_s; diag[s] = own * rest_s; }
      if constexpr (F16) {
        big1 = fmaxf(big1, __shfl_xor(big1, 16));
        big1 = fmaxf(big1, __shfl_xor(big1, 32));
        big2 = fmaxf(big2, __shfl_xor(big2, 16));
        big2 = fmaxf(big2, __shfl_xor(big2, 32));
        // rows of m2 are summed over s as well (dC), so its scale is the wave's: one for 16 rows
        const float s1 = sc_scale_for<T>(big1), s2 = sc_scale_for<T>(sc_wave_max(big2));
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) { lg[tt] *= s1; lh[tt] *= s2; }
        if (g == 0) { back1[s] = sc_inverse(s1); back2[s] = sc_inverse(s2); }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        if (2 * kk + 1 >= wave) {
          *reinterpret_cast<x8*>(m1 + s * MS + 32 * kk + 8 * g) = acc2_to_op<T>(lg[2 * kk], lg[2 * kk + 1]);
          *reinterpret_cast<x8*>(m2 + s * MS + 32 * kk + 8 * g) = acc2_to_op<T>(lh[2 * kk], lh[2 * kk + 1]);
        }
    }
    lds_barrier();

    sc_fence();
    // S in front of the chunk: columns p of this wave's rows n, as the lane's share of an operand, a tile of rows at a time
    f32x4 S[4];
    const f32x4* kept = reinterpret_cast<const f32x4*>(w.chunk_states + ((ss_row_of(seg, 64) + c) * parts + blockIdx.y) * (NP * 64));
    if (has_n) {
#pragma unroll
      for (int q = 0; q < 4; ++q) S[q] = kept[(nt0 * 4 + q) * 64 + lane];
    }

    const float end = dec.end, D_sign = sign * D;
    float dD_chunk = 0.0f;
    // dx of this wave's 16 columns: lane = token 16 st + i, registers = columns 4 g .. + 3
    {
      x8 vy[2];
      sc_columns<T>(ty, VS, 16 * wave, lane, vy);
      float sc = 1.0f;
      f32x4 sback;
      if constexpr (F16) {
        float big = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 4; ++r) big = sc_larger(big, R[nt][r]);
        sc = sc_column_scale<T>(big, lane, sback);
      }
      f32x4 acc[4];
#pragma unroll
      for (int st = 0; st < 4; ++st) acc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        sc_fence();
        x8 st8[PARTS];
        sc_state_operand<T, PARTS>(R[2 * kk], R[2 * kk + 1], sc, st8);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const x8 q = *reinterpret_cast<const x8*>(tb + (16 * st + i) * KS + 32 * kk + 8 * g);
          acc[st] = sc_mfma_right(st8, q, acc[st]);
        }
      }
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        sc_fence();
        const int s = 16 * st + i;
        if constexpr (F16) acc[st] *= sback * dec.left[s];
        else acc[st] *= dec.left[s];
        const int at = s * VS + op_perm32_col(16 * wave + 4 * g);
        const x4 xv = *reinterpret_cast<const x4*>(tx + at), dyv = *reinterpret_cast<const x4*>(ty + at);
        float dot = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          dot = __builtin_fmaf((float)xv[r], acc[st][r], dot);
          dD_chunk = __builtin_fmaf((float)xv[r], (float)dyv[r], dD_chunk);
        }
        dot += __shfl_xor(dot, 16);
        dot += __shfl_xor(dot, 32);
        if (g == 0) left_part[wave][s] = dot;
        f32x4 near = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!F16) near = acc[st];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          if (2 * kk + 1 >= st) near = mfma16(vy[kk], *reinterpret_cast<const x8*>(m1 + s * MS + 32 * kk + 8 * g), near);
        if (F16) near = near * back1[s] + acc[st];
        if (s < n_tok) {
          const float ds = sign * dec.delta[s];
          x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = (T)__builtin_fmaf(ds, near[r], D_sign * (float)dyv[r]);
          const int c0 = 16 * wave + 4 * g;
          T* dst = reinterpret_cast<T*>(reinterpret_cast<char*>(dxb + (t0 + 16 * st) * row_p) + (unsigned)(i * (int)row_p + c0) * (unsigned)sizeof(T));
          if constexpr (VEC) {
            if (c0 < cols) *reinterpret_cast<x4*>(dst) = o;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c0 + r < cols) dst[r] = o[r];
          }
        }
      }
    }
    dD = __builtin_fmaf(sign, dD_chunk, dD);
    sc_fence();
    // dB and dC of this wave's columns n: lane = token, registers = columns 4 g .. + 3 of a tile
    float dot = 0.0f;
    if (has_n) {
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        sc_fence();
        float s1 = 1.0f, s2 = 1.0f;
        f32x4 b1, b2;
        if constexpr (F16) {
          float big1 = 0.0f, big2 = 0.0f;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              big1 = sc_larger(big1, RT[q][j][r]);
              big2 = sc_larger(big2, S[q][r]);
            }
          s1 = sc_column_scale<T>(big1, lane, b1);
          s2 = sc_column_scale<T>(big2, lane, b2);
        }
        f32x4 db[4], dc[4];
#pragma unroll
        for (int st = 0; st < 4; ++st) db[st] = dc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          sc_fence();
          x8 adj[2], state[PARTS];
          sc_state_operand<T, 2>(RT[2 * kk][j], RT[2 * kk + 1][j], s1, adj);
#pragma unroll
          for (int st = 0; st < 4; ++st) {
            const x8 q = *reinterpret_cast<const x8*>(tx + (16 * st + i) * VS + 32 * kk + 8 * g);
            db[st] = sc_mfma_right(adj, q, db[st]);
          }
          sc_fence();
          sc_state_operand<T, PARTS>(S[2 * kk], S[2 * kk + 1], s2, state);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            const x8 q = *reinterpret_cast<const x8*>(ty + (16 * tt + i) * VS + 32 * kk + 8 * g);
            dc[tt] = sc_mfma_right(state, q, dc[tt]);
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int r = 0; r < 4; ++r) dot = __builtin_fmaf(RT[q][j][r], S[q][r], dot);
        if (j + 1 < NW) {
#pragma unroll
          for (int q = 0; q < 4; ++q) S[q] = kept[((nt0 + j + 1) * 4 + q) * 64 + lane];
        }
        sc_fence();
        x8 vb[2], vc[2];
        sc_columns<T>(tb, KS, 16 * (nt0 + j), lane, vb);
        sc_columns<T>(tc, KS, 16 * (nt0 + j), lane, vc);
        const int c0 = 16 * (nt0 + j) + 4 * g;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          sc_fence();
          const int s = 16 * st + i;
          db[st] *= dec.left[s] * dec.delta[s];
          if constexpr (F16) db[st] *= b1;
          if constexpr (F16) {
            f32x4 near = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
              if (2 * kk + 1 >= st) near = mfma16(vc[kk], *reinterpret_cast<const x8*>(m2 + s * MS + 32 * kk + 8 * g), near);
            db[st] += near * back2[s];
          } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
              if (2 * kk + 1 >= st) db[st] = mfma16(vc[kk], *reinterpret_cast<const x8*>(m2 + s * MS + 32 * kk + 8 * g), db[st]);
          }
          dc[st] *= dec.grow[s];
          if constexpr (F16) dc[st] *= b2;
          const x4 cv = *reinterpret_cast<const x4*>(tc + s * KS + op_perm32_col(c0));
          float read = 0.0f;
#pragma unroll
          for (int r = 0; r < 4; ++r) read = __builtin_fmaf((float)cv[r], dc[st][r], read);
          read += __shfl_xor(read, 16);
          read += __shfl_xor(read, 32);
          if (g == 0) read_part[wave][s] = j ? read_part[wave][s] + read : read;
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            if (2 * kk <= st) {
              x8 q = op_ld_tr16<T, true>(m2, MS, 16 * st, 32 * kk, lane);
              if constexpr (F16) {
                // the rows of this product were scaled 16 at a time: undo each half on its own
                x8 q0 = q, q1 = q;
#pragma unroll
                for (int e = 0; e < 4; ++e) { q0[4 + e] = (T)0.0f; q1[e] = (T)0.0f; }
                const f32x4 zero = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                dc[st] += mfma16(vb[kk], q0, zero) * back2[32 * kk] + mfma16(vb[kk], q1, zero) * back2[32 * kk + 16];
              } else {
                dc[st] = mfma16(vb[kk], q, dc[st]);
              }
            }
          db[st] *= sign;
          dc[st] *= sign;
          if (s < n_tok) {
            const int64_t row = ((t0 + 16 * st) * parts + blockIdx.y) * a.N;
            const unsigned at = (unsigned)(i * (int)(parts * a.N) + c0) * 4u;
            float* pdb = reinterpret_cast<float*>(reinterpret_cast<char*>(w.dB_part + row) + at);
            float* pdc = reinterpret_cast<float*>(reinterpret_cast<char*>(w.dC_part + row) + at);
            if constexpr (VEC) {
              if (c0 < a.N) {
                *reinterpret_cast<f32x4*>(pdb) = db[st];
                *reinterpret_cast<f32x4*>(pdc) = dc[st];
              }
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (c0 + r < a.N) {
                  pdb[r] = db[st][r];
                  pdc[r] = dc[st][r];
                }
            }
          }
        }
      }
    } else {
      for (int s = lane; s < 64; s += 64) read_part[wave][s] = 0.0f;
    }
    dot = ss_wave_sum(dot);
    if (lane == 0) dot_part[wave] = dot;

    sc_fence();
    // R in front of the chunk, both ways round, with the sign of the next chunk's dy.
    {
      float wt[2][8];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        sc_row_weights(dec.grow, kk, lane, wt[kk]);
#pragma unroll
        for (int e = 0; e < 8; ++e) wt[kk][e] = -wt[kk][e];
      }
      auto add = [&](f32x4& acc, const x8 (&left)[2], const x8 (&right)[2][PARTS], float back) {
        if constexpr (F16) {
          f32x4 d = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) d = sc_mfma_left(left[kk], right[kk], d);
          acc = d * back - acc * end;
        } else {
          acc *= -end;
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) acc = sc_mfma_left(left[kk], right[kk], acc);
        }
      };
      x8 v[2], vw[2][PARTS], left[2];
      sc_columns<T>(ty, VS, 16 * wave, lane, v);
      float back = sc_weighted<T, PARTS>(v, wt, vw);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sc_columns<T>(tc, KS, 16 * nt, lane, left);
        add(R[nt], left, vw, back);
        sc_fence();
      }
      if (has_n) {
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          sc_columns<T>(tc, KS, 16 * (nt0 + j), lane, v);
          back = sc_weighted<T, PARTS>(v, wt, vw);
#pragma unroll
          for (int pt = 0; pt < 4; ++pt) {
            sc_columns<T>(ty, VS, 16 * pt, lane, left);
            add(RT[pt][j], left, vw, back);
            sc_fence();
          }
          sc_fence();
        }
      }
    }
    lds_barrier();
    if (wave == 0) {  // lane = token: what passes across it
      const float d = dec.delta[lane];
      const float col = col_sum[lane];
      const float r0 = row_part[0][lane], r1 = row_part[1][lane], r2 = row_part[2][lane], r3 = row_part[3][lane];
      const float left = (left_part[0][lane] + left_part[1][lane]) + (left_part[2][lane] + left_part[3][lane]);
      const float read = (read_part[0][lane] + read_part[1][lane]) + (read_part[2][lane] + read_part[3][lane]);
      const float all = end * ((dot_part[0] + dot_part[1]) + (dot_part[2] + dot_part[3]));
      // Pairs across the first token of each 16: of the tiles of pairs, those of later tokens with earlier ones ...
      const int tile = lane >> 4;
      const float from0 = sc_row16_sum(r0), from1 = sc_row16_sum(r1), from2 = sc_row16_sum(r2);
      float across1 = tile >= 1 ? from0 : 0.0f, across2 = tile >= 2 ? from0 + from1 : 0.0f,
            across3 = tile >= 3 ? (from0 + from1) + from2 : 0.0f;
#pragma unroll
      for (int off = 16; off < 64; off <<= 1) {
        across1 += __shfl_xor(across1, off);
        across2 += __shfl_xor(across2, off);
        across3 += __shfl_xor(across3, off);
      }
      // ... and from there on a prefix sum of column minus row sums. (Over all 64 tokens its rounding errors, which stay in every
      // later token, are 3e-6 of dA and d dt_bias.)
      float pairs = d * col - ((r0 + r1) + (r2 + r3));
      pairs += dpp_f32<GDR_DPP_ROW_SHR(1), 0xF>(0.0f, pairs);
      pairs += dpp_f32<GDR_DPP_ROW_SHR(2), 0xF>(0.0f, pairs);
      pairs += dpp_f32<GDR_DPP_ROW_SHR(4), 0xF>(0.0f, pairs);
      pairs += dpp_f32<GDR_DPP_ROW_SHR(8), 0xF>(0.0f, pairs);
      pairs = dpp_f32<GDR_DPP_ROW_SHR(1), 0xF>(0.0f, pairs);
      pairs += tile == 0 ? 0.0f : tile == 1 ? across1 : tile == 2 ? across2 : across3;
      float before = d * left;  // summed over the tokens before this one ...
      float later = read;       // ... and this over this one and those behind it
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const float up = __shfl_up(before, off), down = __shfl_down(later, off);
        if (lane >= off) before += up;
        if (lane + off < 64) later += down;
      }
      before = __shfl_up(before, 1);
      if (lane == 0) before = 0.0f;
      if (lane < n_tok) {
        const int64_t at = (t0 + lane) * parts + blockIdx.y;
        w.dg[at] = sign * ((pairs + before) + (later + all));
        w.reach[at] = sign * (col + diag[lane] + left);
      }
    }
  }
  const int lane = lane0, g = lane >> 4, i = lane & 15, p = 64 * pb + 16 * wave + i;
  // shares of dD: every wave has its own columns
  dD = ss_wave_sum(dD);
  lds_barrier();
  if (lane == 0) dot_part[wave] = dD;
  lds_barrier();
  if (threadIdx.x == 0) w.dD_part[(int64_t)blockIdx.x * parts + blockIdx.y] = (dot_part[0] + dot_part[1]) + (dot_part[2] + dot_part[3]);
  if (single && a.dh0) {
    float* out = a.dh0 + ((int64_t)seg.seq * a.H + h) * a.N * a.P;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = 16 * nt + 4 * g + r;
        if (n < a.N && p < a.P) out[(int64_t)n * a.P + p] = -sign * R[nt][r];
      }
  }
}

template <typename T, bool VEC>
static int sc_grad_launch(const lampa_ss_args& a, const SsGrad& w, hipStream_t s) {
  LAMPA_PROF(s, "start");
  if (a.N <= 32) hipLaunchKernelGGL((sc_grad_kernel<T, 32, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a, w);
  else if (a.N <= 64) hipLaunchKernelGGL((sc_grad_kernel<T, 64, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a, w);
  else hipLaunchKernelGGL((sc_grad_kernel<T, 128, VEC>), sc_grid(a), dim3(SC_BLOCK), 0, s, a, w);
  LAMPA_PROF(s, "sc_grad_kernel");
  return lampa_launch_status();
}
int ss_chunk_grad(const lampa_ss_args& a, const SsGrad& w, hipStream_t s) {
  if (a.dtype == GDR_BF16) return sc_vectors(a) ? sc_grad_launch<__bf16, true>(a, w, s) : sc_grad_launch<__bf16, false>(a, w, s);
  return sc_vectors(a) ? sc_grad_launch<_Float16, true>(a, w, s) : sc_grad_launch<_Float16, false>(a, w, s);
}
