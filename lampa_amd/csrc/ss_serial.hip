// Token-serial walks of the state-space scan on gfx950, fp32 throughout: the form for fp32 tensors.
//
// All four passes of the operator (y, dC, dx, dB) are the same walk: a state of `rows` x 64 whose column l belongs to lane l
// and whose rows are that lane's registers,
//   S[r] = a_t S[r] + U_t[r] v_t[l],   out_t[l] = sum_r Q_t[r] S[r],
// with (rows, lane; U, v, Q) = (n, p; B, delta x, C) for y, (p, n; x, delta B, dy) for dC, and from the end of the segment
// (n, p; C, dy, B) for dx, (p, n; dy, C, x) for dB. U_t and Q_t are the same for every lane: they are staged in LDS a few
// tokens at a time and read as broadcasts, so a token costs 3 vector instructions a row and no reduction across lanes.
// One wave a workgroup; nothing is shared between waves, so no barrier waits for another wave.
//
// Bound by the latency of a token (0.4 to 0.6 us with one wave a SIMD: 3 instructions a row, the staged rows' reads, and the
// stores), so segments are short. Measured, fp32: 6 007 packed tokens x 4 heads, P = N = 32, in segments of 64: y 26, dC 40, dx 39, dB
// 25 us, local states and adjoints 18 each; 77 tokens x 2 sequences whole 28 us; forward of 20 000 x 8 x 64 at N = 64 / 128 in all 235 /
// 404 us.
//
// Errors: a token's part of a later state is a product of as many fp32 decays as lie between them, each rounded, where exponents
// summed up in 64 bits would be rounded once: y is off by 3e-7 at 77 tokens of slow decay against 6e-8, and by 4e-8 either way where
// heads forget within a few tokens.
#include "ss_kernels.h"

#define SS_TILE 8  // tokens staged at once; SS_DOT is a multiple of it

// Waves a SIMD that fit: the adjoints' walk holds the state and one that was kept.
template <int ROWS, int KIND, bool MAP>
constexpr int ss_serial_waves() { return ROWS == 128 && KIND == SS_DX && !MAP ? 1 : 2; }

// ROWS: rows of the state a wave holds. LG: where the lanes' dimension has at most 64 / LG columns, the wave's LG parts hold
// ROWS / LG rows each of the same columns and their read-outs are added up.
template <int ROWS, int LG, int KIND, bool MAP>
__global__ void __launch_bounds__(64, (ss_serial_waves<ROWS, KIND, MAP>())) ss_serial_kernel(lampa_ss_args a, SsGrad w) {
  constexpr bool REV = KIND == SS_DX || KIND == SS_DB;  // from the end of the segment
  constexpr bool LANE_P = KIND == SS_Y || KIND == SS_DX;
  // Walks that also leave dots of their read-outs with a second lane vector, C or x: these read out what the state holds without the
  // token's own part, U_t (Q_t . U_t for the rows), which goes to the output alone.
  constexpr bool SUMS = !MAP && (KIND == SS_DC || KIND == SS_DX);
  constexpr int PIECES = ROWS * SS_TILE / 64, RL = ROWS / LG, COLS = 64 / LG;
  const SsSegment seg = ss_segment(a, blockIdx.x);
  if (!seg.live) return;
  const int lane = threadIdx.x;
  const int npb = (a.P + 63) / 64, nnb = (a.N + 63) / 64;
  int rest = blockIdx.y, lane_block, row_block = 0;
  if constexpr (LANE_P) {
    lane_block = rest % npb;
    rest /= npb;
  } else {
    lane_block = rest % nnb;
    rest /= nnb;
    row_block = rest % npb;
    rest /= npb;
  }
  const int h = rest, grp = h / (a.H / a.G);
  const int pb = LANE_P ? lane_block : row_block;
  const int width = LANE_P ? a.P : a.N;  // of the lanes' dimension
  const int l = lane_block * 64 + lane % COLS, row0 = lane / COLS * RL;
  const bool lane_on = l < width;
  const int r0 = row_block * 64, rn = (LANE_P ? a.N : a.P) - r0;  // rows r0 .. of the state; rn of them exist
  const int64_t per_h = (int64_t)a.N * a.P, hp = (int64_t)a.H * a.P, parts = (int64_t)a.H * npb;
  // element (row r of this lane's) of a state [N, P]
  auto at = [&](int r) { return LANE_P ? (int64_t)(r0 + row0 + r) * a.P + l : (int64_t)l * a.P + r0 + row0 + r; };
  auto has = [&](int r) { return lane_on && row0 + r < rn; };

  // What a token leaves behind, column l: a row of y, dx, or of this head's part of dC or dB.
  float* out_rows;
  int64_t out_stride;
  if constexpr (KIND == SS_Y) { out_rows = (float*)a.y + (int64_t)h * a.P; out_stride = a.y_stride; }
  else if constexpr (KIND == SS_DX) { out_rows = (float*)a.dx + (int64_t)h * a.P; out_stride = hp; }
  else { out_rows = (KIND == SS_DC ? w.dC_part : w.dB_part) + ((int64_t)h * npb + pb) * a.N; out_stride = parts * a.N; }
  const bool writes = lane < COLS && lane_on;
  if (seg.outside) {
    if (!MAP && writes)
      for (int64_t t = seg.t0; t < seg.t1; ++t) out_rows[t * out_stride + l] = 0.0f;
    if (!MAP && KIND == SS_DX && lane == 0) w.dD_part[((int64_t)blockIdx.x * a.H + h) * npb + pb] = 0.0f;
    return;
  }

  const bool single = !MAP && (a.cu_seqlens ? a.n_tokens : a.seq_len) <= a.seg_tokens;
  float S[RL];
#pragma unroll
  for (int r = 0; r < RL; ++r) S[r] = 0.0f;
  if (!MAP) {
    const float* init = single ? (REV ? a.dht : a.h0) : (REV ? w.adjoints : a.slot_states);
    if (init) {
      init += ((single ? (int64_t)seg.seq : (int64_t)blockIdx.x) * a.H + h) * per_h;
#pragma unroll
      for (int r = 0; r < RL; ++r)
        if (has(r)) S[r] = init[at(r)];
    }
  }

  const float* x = (const float*)a.x + (int64_t)h * a.P;
  const float* dy = (const float*)a.dy + (int64_t)h * a.P;
  const float* Bm = (const float*)a.B + (int64_t)grp * a.N;
  const float* Cm = (const float*)a.C + (int64_t)grp * a.N;
  const float *U, *Q, *V;
  int64_t us, qs, vs;
  if constexpr (KIND == SS_Y) { U = Bm; us = a.B_stride; Q = Cm; qs = a.C_stride; V = x; vs = a.x_stride; }
  else if constexpr (KIND == SS_DC) { U = x; us = a.x_stride; Q = dy; qs = hp; V = Bm; vs = a.B_stride; }
  else if constexpr (KIND == SS_DX) { U = Cm; us = a.C_stride; Q = Bm; qs = a.B_stride; V = dy; vs = hp; }
  else { U = dy; us = hp; Q = x; qs = a.x_stride; V = Cm; vs = a.C_stride; }
  const float* E = KIND == SS_DC ? Cm : x;
  const int64_t es = KIND == SS_DC ? a.C_stride : a.x_stride;
  const float A = a.A[h], D = a.D ? a.D[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;

  __shared__ __align__(16) float lu[SS_TILE][ROWS], lq[MAP ? 1 : SS_TILE][ROWS], lv[SS_TILE][64], le[SUMS ? SS_TILE : 1][64];
  __shared__ __align__(16) float ldelta[SS_TILE], ldecay[SS_TILE];
  float pu[PIECES], pq[MAP ? 1 : PIECES], pv[SS_TILE], pe[SUMS ? SS_TILE : 1], pdt = 0.0f;
  const int64_t count = seg.t1 - seg.t0, tiles = (count + SS_TILE - 1) / SS_TILE;
  auto base_of = [&](int64_t tile) { return seg.t0 + (REV ? tiles - 1 - tile : tile) * SS_TILE; };
  // Rows and columns that do not exist are read from where the last one lies and put down as zero: no branch around a load, and
  // a row's offset within the tile fits 32 bits (strides are below 2^24).
  auto load = [](const float* base, unsigned off) {
    return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(base) + off * (unsigned)sizeof(float));
  };
  const unsigned lc = lane_on ? l : width - 1;
  auto fetch = [&](int64_t tile) {
    const int64_t t0 = base_of(tile);
    const int last = (int)(seg.t1 - t0 < SS_TILE ? seg.t1 - t0 : SS_TILE) - 1;
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int i = lane + 64 * k, t = i / ROWS < last ? i / ROWS : last, r = r0 + (i % ROWS < rn ? i % ROWS : rn - 1);
      pu[k] = load(U + t0 * us, (unsigned)(t * (int)us + r));
      if (!MAP) pq[k] = load(Q + t0 * qs, (unsigned)(t * (int)qs + r));
    }
#pragma unroll
    for (int t = 0; t < SS_TILE; ++t) {
      const int64_t tok = t0 + (t < last ? t : last);
      pv[t] = load(V + tok * vs, lc);
      if (SUMS) pe[t] = load(E + tok * es, lc);
    }
    pdt = ((const float*)a.dt)[(t0 + (lane < last ? lane : last)) * a.dt_stride + h];
  };
  // The states kept every SS_DOT tokens: written in front of the adjoints' walk, read by it one ahead, but for 64 whole rows, which two
  // waves a SIMD have no room to hold twice (136 registers spilled, gradients of 60 000 x 8 x 64 2 620 us against 2 230).
  constexpr bool AHEAD = !(ROWS == 64 && LG == 1);
  auto kept_of = [&](int64_t done) { return w.chunk_states + ((ss_row_of(seg, SS_DOT) + (done - 1) / SS_DOT) * a.H + h) * per_h; };
  float kept[KIND == SS_DX && !MAP ? RL : 1];
  auto fetch_kept = [&](int64_t done) {
    // row by row from a row length the compiler does not know: ROWS addresses of 64 bits would stay in registers all along
    int P = a.P;
    asm volatile("" : "+s"(P));
    const float* from = kept_of(done) + (int64_t)row0 * P + l;
#pragma unroll
    for (int r = 0; r < RL; ++r, from += P) kept[KIND == SS_DX && !MAP ? r : 0] = has(r) ? *from : 0.0f;
  };

  float carry = 1.0f;   // reverse walks: the decay between the token before (later in time) and this one
  float sum_g = 0.0f;   // maps: this lane's share of the segment's whole exponent
  float dD = 0.0f;
  if (tiles) {
    fetch(0);
    if constexpr (KIND == SS_DX && !MAP && AHEAD) fetch_kept(count);
  }
  for (int64_t tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = base_of(tile);
    const int n = (int)(seg.t1 - t0 < SS_TILE ? seg.t1 - t0 : SS_TILE);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int i = lane + 64 * k;
      const bool on = i / ROWS < n && i % ROWS < rn;
      lu[i / ROWS][i % ROWS] = on ? pu[k] : 0.0f;
      if (!MAP) lq[i / ROWS][i % ROWS] = on ? pq[k] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < SS_TILE; ++t) {
      lv[t][lane] = t < n && lane_on ? pv[t] : 0.0f;
      if (SUMS) le[t][lane] = t < n && lane_on ? pe[t] : 0.0f;
    }
    {
      const float d = lane < n ? ss_delta(pdt, bias, a.softplus) : 0.0f;
      const float g = lane < n ? ss_log_decay(d, A) : 0.0f;
      if (lane < SS_TILE) {
        ldelta[lane] = d;
        ldecay[lane] = expf(g);
      }
      if (MAP) sum_g += g;
    }
    __builtin_amdgcn_sched_barrier(0);
    if (tile + 1 < tiles) fetch(tile + 1);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (KIND == SS_DX && !MAP) {
      // S times the last decay is the adjoint behind the tile
      const int64_t done = t0 + n - seg.t0;
      if (tile == 0 || done % SS_DOT == 0) {
        float dot = 0.0f;
        if constexpr (!AHEAD) fetch_kept(done);
#pragma unroll
        for (int r = 0; r < RL; ++r) dot = __builtin_fmaf(S[r], kept[r], dot);
        dot = ss_wave_sum(dot) * carry;
        if (lane == 0) w.chunk_dots[((ss_row_of(seg, SS_DOT) + (done - 1) / SS_DOT) * a.H + h) * npb + pb] = dot;
        const int64_t next = (done - 1) / SS_DOT * SS_DOT;
        if (AHEAD && next > 0) fetch_kept(next);
      }
    }
    float own = 0.0f;  // U_t . Q_t of token lane / 8
    if constexpr (SUMS) {
#pragma unroll
      for (int r = 0; r < ROWS / 8; ++r) own = __builtin_fmaf(lu[lane >> 3][(lane & 7) + 8 * r], lq[lane >> 3][(lane & 7) + 8 * r], own);
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) own += __shfl_xor(own, off);
    }
    // Tokens behind the segment's last one have no step, no input and a decay of one: every tile is walked whole, without a branch,
    // so that the staged rows of the next tokens are read while one is worked on.
    auto own_of = [&](int t) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(own), 8 * t)); };
    float outs[MAP ? 1 : SS_TILE];
#pragma unroll
    for (int i = 0; i < SS_TILE; ++i) {
      const int t = REV ? SS_TILE - 1 - i : i;
      const float delta = ldelta[t], decay = ldecay[t];
      const float v = KIND == SS_Y || KIND == SS_DC ? delta * lv[t][lane] : lv[t][lane];
      const float s = REV ? carry : decay;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < RL; ++r) {
        if (SUMS) o[r & 3] = __builtin_fmaf(lq[t][row0 + r], S[r], o[r & 3]);
        S[r] = __builtin_fmaf(lu[t][row0 + r], v, S[r] * s);
        // both at once: left alone, the old and the new state are kept side by side (64 rows x 64 lanes: 31 to 196 registers spilled,
        // gradients of 60 000 x 8 x 64 2 790 us against 2 230)
        if (SUMS) asm("" : "+v"(S[r]), "+v"(o[r & 3]));
        if (!MAP && !SUMS) o[r & 3] = __builtin_fmaf(lq[t][row0 + r], S[r], o[r & 3]);
        if (RL > 64 && r % 32 == 31) __builtin_amdgcn_sched_barrier(0);  // no registers for the rows of more tokens
      }
      carry = decay;
      if constexpr (!MAP) {
        float out = (o[0] + o[1]) + (o[2] + o[3]);
        if (SUMS) out *= s;
#pragma unroll
        for (int off = COLS; off < 64; off <<= 1) out += __shfl_xor(out, off);
        // made here and now: used only under a condition, it would be formed there, from every token's state
        asm volatile("" : "+v"(out));
        if constexpr (KIND == SS_Y) {
          outs[t] = __builtin_fmaf(D, lv[t][lane], out);
        } else if constexpr (KIND == SS_DX) {
          const float xv = le[t][lane];
          outs[t] = __builtin_fmaf(delta, __builtin_fmaf(own_of(t), v, out), D * lv[t][lane]);
          if (lane < COLS) dD = __builtin_fmaf(xv, lv[t][lane], dD);
          le[t][lane] = lane < COLS ? xv * out : 0.0f;
        } else if constexpr (KIND == SS_DC) {
          outs[t] = __builtin_fmaf(own_of(t), v, out);
          le[t][lane] = lane < COLS ? le[t][lane] * out : 0.0f;
        } else {
          outs[t] = delta * out;
        }
      }
    }
    if constexpr (!MAP) {
      float* rows = out_rows + t0 * out_stride;
#pragma unroll
      for (int t = 0; t < SS_TILE; ++t)
        if (writes && t < n) rows[t * out_stride + l] = outs[t];
    }
    if constexpr (SUMS) {  // the tile's dots: 8 lanes a token
      __syncthreads();
      const float* p = &le[lane >> 3][(lane & 7) * 8];
      const f32x4 u = *reinterpret_cast<const f32x4*>(p), v = *reinterpret_cast<const f32x4*>(p + 4);
      float sum = ((u[0] + u[1]) + (u[2] + u[3])) + ((v[0] + v[1]) + (v[2] + v[3]));
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor(sum, off);
      const int t = lane >> 3;
      if ((lane & 7) == 0 && t < n) {
        const int64_t row = (t0 + t) * a.H + h;
        float* pair = w.pair + row * (1 + npb);
        if constexpr (KIND == SS_DX) {
          w.behind[row * npb + pb] = sum;
          if (pb == 0) pair[0] = own;
        } else {
          w.dg[(row * npb + pb) * nnb + lane_block] = sum;
          if (lane_block == 0) pair[1 + pb] = own;
        }
      }
    }
    if constexpr (KIND == SS_DC && !MAP) {
      const int64_t done = t0 + n - seg.t0;
      if (done % SS_DOT == 0 || tile + 1 == tiles) {
        float* keep = const_cast<float*>(kept_of(done));
#pragma unroll
        for (int r = 0; r < RL; ++r)
          if (has(r)) keep[at(r)] = S[r];
      }
    }
  }

  if constexpr (MAP) {
    float* local = (REV ? w.adjoints : a.slot_states) + ((int64_t)blockIdx.x * a.H + h) * per_h;
#pragma unroll
    for (int r = 0; r < RL; ++r)
      if (has(r)) local[at(r)] = REV ? S[r] * carry : S[r];
    sum_g = ss_wave_sum(sum_g);
    if (!REV && lane == 0 && pb == 0) a.slot_decay[(int64_t)blockIdx.x * a.H + h] = expf(sum_g);
  } else if (LANE_P) {
    if (KIND == SS_DX) {
      dD = ss_wave_sum(dD);
      if (lane == 0) w.dD_part[((int64_t)blockIdx.x * a.H + h) * npb + pb] = dD;
    }
    float* final_state = KIND == SS_DX ? a.dh0 : a.ht;
    if (single && final_state) {
      final_state += ((int64_t)seg.seq * a.H + h) * per_h;
#pragma unroll
      for (int r = 0; r < RL; ++r)
        if (has(r)) final_state[at(r)] = REV ? S[r] * carry : S[r];
    }
  }
}

template <int KIND, bool MAP>
static int ss_serial_launch(const lampa_ss_args& a, const SsGrad& w, hipStream_t s) {
  const int npb = ss_blocks64(a.P), nnb = ss_blocks64(a.N);
  constexpr bool LANE_P = KIND == SS_Y || KIND == SS_DX;
  const dim3 grid((unsigned)ss_slots(&a), (unsigned)(a.H * npb * (LANE_P ? 1 : nnb)));
  const int rows = LANE_P ? a.N : (a.P < 64 ? a.P : 64);
  const bool narrow = (LANE_P ? a.P : a.N) <= 32;
  LAMPA_PROF(s, "start");
#define SS_GO(ROWS)                                                                                            \
  if (narrow) hipLaunchKernelGGL((ss_serial_kernel<ROWS, 2, KIND, MAP>), grid, dim3(64), 0, s, a, w);         \
  else hipLaunchKernelGGL((ss_serial_kernel<ROWS, 1, KIND, MAP>), grid, dim3(64), 0, s, a, w)
  if (rows <= 32) { SS_GO(32); }
  else if (rows <= 64) { SS_GO(64); }
  else if constexpr (LANE_P) { SS_GO(128); }
#undef SS_GO
  LAMPA_PROF(s, MAP ? "ss_serial_kernel<map>" : "ss_serial_kernel<walk>");
  return lampa_launch_status();
}

int ss_serial_maps(const lampa_ss_args& a, const SsGrad* grad, hipStream_t s) {
  return grad ? ss_serial_launch<SS_DX, true>(a, *grad, s) : ss_serial_launch<SS_Y, true>(a, SsGrad{}, s);
}

int ss_serial_walk(const lampa_ss_args& a, int kind, const SsGrad& grad, hipStream_t s) {
  switch (kind) {
    case SS_Y: return ss_serial_launch<SS_Y, false>(a, grad, s);
    case SS_DC: return ss_serial_launch<SS_DC, false>(a, grad, s);
    case SS_DX: return ss_serial_launch<SS_DX, false>(a, grad, s);
    default: return ss_serial_launch<SS_DB, false>(a, grad, s);
  }
}
