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
// Bound by the latency of a token (about 0.5 us with one wave a SIMD: 3 instructions a row, the staged rows' reads, and the
// stores), so segments are short. Measured, fp32: gradients of 6 007 packed tokens x 4 heads, P = N = 32, 241 us for the four
// walks in segments of 64; 77 tokens x 2 sequences whole 50 us.
#include "ss_kernels.h"

#define SS_TILE 8  // tokens staged at once

template <int ROWS, int KIND, bool MAP>
__global__ void __launch_bounds__(64) ss_serial_kernel(lampa_ss_args a, SsGrad w) {
  constexpr bool REV = KIND == SS_DX || KIND == SS_DB;  // from the end of the segment
  constexpr bool LANE_P = KIND == SS_Y || KIND == SS_DX;
  constexpr int PIECES = ROWS * SS_TILE / 64;
  constexpr int UNROLL = ROWS <= 64 ? 4 : 2;
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
  const int l = lane_block * 64 + lane;
  const bool lane_on = l < (LANE_P ? a.P : a.N);
  const int r0 = row_block * 64, rn = (LANE_P ? a.N : a.P) - r0;  // rows r0 .. of the state; rn of them exist
  const int64_t per_h = (int64_t)a.N * a.P;
  // element (row r, lane) of a state [N, P]
  auto at = [&](int r) { return LANE_P ? (int64_t)(r0 + r) * a.P + l : (int64_t)l * a.P + r0 + r; };

  const bool single = !MAP && (a.cu_seqlens ? a.n_tokens : a.seq_len) <= a.seg_tokens;
  float S[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) S[r] = 0.0f;
  if (!MAP && !seg.outside) {
    const float* init = single ? (REV ? a.dht : a.h0) : (REV ? w.adjoints : a.slot_states);
    if (init) {
      init += ((single ? (int64_t)seg.seq : (int64_t)blockIdx.x) * a.H + h) * per_h;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (lane_on && r < rn) S[r] = init[at(r)];
    }
  }

  const float* x = (const float*)a.x + (int64_t)h * a.P;
  const float* dy = (const float*)a.dy + (int64_t)h * a.P;
  const float* Bm = (const float*)a.B + (int64_t)grp * a.N;
  const float* Cm = (const float*)a.C + (int64_t)grp * a.N;
  const int64_t dy_stride = (int64_t)a.H * a.P;
  const float *U, *Q, *V;
  int64_t us, qs, vs;
  if constexpr (KIND == SS_Y) { U = Bm; us = a.B_stride; Q = Cm; qs = a.C_stride; V = x; vs = a.x_stride; }
  else if constexpr (KIND == SS_DC) { U = x; us = a.x_stride; Q = dy; qs = dy_stride; V = Bm; vs = a.B_stride; }
  else if constexpr (KIND == SS_DX) { U = Cm; us = a.C_stride; Q = Bm; qs = a.B_stride; V = dy; vs = dy_stride; }
  else { U = dy; us = dy_stride; Q = x; qs = a.x_stride; V = Cm; vs = a.C_stride; }
  // a second lane vector: C (dC's dot with it), x (dx's)
  constexpr bool EXTRA = !MAP && (KIND == SS_DC || KIND == SS_DX);
  const float* E = KIND == SS_DC ? Cm : x;
  const int64_t es = KIND == SS_DC ? a.C_stride : a.x_stride;
  const float A = a.A[h], D = a.D ? a.D[h] : 0.0f, bias = a.dt_bias ? a.dt_bias[h] : 0.0f;

  __shared__ float lu[SS_TILE][ROWS], lq[MAP ? 1 : SS_TILE][ROWS], lv[SS_TILE][64], le[EXTRA ? SS_TILE : 1][64];
  __shared__ float ldelta[SS_TILE], ldecay[SS_TILE];
  float pu[PIECES], pq[PIECES], pv[SS_TILE], pe[SS_TILE], pdt = 0.0f;
  const int64_t count = seg.t1 - seg.t0, tiles = (count + SS_TILE - 1) / SS_TILE;
  auto base_of = [&](int64_t tile) { return seg.t0 + (REV ? tiles - 1 - tile : tile) * SS_TILE; };
  auto fetch = [&](int64_t tile) {
    const int64_t t0 = base_of(tile);
    const int n = (int)(seg.t1 - t0 < SS_TILE ? seg.t1 - t0 : SS_TILE);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int i = lane + 64 * k, t = i / ROWS, r = i % ROWS;
      const bool on = t < n && r < rn;
      pu[k] = on ? U[(t0 + t) * us + r0 + r] : 0.0f;
      if (!MAP) pq[k] = on ? Q[(t0 + t) * qs + r0 + r] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < SS_TILE; ++t) {
      const bool on = t < n && lane_on;
      pv[t] = on ? V[(t0 + t) * vs + l] : 0.0f;
      if (EXTRA) pe[t] = on ? E[(t0 + t) * es + l] : 0.0f;
    }
    if (lane < n) pdt = ((const float*)a.dt)[(t0 + lane) * a.dt_stride + h];
  };

  float carry = 1.0f;   // reverse walks: the decay between the token before (later in time) and this one
  float sum_g = 0.0f;   // maps: this lane's share of the segment's whole exponent
  float dD = 0.0f;
  if (tiles && !seg.outside) fetch(0);
  for (int64_t tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = base_of(tile);
    const int n = (int)(seg.t1 - t0 < SS_TILE ? seg.t1 - t0 : SS_TILE);
    __syncthreads();
    if (!seg.outside) {
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const int i = lane + 64 * k;
        lu[i / ROWS][i % ROWS] = pu[k];
        if (!MAP) lq[i / ROWS][i % ROWS] = pq[k];
      }
#pragma unroll
      for (int t = 0; t < SS_TILE; ++t) {
        lv[t][lane] = pv[t];
        if (EXTRA) le[t][lane] = pe[t];
      }
      if (lane < SS_TILE) {
        const float d = lane < n ? ss_delta(pdt, bias, a.softplus) : 0.0f;
        const float g = lane < n ? ss_log_decay(d, A) : 0.0f;
        ldelta[lane] = d;
        ldecay[lane] = expf(g);
        if (MAP) sum_g += g;
      }
      if (tile + 1 < tiles) fetch(tile + 1);
    }
    __syncthreads();
    // Tokens behind the segment's last one have no step, no input and a decay of one: every tile is walked whole, so that the
    // staged rows of one token can be read while the one before is worked on.
#pragma unroll UNROLL
    for (int i = 0; i < SS_TILE; ++i) {
      const int t = REV ? SS_TILE - 1 - i : i;
      const int64_t tok = t0 + t;
      const bool real = t < n;
      float out = 0.0f, delta = 0.0f;
      if (!seg.outside) {
        delta = ldelta[t];
        const float decay = ldecay[t];
        const float v = KIND == SS_Y || KIND == SS_DC ? delta * lv[t][lane] : lv[t][lane];
        const float s = REV ? carry : decay;
        if constexpr (KIND == SS_DX && !MAP) {
          const int64_t done = tok + 1 - seg.t0;
          if (real && (done % SS_DOT == 0 || tok + 1 == seg.t1)) {  // S times the last decay is the adjoint behind this token
            const int64_t row = (ss_row_of(seg, SS_DOT) + (done - 1) / SS_DOT) * a.H + h;
            const float* kept = w.chunk_states + row * per_h;
            float dot = 0.0f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
              if (lane_on && r < rn) dot = __builtin_fmaf(S[r], kept[at(r)], dot);
            dot = ss_wave_sum(dot) * carry;
            if (lane == 0) w.chunk_dots[row * npb + pb] = dot;
          }
        }
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          S[r] = __builtin_fmaf(lu[t][r], v, S[r] * s);
          if (!MAP) o[r & 3] = __builtin_fmaf(lq[t][r], S[r], o[r & 3]);
        }
        out = (o[0] + o[1]) + (o[2] + o[3]);
        carry = decay;
      }
      if (!real) continue;
      if constexpr (!MAP) {
        if constexpr (KIND == SS_Y) {
          if (lane_on)
            ((float*)a.y)[tok * a.y_stride + (int64_t)h * a.P + l] =
                seg.outside ? 0.0f : __builtin_fmaf(D, lv[t][lane], out);
        } else if constexpr (KIND == SS_DX) {
          const float dyv = seg.outside ? 0.0f : lv[t][lane], xv = seg.outside ? 0.0f : le[t][lane];
          if (lane_on) ((float*)a.dx)[tok * dy_stride + (int64_t)h * a.P + l] =
              __builtin_fmaf(delta, out, D * dyv);
          const float q = ss_wave_sum(lane_on ? xv * out : 0.0f);
          if (lane == 0) w.reach[(tok * a.H + h) * npb + pb] = q;
          dD = __builtin_fmaf(xv, dyv, dD);
        } else if constexpr (KIND == SS_DC) {
          if (lane_on) w.dC_part[(tok * a.H * npb + h * npb + pb) * a.N + l] = out;
          const float u = ss_wave_sum(lane_on && !seg.outside ? le[t][lane] * out : 0.0f);
          if (lane == 0) w.dg[((tok * a.H + h) * npb + pb) * nnb + lane_block] = u;
          // the state behind every SS_DOT tokens (and behind the last one), for <R, S> there
          const int64_t done = tok + 1 - seg.t0;
          if (!seg.outside && (done % SS_DOT == 0 || tok + 1 == seg.t1)) {
            float* keep = w.chunk_states + ((ss_row_of(seg, SS_DOT) + (done - 1) / SS_DOT) * a.H + h) * per_h;
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
              if (lane_on && r < rn) keep[at(r)] = S[r];
          }
        } else {
          if (lane_on) w.dB_part[(tok * a.H * npb + h * npb + pb) * a.N + l] = delta * out;
        }
      }
    }
  }

  if constexpr (MAP) {
    float* local = (REV ? w.adjoints : a.slot_states) + ((int64_t)blockIdx.x * a.H + h) * per_h;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (lane_on && r < rn) local[at(r)] = REV ? S[r] * carry : S[r];
    sum_g = ss_wave_sum(sum_g);
    if (!REV && lane == 0 && pb == 0) a.slot_decay[(int64_t)blockIdx.x * a.H + h] = expf(sum_g);
  } else if (LANE_P) {
    if (KIND == SS_DX) {
      dD = ss_wave_sum(dD);
      if (lane == 0) w.dD_part[((int64_t)blockIdx.x * a.H + h) * npb + pb] = seg.outside ? 0.0f : dD;
    }
    float* final_state = KIND == SS_DX ? a.dh0 : a.ht;
    if (single && final_state && !seg.outside) {
      final_state += ((int64_t)seg.seq * a.H + h) * per_h;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (lane_on && r < rn) final_state[at(r)] = REV ? S[r] * carry : S[r];
    }
  }
}

template <int KIND, bool MAP>
static int ss_serial_launch(const lampa_ss_args& a, const SsGrad& w, hipStream_t s) {
  const int npb = ss_blocks64(a.P), nnb = ss_blocks64(a.N);
  constexpr bool LANE_P = KIND == SS_Y || KIND == SS_DX;
  const dim3 grid((unsigned)ss_slots(&a), (unsigned)(a.H * npb * (LANE_P ? 1 : nnb)));
  const int rows = LANE_P ? a.N : (a.P < 64 ? a.P : 64);
  LAMPA_PROF(s, "start");
  if (rows <= 32) hipLaunchKernelGGL((ss_serial_kernel<32, KIND, MAP>), grid, dim3(64), 0, s, a, w);
  else if (rows <= 64) hipLaunchKernelGGL((ss_serial_kernel<64, KIND, MAP>), grid, dim3(64), 0, s, a, w);
  else if constexpr (LANE_P) hipLaunchKernelGGL((ss_serial_kernel<128, KIND, MAP>), grid, dim3(64), 0, s, a, w);
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
