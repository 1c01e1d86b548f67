// Pieces of the chunked form of the state-space scan on the matrix cores (gfx950), 64 tokens at a time, for 16-bit types.
//
// With gamma_t the sum of the decay exponents of a chunk's tokens up to t and S the state before the chunk,
//   y_t = e^{gamma_t} S^T C_t + sum_{s <= t} M[t, s] x_s,     M[t, s] = e^{gamma_t - gamma_s} delta_s (B_s . C_t),
//   S  <- e^{gamma_end} S + sum_s B_s (delta_s e^{gamma_end - gamma_s} x_s)^T.
// A workgroup of four waves walks a segment for one head and 64 columns of x; wave w keeps columns 16 w .. + 15 of the state in
// accumulators (16 x 16 x 32 products). The accumulator layout of one product is the operand layout of the next: the state is
// read out of the registers it is summed up in, and the pair weights go through LDS only because the four waves share them.
//
// Rounding: B, C, x (and dy) enter as they are. The pair weights are rounded once to the input type, as any operand of the
// matrix cores has to be; they carry the same relative error as the output's own rounding. The state and the decayed x enter as
// two or three operands of the input type each, value and remainders (ScParts): the state is handed from chunk to chunk and out
// to the caller in fp32, and its sums are what the gradient of the decays is made of.
//
// Measured, 60 000 tokens x 8 heads of 64 in bf16, one group of B and C. N = 64, forward: local states 29 us, join 11, outputs 62 (137
// MB; 600 vector instructions a wave and chunk keep the vector units two thirds busy, the matrix cores a sixth). N = 128 with
// gradients: local states 56, join 11 and 13 from the end, outputs 105, kept states and local adjoints 153 (of them 246 MB of kept
// states written), gradients 330, sums of dB and dC over the heads 125 (490 MB, 3.9 TB/s). fp16, whose operands are scaled: 134 us
// forward at N = 64 where bf16 takes 116 (with the host), 531 against 497 with gradients.
#pragma once
#include "ss_kernels.h"

#define SC_BLOCK 256

template <typename T>
using sc_x8 = typename OpVec<T>::x8;
template <typename T>
using sc_x4 = typename OpVec<T>::x4;

// An fp32 value as a sum of operand values: fp16 has it to 2^-22 in two, bf16 to 2^-17 in two and whole in three. Three go in
// wherever a state or adjoint that is handed on, or a sum that dA and d dt_bias are made of, comes out; two where the product
// itself is rounded to the input type.
template <typename T>
struct ScParts { static const int n = __is_same(T, __bf16) ? 3 : 2; };
// Two values at a time, as they are converted. fp16: the values are taken out of the compiler's sight, which would form the first
// part of a product in one rounding and the remainder from one of two, which now and then (ties) is another value.
template <typename T, int PARTS>
__device__ __forceinline__ void sc_split(float a, float b, typename OpVec<T>::x2 (&part)[PARTS]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, _Float16)) asm("" : "+v"(a), "+v"(b));
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    part[k] = __builtin_convertvector(f32x2{a, b}, typename OpVec<T>::x2);
    if (k + 1 < PARTS) {
      a -= (float)part[k][0];
      b -= (float)part[k][1];
    }
  }
}

// fp16 has no room for every fp32 value: operands made from fp32 are scaled by a power of two that brings the largest of
// them below 2^15 (and small ones up to it), and the product is scaled back. bf16 has fp32's range: 1.
template <typename T>
__device__ __forceinline__ float sc_scale_for(float largest) {
  if constexpr (__is_same(T, _Float16)) {
    if (!(largest > 0.0f) || !(largest < __builtin_inff())) return 1.0f;
    int e = 14 - (int)((__float_as_uint(largest) >> 23) - 127);
    e = e < -100 ? -100 : (e > 100 ? 100 : e);
    return __uint_as_float((unsigned)(127 + e) << 23);
  }
  return 1.0f;
}
// The largest so far: a value that is not finite does not set the scale of the others that share it.
__device__ __forceinline__ float sc_larger(float big, float v) {
  v = fabsf(v);
  return v < __builtin_inff() ? fmaxf(big, v) : big;
}
__device__ __forceinline__ float sc_inverse(float power_of_two) { return __uint_as_float((254u << 23) - __float_as_uint(power_of_two)); }

// The scale of a lane's column (row or column i of an operand whose values lie in the lanes i, 16 + i, 32 + i and 48 + i), from the
// largest value of each lane, and its inverse for the rows 4 g + r of a product that has the operand on the left. A scale of its own
// for each: a column of small values loses no bits to a large one beside it.
template <typename T>
__device__ __forceinline__ float sc_column_scale(float largest, int lane, f32x4& back) {
  largest = fmaxf(largest, __shfl_xor(largest, 16));
  largest = fmaxf(largest, __shfl_xor(largest, 32));
  const float s = sc_scale_for<T>(largest), inverse = sc_inverse(s);
#pragma unroll
  for (int r = 0; r < 4; ++r) back[r] = __shfl(inverse, 4 * (lane >> 4) + r);
  return s;
}

__device__ __forceinline__ float sc_wave_max(float v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}

// The compiler moves nothing across: left alone it requests the operands of many products at once and runs out of registers.
__device__ __forceinline__ void sc_fence() { __builtin_amdgcn_sched_barrier(0); }

// The lane's number, as a value the compiler knows nothing about: addresses and comparisons made from it are formed anew in every
// turn of a loop instead of being kept in registers all through it.
__device__ __forceinline__ int sc_fresh(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// One thread's share of a [64, W] tile on its way from memory to LDS. Rows from `n` on and columns from `cols` on are zero.
template <typename T, int W>
struct ScTile {
  sc_x8<T> v[W / 32];
  // `base`: column 0 of row 0, the same in the whole workgroup, as are stride and n: a row's address is a scalar and the lane's
  // offset within 32 bits, one for all rows (64-bit pointers of their own for each would cost more registers than the state).
  template <bool VEC>
  __device__ __forceinline__ void fetch(const T* base, int64_t stride, int n, int cols) {
    const int row0 = threadIdx.x / (W / 8), c = threadIdx.x % (W / 8) * 8;
    const unsigned off = (unsigned)(row0 * (int)stride + c) * (unsigned)sizeof(T);
    if (VEC && n == 64 && cols >= W) {  // nothing to leave out
#pragma unroll
      for (int k = 0; k < W / 32; ++k)
        v[k] = *reinterpret_cast<const sc_x8<T>*>(reinterpret_cast<const char*>(base + (int64_t)(k * (2048 / W)) * stride) + off);
      return;
    }
#pragma unroll
    for (int k = 0; k < W / 32; ++k) {
      const int row = row0 + k * (2048 / W);
      const char* p = reinterpret_cast<const char*>(base + (int64_t)(k * (2048 / W)) * stride);
      sc_x8<T> x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (T)0.0f;
      if (row < n && c < cols) {
        if constexpr (VEC) x = *reinterpret_cast<const sc_x8<T>*>(p + off);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < cols) x[e] = *reinterpret_cast<const T*>(p + (off + e * (unsigned)sizeof(T)));
      }
      v[k] = x;
    }
  }
  // Values of a 16-bit type with their sign bits changed where `bits` (two to a word) has ones.
  __device__ __forceinline__ void flip(unsigned bits) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int k = 0; k < W / 32; ++k) v[k] = __builtin_bit_cast(sc_x8<T>, __builtin_bit_cast(u32x4, v[k]) ^ bits);
  }
  // Stored in the column order of op_perm32: a lane's share of a 32-wide contraction step is one 16-byte piece.
  __device__ __forceinline__ void put(T* tile, int stride) const {
#pragma unroll
    for (int k = 0; k < W / 32; ++k) {
      const int q = threadIdx.x + SC_BLOCK * k, row = q / (W / 8), c = q % (W / 8) * 8;
      T* p = tile + row * stride + (c & ~31) + op_perm32_piece((c >> 3) & 3);
      sc_x4<T> a, b;
#pragma unroll
      for (int e = 0; e < 4; ++e) { a[e] = v[k][e]; b[e] = v[k][4 + e]; }
      *reinterpret_cast<sc_x4<T>*>(p) = a;
      *reinterpret_cast<sc_x4<T>*>(p + 8) = b;
    }
  }
  // The first row of this thread that holds a value which is not finite, 64 if none.
  __device__ __forceinline__ int first_bad() const {
    int bad = 64;
#pragma unroll
    for (int k = W / 32 - 1; k >= 0; --k) {
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      const u32x4 w = __builtin_bit_cast(u32x4, v[k]);
      constexpr unsigned E = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
      bool b = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) b |= (w[e] & E) == E || (w[e] >> 16 & E) == E;
      if (b) bad = (threadIdx.x + SC_BLOCK * k) / (W / 8);
    }
    return bad;
  }
};

// The matrix instructions round an accumulator that is smaller than the products added to it towards minus infinity (measured: 1.5
// beside an accumulator of +-0.75 last places comes out as 1.5 + 0 and 1.5 - 1). What is formed that way is too small by about 2^-25 of
// the largest summand, whatever its sign, which sums over all tokens (dA, d dt_bias) do not average out as they do ordinary
// rounding. So the gradients work on dy with its sign changed in every other chunk, and change the signs of what comes out back:
// everything of theirs is linear in dy, and the errors of one chunk make up for those of the next.
__device__ __forceinline__ unsigned sc_flip_bits(float sign) { return sign < 0.0f ? 0x80008000u : 0u; }

// What a chunk's steps and decays come to, one entry a token. gamma is summed up in 64 bits: it reaches -200 and beyond where a
// head decays fast, and the exponents of neighbouring tokens are differences of it, which have to be right to 2^-24 for dA and
// d dt_bias, sums over all tokens, to be.
struct ScDecay {
  float gamma[64];  // gamma_t log2(e), rounded (what that leaves out goes to `rest`, as 2 to its power)
  float delta[64];
  float grow[64];   // e^{gamma_t}
  float left[64];   // e^{gamma_end - gamma_t}
  float end;        // e^{gamma_end}
  float sum;        // gamma_end log2(e)
};
template <int CTRL, int ROWS>
__device__ __forceinline__ double sc_dpp_add(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xF, false);
  return x + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// One wave, lane = token; tokens from n on have no step.
__device__ __forceinline__ void sc_decays(ScDecay& d, float* rest, float raw, int n, float bias, float A, int softplus) {
  const int lane = lane_id();
  const float delta = lane < n ? ss_delta(raw, bias, softplus) : 0.0f;
  double g = 0.0;
  if (lane < n) {
    g = (double)delta * (double)A;
    g = (g < SS_MIN_LOG_DECAY ? (double)SS_MIN_LOG_DECAY : g) * 1.4426950408889634;
  }
  g = sc_dpp_add<GDR_DPP_ROW_SHR(1), 0xF>(g);
  g = sc_dpp_add<GDR_DPP_ROW_SHR(2), 0xF>(g);
  g = sc_dpp_add<GDR_DPP_ROW_SHR(4), 0xF>(g);
  g = sc_dpp_add<GDR_DPP_ROW_SHR(8), 0xF>(g);
  g = sc_dpp_add<GDR_DPP_ROW_BCAST15, 0xA>(g);
  g = sc_dpp_add<GDR_DPP_ROW_BCAST31, 0xC>(g);
  const double end = __shfl(g, 63);
  const float rounded = (float)g;
  d.gamma[lane] = rounded;
  if (rest) rest[lane] = __builtin_amdgcn_exp2f((float)(g - (double)rounded));
  d.delta[lane] = delta;
  d.grow[lane] = __builtin_amdgcn_exp2f(rounded);
  d.left[lane] = __builtin_amdgcn_exp2f((float)(end - g));
  if (lane == 63) {
    d.end = __builtin_amdgcn_exp2f((float)end);
    d.sum = (float)end;
  }
}

// Element (n, p) of a state [N, P], zero outside; the address is held inside, so that loads need no branch.
__device__ __forceinline__ float sc_state_at(const float* state, int n, int p, int N, int P) {
  const float v = state[(unsigned)((n < N ? n : N - 1) * P + (p < P ? p : P - 1))];
  return n < N && p < P ? v : 0.0f;
}

// Columns 16 w .. of a 64-row tile as an operand of the products over its rows (rows 32 kk ..): one for each kk.
template <typename T>
__device__ __forceinline__ void sc_columns(const T* tile, int stride, int col0, int lane, sc_x8<T> (&out)[2]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) out[kk] = op_ld_tr16<T, true>(tile, stride, col0, 32 * kk, lane);
}
// The weights of a lane's rows in such an operand.
__device__ __forceinline__ void sc_row_weights(const float* w, int kk, int lane, float (&out)[8]) {
  const int g = lane >> 4;
  const f32x4 a = *reinterpret_cast<const f32x4*>(w + 32 * kk + 4 * g), b = *reinterpret_cast<const f32x4*>(w + 32 * kk + 16 + 4 * g);
#pragma unroll
  for (int e = 0; e < 4; ++e) { out[e] = a[e]; out[4 + e] = b[e]; }
}
// An operand over a chunk's 64 rows, weighted row by row, in parts. Returns what a product with it on the right is to be multiplied with:
// fp16's weighted values are scaled so that the largest of a lane's column (the product's column) comes to between 2^14 and 2^15. The
// scale is made from the values, not from the weights alone: x or dy of 1e-4 would leave remainders below fp16's smallest step (states
// were off by 3e-4, now by 1e-7 as with any other size of x).
template <typename T, int PARTS>
__device__ __forceinline__ float sc_weighted(const sc_x8<T> (&x)[2], const float (&w)[2][8], sc_x8<T> (&out)[2][PARTS]) {
  constexpr bool F16 = __is_same(T, _Float16);
  float s = 1.0f;
  if constexpr (F16) {
    float big = 0.0f;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) big = sc_larger(big, (float)x[kk][e] * w[kk][e]);
    big = fmaxf(big, __shfl_xor(big, 16));
    big = fmaxf(big, __shfl_xor(big, 32));
    s = sc_scale_for<T>(big);
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float a = (float)x[kk][e] * w[kk][e], b = (float)x[kk][e + 1] * w[kk][e + 1];
      if constexpr (F16) {
        a *= s;
        b *= s;
      }
      typename OpVec<T>::x2 part[PARTS];
      sc_split<T, PARTS>(a, b, part);
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        out[kk][k][e] = part[k][0];
        out[kk][k][e + 1] = part[k][1];
      }
    }
  return sc_inverse(s);
}
// Two accumulator tiles (32 rows) as an operand in parts.
template <typename T, int PARTS>
__device__ __forceinline__ void sc_state_operand(const f32x4& a, const f32x4& b, float scale, sc_x8<T> (&out)[PARTS]) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float u = e < 4 ? a[e] : b[e - 4], v = e < 4 ? a[e + 1] : b[e - 3];
    typename OpVec<T>::x2 part[PARTS];
    if constexpr (__is_same(T, _Float16)) sc_split<T, PARTS>(u * scale, v * scale, part);
    else sc_split<T, PARTS>(u, v, part);
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      out[k][e] = part[k][0];
      out[k][e + 1] = part[k][1];
    }
  }
}
// acc + left * (the operand's parts), the smallest first
template <typename X8, int PARTS>
__device__ __forceinline__ f32x4 sc_mfma_left(const X8& left, const X8 (&right)[PARTS], f32x4 acc) {
#pragma unroll
  for (int k = PARTS - 1; k >= 0; --k) acc = mfma16(left, right[k], acc);
  return acc;
}
template <typename X8, int PARTS>
__device__ __forceinline__ f32x4 sc_mfma_right(const X8 (&left)[PARTS], const X8& right, f32x4 acc) {
#pragma unroll
  for (int k = PARTS - 1; k >= 0; --k) acc = mfma16(left[k], right, acc);
  return acc;
}

// acc[nt] += (columns 16 nt .. of the tile)^T * (an operand over its 64 rows, in parts). Every product goes to
// another tile than the one before it, which it would otherwise wait for.
template <typename T, int NT, int PARTS>
__device__ __forceinline__ void sc_add_products(const T* tile, int stride, int lane, const sc_x8<T> (&right)[2][PARTS],
                                                f32x4 (&acc)[NT]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    sc_x8<T> left[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) left[nt] = op_ld_tr16<T, true>(tile, stride, 16 * nt, 32 * kk, lane);
#pragma unroll
    for (int k = PARTS - 1; k >= 0; --k) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt] = mfma16(left[nt], right[kk][k], acc[nt]);
    }
  }
}

// S <- end S + (tile)^T * (v, its rows weighted), the product of a wave's 16 columns with all rows of the state.
template <typename T, int NT, int PARTS>
__device__ __forceinline__ void sc_update(const T* tile, int stride, int lane, const sc_x8<T> (&v)[2], const float (&wt)[2][8], float end,
                                          f32x4 (&S)[NT]) {
  sc_x8<T> vw[2][PARTS];
  const float back = sc_weighted<T, PARTS>(v, wt, vw);
  if constexpr (__is_same(T, _Float16)) {
    f32x4 d[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) d[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    sc_add_products<T, NT, PARTS>(tile, stride, lane, vw, d);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) S[nt] = S[nt] * end + d[nt] * back;
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) S[nt] *= end;
    sc_add_products<T, NT, PARTS>(tile, stride, lane, vw, S);
  }
}

// Whether every row of a call can be read in 16-byte pieces and written in 8-byte ones. The kernels are built for both: loads
// element by element beside the others would cost those registers (local states at N = 64: 182 against 122).
static bool sc_vectors(const lampa_ss_args& a) {
  auto rows = [](const void* p, int64_t stride, int inner) { return (uintptr_t)p % 16 == 0 && stride % 8 == 0 && inner % 8 == 0; };
  return rows(a.x, a.x_stride, a.P) && rows(a.B, a.B_stride, a.N) && rows(a.C, a.C_stride, a.N) && rows(a.dy, 8, a.P) &&
         rows(a.dx, 8, a.P) && (uintptr_t)a.y % 8 == 0 && a.y_stride % 4 == 0;
}

// Slots along x in a multiple of 8: workgroups are dealt to the 8 dies in turn, so the heads of a segment, which read the same
// rows of B and C, meet in one die's L2.
static dim3 sc_grid(const lampa_ss_args& a) {
  return dim3((unsigned)((ss_slots(&a) + 7) / 8 * 8), (unsigned)(a.H * ss_blocks64(a.P)));
}


// Place of element (row 16 nt + row, column 16 w + col) of a chunk's kept state: float4 number (tile nt, columns 32 (w / 2) + 16
// (w % 2) + 4 g ..) of lane 16 g + row, so that a lane of the gradients reads its operand's columns of one row in whole float4s, a
// wave 1 KiB at a time.
__device__ __forceinline__ int sc_kept_at(int nt, int w, int row, int col) { return ((nt * 4 + w) * 64 + 16 * (col >> 2) + row) * 4 + (col & 3); }

// Sum over the 16 lanes of a row, in every lane of it.
__device__ __forceinline__ float sc_row16_sum(float x) {
  x += dpp_f32<GDR_DPP_QUAD_XOR1, 0xF>(0.0f, x);
  x += dpp_f32<GDR_DPP_QUAD_XOR2, 0xF>(0.0f, x);
  x += dpp_f32<0x141, 0xF>(0.0f, x);  // mirrored within 8 lanes
  x += dpp_f32<0x140, 0xF>(0.0f, x);  // mirrored within 16
  return x;
}
