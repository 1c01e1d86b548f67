// What the state-space scan's kernels share beside the call's arguments: the buffers of the gradients, and the launchers of
// the walks (token-serial for fp32, chunks on the matrix cores for 16-bit types).
#pragma once
#include "ss_common.h"

#define SS_DOT 16  // tokens between two places where the token-serial gradients form <R, S>

struct SsGrad {
  float* adjoints;           // [slots, H, N, P]: the segments' local adjoints, then the adjoint at each segment's end
  float *dB_part, *dC_part;  // [tokens, H * blocks, N]: one part for each head and block of 64 columns of x
  float* dg;                 // [tokens, H, blocks]: the decay exponent's gradient (chunks), or dy_t . ((a_t S_{t-1})^T C_t) (token-serial)
  float* reach;              // chunks: [tokens, H, blocks]: x_t . (R_t^T B_t)
  float* behind;             // token-serial: [tokens, H, blocks]: x_t . ((a_{t+1} R_{t+1})^T B_t), reach without the token's own output
  float* pair;               // token-serial: [tokens, H, 1 + blocks]: C_t . B_t, and dy_t . x_t of each block
  float* chunk_states;       // chunks: the state in front of every 64 tokens, [rows, H, blocks, N padded, 64]
                             // token-serial: the state behind every SS_DOT, [rows, H, N, P]
  float* chunk_dots;         // token-serial: <R, S> behind every SS_DOT tokens, [rows, H, blocks]
  float* param_part;         // [slots * pieces, H, 2]: 256 tokens' share of dA and d dt_bias (pieces of a segment)
  float* dD_part;            // [slots, H, blocks]
};

enum { SS_Y = 0, SS_DC = 1, SS_DX = 2, SS_DB = 3 };

int ss_serial_maps(const lampa_ss_args& a, const SsGrad* grad, hipStream_t s);
int ss_serial_walk(const lampa_ss_args& a, int kind, const SsGrad& grad, hipStream_t s);

int ss_chunk_maps(const lampa_ss_args& a, const SsGrad* grad, hipStream_t s);
int ss_chunk_out(const lampa_ss_args& a, hipStream_t s);
int ss_chunk_grad(const lampa_ss_args& a, const SsGrad& w, hipStream_t s);
static inline int ss_chunk_n(int N) { return N <= 32 ? 32 : N <= 64 ? 64 : 128; }  // N as the chunk kernels are built for it
