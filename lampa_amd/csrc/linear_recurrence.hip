// The gated linear recurrence, its gradients and its single-token step (gfx950). For every channel of every sequence
//   a_t = exp(A sigmoid(r_t)),  u_t = [sqrt(1 - a_t^2)] sigmoid(i_t) x_t,  h_t = a_t h_{t-1} + u_t,  y_t = act(z_t) h_t;
// gradients, with the adjoint G run from the end:
//   G_t = act(z_t) dy_t + a_{t+1} G_{t+1},   dz_t = dy_t h_t act'(z_t),   dx = G m sigmoid(i),   di = G m x sigmoid(i)(1 - sigmoid(i)),
//   d log a = G (a h_{t-1} - sigmoid(i) x a^2 / m),   dr = d log a  A sigmoid(r)(1 - sigmoid(r)),   dA = sum d log a sigmoid(r).
//
// Bound by bytes: every input is read once and every output written once, in one pass. A workgroup takes a tile of tokens of
// one sequence x 2 LR channels: LR lanes side by side over channels, 256 / LR runs of LR_TOK tokens one after the other. A run's
// effect on the state is the map h -> P h + H with P = prod a; the runs' maps are joined in LDS, and the tile's map is left for the
// tiles behind it. LR_GROUP tiles form a group, whose last tile leaves the group's map as soon as it has the others'; LR_GROUP
// groups form a block, whose last tile leaves the state. A tile starts from the state before its block under the maps of the
// block's groups before its own and of its group's tiles before it: two steps behind the slowest of them, where a chain of
// states would cost a step a tile. The order is always this one, so repeated calls give the same bits. Maps and states are words that
// are written whole and hold a pattern no result has until then, so the value is its own flag and no fence is needed.
// Tiles are handed out by a counter, in the order in which they wait for each other: a tile waits only for tiles that were
// handed out before it, so every wait ends.
//
// Measured (medians of a kernel trace; a copy of 1 GiB runs at 5.1 TB/s): 60 000 x 512 in bf16, both gates: forward 101 us (307 MB,
// 3.0 TB/s), gradients 182 us (553 MB, 3.0 TB/s) and 10 for the sums of dA; 24 packed sequences of 15 000 x 192 in fp16 19 us; fp32, 5
// packed sequences of 6 007 x 128: 13 and 18 us; one token of 250 x 1024 in bf16 3.5 us. What is left is that tiles under way together finish together, whose loads and whose
// arithmetic (35 us of the forward) so come one after the other: the forward without any wait, on states of zero, takes 68 us. More
// or fewer workgroups a CU, tiles of 128 or 256 tokens, fewer polls and a chain of states in place of the groups' maps change it by
// less than 5 us; tiles of 32 take 128.
#include "../../include/lampa_amd.h"
#include "gdr_common.h"
#include "row_sums.h"

#include <type_traits>

#pragma clang fp contract(off)  // fused only where it is written: the kernels for one and two channels a lane give the same bits

#define LR_FWD_BLOCK 256
#define LR_TOK 16    // tokens of a forward run
#define LR_BWD_BLOCK 512
#define LR_BWD_TOK 8  // tokens of a run of the gradients: tiles of the same length
#define LR_GROUP 16  // tiles of a group, groups of a block
#define LR_POLLS (1 << 22)  // polls a wait may take (seconds); it then ends with NaN
#define LR_EMPTY64 0xffffffffffffffffull
#define LR_EMPTY32 0xffffffffu
#define LR_OFF 0x80000000u  // byte offset of a lane without a channel: past the end of every buffer

enum { LR_ACT_NONE = 0, LR_ACT_SILU = 1, LR_ACT_SIGMOID = 2 };

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------------------------------------------ sequences and tiles
struct LrSeqs {
  const int64_t* cu;  // device [n_seq + 1] or null: dense sequences of len tokens
  int64_t len, n_tokens;
  int n_seq, tile;    // tokens of a tile
  bool one_tile;      // no more tokens than a tile: cu are the caller's boundaries, which nobody has put in order
};
struct LrTile {
  int64_t t0, t1;  // its tokens
  int64_t first;   // slot of the sequence's first tile
  int seq, index, count;  // place among the `count` tiles of sequence seq
  bool live, outside;     // a slot without a tile; rows behind the last sequence
};

__device__ __forceinline__ int64_t lr_bound(const LrSeqs& q, int i) {
  if (!q.cu) return (int64_t)i * q.len;
  if (i == 0) return 0;
  if (i > q.n_seq) return q.n_tokens;
  return q.cu[i];
}
// Boundary i of a call of one tile: the largest of the first i as the caller gave them, held inside the tokens; by the whole wave.
__device__ __forceinline__ int lr_bound_of_one_tile(const LrSeqs& q, int i) {
  const int n = (int)q.n_tokens;
  if (i > q.n_seq) return n;
  int most = 0;
  for (int64_t k = 1 + (threadIdx.x & 63); k <= i; k += 64) {
    const int64_t c = q.cu[k];
    const int in = c < 0 ? 0 : (c > n ? n : (int)c);
    most = in > most ? in : most;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const int other = __shfl_xor(most, d);
    most = other > most ? other : most;
  }
  return __builtin_amdgcn_readfirstlane(most);
}
// Sequence i takes its slots from floor(begin / tile) + i on: room for its ceil(length / tile) tiles (one where it is empty)
// without knowing the lengths on the host. In a call of one tile slot i is sequence i's.
__device__ __forceinline__ LrTile lr_tile(const LrSeqs& q, int64_t slot) {
  LrTile s;
  int64_t b, e;
  s.live = true;
  s.outside = false;
  if (!q.cu) {
    const int64_t per = q.len ? (q.len + q.tile - 1) / q.tile : 1;
    s.seq = (int)(slot / per);
    s.index = (int)(slot % per);
    s.first = s.seq * per;
    b = (int64_t)s.seq * q.len;
    e = b + q.len;
  } else if (q.one_tile) {
    s.live = slot <= q.n_seq;
    s.seq = s.live ? (int)slot : q.n_seq;  // the rows behind the last sequence count as sequence n_seq
    s.index = 0;
    s.first = slot;
    s.outside = s.seq == q.n_seq;
    b = lr_bound_of_one_tile(q, s.seq);
    e = lr_bound_of_one_tile(q, s.seq + 1);
  } else {
    int lo = 0, hi = q.n_seq;  // the rows behind the last sequence count as sequence n_seq
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (lr_bound(q, mid) / q.tile + mid <= slot) lo = mid; else hi = mid - 1;
    }
    s.seq = lo;
    b = lr_bound(q, lo);
    e = lr_bound(q, lo + 1);
    s.first = b / q.tile + lo;
    s.index = (int)(slot - s.first);
    s.outside = lo == q.n_seq;
    s.live = s.index >= 0 && (s.index == 0 || b + (int64_t)s.index * q.tile < e);
  }
  const int64_t n = e > b ? e - b : 0;
  s.count = n ? (int)((n + q.tile - 1) / q.tile) : 1;
  s.t0 = b + (int64_t)s.index * q.tile;
  s.t1 = s.t0 + q.tile < e ? s.t0 + q.tile : e;
  if (s.t1 < s.t0) s.t1 = s.t0;
  return s;
}

#define LR_BLOCK_TILES (LR_GROUP * LR_GROUP)

// Words of a call: a counter, the tiles' maps [slots, D] (P low, H high), the groups' [slots / LR_GROUP + 1, D], the blocks' states
// [slots / LR_BLOCK_TILES + 1, D] (a slot's group and block: tiles that leave theirs are that many slots or more apart), the
// boundaries in order.
struct LrWords {
  unsigned* ticket;
  unsigned long long *maps, *group_maps;
  unsigned* states;
  int64_t* cu;
};

// Every word empty, the counter at 0; workgroup 0 also copies the boundaries, held inside the tokens and made monotone (tiles
// wait for each other by them: whatever the caller's memory holds, every tile that is waited for has to exist).
__global__ void __launch_bounds__(256) lr_init_kernel(LrWords w, int64_t n_maps, int64_t n_states, const int64_t* __restrict__ cu, int n_seq,
                                                      int64_t n_tokens) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = at; i < n_maps; i += step) w.maps[i] = LR_EMPTY64;
  for (int64_t i = at; i < n_states; i += step) w.states[i] = LR_EMPTY32;
  if (blockIdx.x) return;
  if (threadIdx.x == 0) *w.ticket = 0;
  if (!cu) return;
  __shared__ int64_t most[256];
  int64_t before = 0;
  for (int64_t i0 = 0; i0 <= n_seq; i0 += 256) {
    const int64_t i = i0 + threadIdx.x;
    int64_t c = i <= n_seq && i > 0 ? cu[i] : 0;
    c = c < 0 ? 0 : (c > n_tokens ? n_tokens : c);
    most[threadIdx.x] = c;
    __syncthreads();
    for (int d = 1; d < 256; d <<= 1) {
      const int64_t o = threadIdx.x >= d ? most[threadIdx.x - d] : 0;
      __syncthreads();
      if (o > most[threadIdx.x]) most[threadIdx.x] = o;
      __syncthreads();
    }
    int64_t v = most[threadIdx.x];
    if (v < before) v = before;
    if (i <= n_seq) w.cu[i] = v;
    const int64_t top = most[255];
    before = top > before ? top : before;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ loads and arithmetic
// A lane's V channels of one row. Rows are read and written through buffer descriptors that end with the tile's last row: what lies
// outside reads as zero and is not written, so tails need no branches.
template <typename T, int V>
struct LrRaw;
template <> struct LrRaw<float, 2> { typedef u32x2 type; };
template <> struct LrRaw<float, 1> { typedef unsigned type; };
template <> struct LrRaw<__bf16, 2> { typedef unsigned type; };
template <> struct LrRaw<__bf16, 1> { typedef unsigned short type; };
template <> struct LrRaw<_Float16, 2> { typedef unsigned type; };
template <> struct LrRaw<_Float16, 1> { typedef unsigned short type; };

template <typename R>
__device__ __forceinline__ R lr_load(__amdgpu_buffer_rsrc_t buf, unsigned offset) {
  if constexpr (sizeof(R) == 8) return __builtin_bit_cast(R, __builtin_amdgcn_raw_buffer_load_b64(buf, offset, 0, 0));
  else if constexpr (sizeof(R) == 4) return __builtin_bit_cast(R, __builtin_amdgcn_raw_buffer_load_b32(buf, offset, 0, 0));
  else return __builtin_bit_cast(R, __builtin_amdgcn_raw_buffer_load_b16(buf, offset, 0, 0));
}
template <typename R>
__device__ __forceinline__ void lr_store(__amdgpu_buffer_rsrc_t buf, unsigned offset, R v) {
  if constexpr (sizeof(R) == 8) __builtin_amdgcn_raw_buffer_store_b64(v, buf, offset, 0, 0);
  else if constexpr (sizeof(R) == 4) __builtin_amdgcn_raw_buffer_store_b32(v, buf, offset, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b16(v, buf, offset, 0, 0);
}
template <typename T, int V>
__device__ __forceinline__ void lr_widen(typename LrRaw<T, V>::type raw, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = GdrElem<T>::to_float(__builtin_bit_cast(T, raw));
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    const vec x = __builtin_bit_cast(vec, raw);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = GdrElem<T>::to_float(x[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ typename LrRaw<T, V>::type lr_narrow(const float (&v)[V]) {
  if constexpr (V == 1) {
    return __builtin_bit_cast(typename LrRaw<T, V>::type, GdrElem<T>::from_float(v[0]));
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = GdrElem<T>::from_float(v[i]);
    return __builtin_bit_cast(typename LrRaw<T, V>::type, x);
  }
}
// Rows t0 .. t1 - 1 of a tensor of D columns.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t lr_buffer(const void* base, int64_t stride, int elem, const LrTile& s, int D) {
  const int64_t rows = s.t1 - s.t0;
  const unsigned size = rows > 0 && base ? (unsigned)(((rows - 1) * stride + D) * elem) : 0u;
  return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + s.t0 * stride * elem), 0, size, 0x00020000);
}

__device__ __forceinline__ float lr_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// a = exp(l) and k = 1 - a, near a = 1 without loss: there k is the sum of its series in t = -l (8 terms: t^8 / 9! = 1e-8 of it at
// t = 1/2) and a = 1 - k is off by its own rounding alone. (The exponential instruction's error, up to a step of a and not
// the same in both directions, adds up over the thousands of tokens that such a channel remembers: 7e-6 of dA at 6 007 tokens.)
// SMALL: |l| is below 1/2 whatever the gates hold.
template <bool SMALL>
__device__ __forceinline__ void lr_decay(float l, float& a, float& k) {
  const float t = -l;
  float p = __builtin_fmaf(t, -1.0f / 40320.0f, 1.0f / 5040.0f);
  p = __builtin_fmaf(t, p, -1.0f / 720.0f);
  p = __builtin_fmaf(t, p, 1.0f / 120.0f);
  p = __builtin_fmaf(t, p, -1.0f / 24.0f);
  p = __builtin_fmaf(t, p, 1.0f / 6.0f);
  p = __builtin_fmaf(t, p, -0.5f);
  p = __builtin_fmaf(t, p, 1.0f);
  k = t * p;
  a = 1.0f - k;
  if constexpr (!SMALL) {
    const float e = __expf(l);
    const bool far = !(__builtin_fabsf(t) < 0.5f);
    a = far ? e : a;
    k = far ? 1.0f - e : k;
  }
}
// sqrt(1 - a^2) of a and 1 - a.
__device__ __forceinline__ float lr_unit(float a, float k) { return __builtin_amdgcn_sqrtf(k * (1.0f + a)); }
__device__ __forceinline__ float lr_act(float z, int act) {
  if (act == LR_ACT_NONE) return z;
  const float s = lr_sigmoid(z);
  return act == LR_ACT_SILU ? z * s : s;
}

// ------------------------------------------------------------------------------------------------ maps between tiles
__device__ __forceinline__ unsigned lr_bits(float x) { return x != x ? 0x7fc00000u : __float_as_uint(x); }  // never the empty pattern
__device__ __forceinline__ void lr_put_map(unsigned long long* p, float P, float H) {
  __hip_atomic_store(p, ((unsigned long long)lr_bits(H) << 32) | lr_bits(P), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void lr_put_state(unsigned* p, float h) {
  __hip_atomic_store(p, lr_bits(h), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// N words of a lane's V channels, the first n of them wanted, `step` words apart; `ok`: none of them is empty. AGAIN: only those that
// were are asked for.
template <int V, int N, bool AGAIN>
__device__ __forceinline__ void lr_look(const unsigned long long* at, int64_t step, int n, unsigned long long (&w)[N][V], bool& ok) {
  ok = true;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (k < n && (!AGAIN || w[k][v] == LR_EMPTY64))
        w[k][v] = __hip_atomic_load(at + k * step + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) ok = ok && (k >= n || w[k][v] != LR_EMPTY64);
}
// (P, H) <- the maps of the first n words, one behind the other.
template <int V, int N>
__device__ __forceinline__ void lr_compose(const unsigned long long (&w)[N][V], int n, float (&P)[V], float (&H)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    P[v] = 1.0f;
    H[v] = 0.0f;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (k < n) {
        const float p = __uint_as_float((unsigned)w[k][v]), h = __uint_as_float((unsigned)(w[k][v] >> 32));
        H[v] = __builtin_fmaf(p, H[v], h);
        P[v] *= p;
      }
}

struct LrArgs {
  const void *x, *r, *i, *z;
  const float *A, *h0;
  void* y;
  float *ht, *tile_states;
  const void* dy;
  const float* dht;
  void *dx, *dr, *di, *dz;
  float *dA_parts, *dh0;
  int64_t xs, rs, is, zs;
  LrSeqs q;
  LrWords w;
  int64_t slots, jobs;    // tiles, and their workgroups
  int D, lanes, cblocks;  // lanes side by side, workgroups over the channels
  int act, normalize;
  int handed_out;  // tiles wait for each other and are handed out by the counter
};

// The workgroup's tile and block of channels; false: none (the grid's last row is not full). BACK: in the order of the gradients, last
// tiles first.
template <bool BACK>
__device__ __forceinline__ bool lr_job(const LrArgs& a, int64_t& slot, int& cb) {
  __shared__ unsigned ticket;
  unsigned job = blockIdx.y * gridDim.x + blockIdx.x;
  if (a.handed_out) {
    if (threadIdx.x == 0) ticket = atomicAdd(a.w.ticket, 1u);
    __syncthreads();
    job = ticket;
  }
  job = __builtin_amdgcn_readfirstlane(job);  // the same for all: tiles' places and buffers stay in scalar registers
  if (job >= a.jobs) return false;
  slot = job / (unsigned)a.cblocks;
  cb = (int)(job % (unsigned)a.cblocks);
  if (BACK) slot = a.slots - 1 - slot;
  return true;
}

// What a tile of the forward starts from (or, BACK, what reaches a tile from behind), in every thread for its channels; leaves the
// group's map and the block's state where the tile is the last of one. `place` counts the sequence's tiles in the order of the walk,
// Pt and Ht are the tile's own map (in the threads of run `writer`), `more`: tiles follow; `meanwhile` is called once the first look is
// under way, for loads that nobody waits for.
template <int V, int BLOCK, bool BACK, typename F>
__device__ __forceinline__ void lr_enter(const LrArgs& a, const LrTile& s, int64_t slot, int place, int c, bool on, int lane, int run,
                                         int writer, bool more, const float (&Pt)[V], const float (&Ht)[V], const float* first,
                                         float2 (*sm)[V], float (*base)[V], float (&h)[V], F meanwhile) {
  const int runs = BLOCK / a.lanes, pos = place % LR_GROUP, grp = place / LR_GROUP % LR_GROUP;
  const int64_t dir = BACK ? 1 : -1;  // towards the tiles that were walked before
  // each run takes `per` places of the group, and of the block's groups, oldest first
  constexpr int MOST = LR_GROUP * 64 / BLOCK, PER = MOST < 1 ? 1 : MOST;  // 64 lanes side by side; fewer lanes, more runs
  const int per = runs >= LR_GROUP ? 1 : LR_GROUP / runs, p0 = run * per;
  const int nt = on ? (pos - p0 < per ? pos - p0 : per) : 0, ng = on ? (grp - p0 < per ? grp - p0 : per) : 0;
  const unsigned long long* tiles = a.w.maps + (slot + dir * (pos - p0)) * a.D + c;
  // group g of the block before this one's: its last tile lies pos + 1 + LR_GROUP (grp - 1 - g) tiles away
  const int64_t last0 = slot + dir * (pos + 1 + (int64_t)LR_GROUP * (grp - 1 - p0));
  const unsigned long long* groups = a.w.group_maps + last0 / LR_GROUP * a.D + c;
  const bool from_block = run == 0 && on && place >= LR_BLOCK_TILES;
  const unsigned* state = a.w.states + (slot + dir * (place % LR_BLOCK_TILES + 1)) / LR_BLOCK_TILES * a.D + c;
  unsigned long long wt[PER][V], wg[PER][V];
  unsigned ws[V];
  bool have_tiles, have_groups;
  lr_look<V, PER, false>(tiles, -dir * a.D, nt, wt, have_tiles);
  lr_look<V, PER, false>(groups, -dir * a.D, ng, wg, have_groups);
  bool have_state = true;
  auto look_state = [&]() {
    if (!from_block) return;
    have_state = true;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ws[v] = __hip_atomic_load(state + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      have_state = have_state && ws[v] != LR_EMPTY32;
    }
  };
  look_state();
  meanwhile();
  // a wait that runs out leaves empty words, which are NaN
  for (int polls = 0; !have_tiles && polls < LR_POLLS; ++polls) {
    __builtin_amdgcn_s_sleep(2);
    lr_look<V, PER, true>(tiles, -dir * a.D, nt, wt, have_tiles);
  }
  float P[V], H[V];
  lr_compose<V, PER>(wt, nt, P, H);
#pragma unroll
  for (int v = 0; v < V; ++v) sm[threadIdx.x][v] = float2{P[v], H[v]};
  __syncthreads();
  float Pg[V], Hg[V];  // the tiles of the group before this one
#pragma unroll
  for (int v = 0; v < V; ++v) { Pg[v] = 1.0f; Hg[v] = 0.0f; }
  for (int k = 0; k < runs && k * per < pos; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = sm[k * a.lanes + lane][v];
      Hg[v] = __builtin_fmaf(m.x, Hg[v], m.y);
      Pg[v] *= m.x;
    }
  }
  if (run == writer && on && more && pos == LR_GROUP - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      lr_put_map(a.w.group_maps + slot / LR_GROUP * a.D + c + v, Pt[v] * Pg[v], __builtin_fmaf(Pt[v], Hg[v], Ht[v]));
  }
  for (int polls = 0; !(have_groups && have_state) && polls < LR_POLLS; ++polls) {
    __builtin_amdgcn_s_sleep(2);
    lr_look<V, PER, true>(groups, -dir * a.D, ng, wg, have_groups);
    look_state();
  }
  lr_compose<V, PER>(wg, ng, P, H);
  __syncthreads();  // the tiles' maps have been read
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sm[threadIdx.x][v] = float2{P[v], H[v]};
    if (run == 0) base[lane][v] = from_block ? __uint_as_float(ws[v]) : (on && first ? first[(int64_t)s.seq * a.D + c + v] : 0.0f);
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = base[lane][v];
  for (int k = 0; k < runs && k * per < grp; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = sm[k * a.lanes + lane][v];
      h[v] = __builtin_fmaf(m.x, h[v], m.y);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = __builtin_fmaf(Pg[v], h[v], Hg[v]);
    if (run == writer && on && more && place % LR_BLOCK_TILES == LR_BLOCK_TILES - 1)
      lr_put_state(a.w.states + slot / LR_BLOCK_TILES * a.D + c + v, __builtin_fmaf(Pt[v], h[v], Ht[v]));
  }
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int V, bool HASI, bool HASZ>
__global__ void __launch_bounds__(LR_FWD_BLOCK) lr_fwd_kernel(const LrArgs a) {
  typedef typename LrRaw<T, V>::type raw;
  constexpr int E = sizeof(T);
  __shared__ float2 maps[LR_FWD_BLOCK][V], before[LR_FWD_BLOCK][V];
  __shared__ float base[64][V];
  int64_t slot;
  int cb;
  if (!lr_job<false>(a, slot, cb)) return;
  const LrTile s = lr_tile(a.q, slot);
  if (!s.live) return;
  const int lane = threadIdx.x % a.lanes, run = threadIdx.x / a.lanes, runs = LR_FWD_BLOCK / a.lanes;
  const int c = (cb * a.lanes + lane) * V;
  const bool on = c < a.D;  // V divides D
  const int row = run * LR_TOK;
  const __amdgpu_buffer_rsrc_t yb = lr_buffer(a.y, a.D, E, s, a.D);
  const unsigned yo = on ? (unsigned)(row * a.D + c) * E : LR_OFF;
  if (s.outside) {  // as many tiles as it takes, zero
    float zero[V];
#pragma unroll
    for (int v = 0; v < V; ++v) zero[v] = 0.0f;
#pragma unroll
    for (int j = 0; j < LR_TOK; ++j) lr_store<raw>(yb, yo + j * a.D * E, lr_narrow<T, V>(zero));
    return;
  }
  raw rr[LR_TOK], rx[LR_TOK], ri[HASI ? LR_TOK : 1];
  {
    const __amdgpu_buffer_rsrc_t rb = lr_buffer(a.r, a.rs, E, s, a.D), xb = lr_buffer(a.x, a.xs, E, s, a.D);
    const unsigned ro = on ? (unsigned)(row * a.rs + c) * E : LR_OFF, xo = on ? (unsigned)(row * a.xs + c) * E : LR_OFF;
    const unsigned rstep = (unsigned)a.rs * E, xstep = (unsigned)a.xs * E;
#pragma unroll
    for (int j = 0; j < LR_TOK; ++j) {
      rr[j] = lr_load<raw>(rb, ro + j * rstep);
      rx[j] = lr_load<raw>(xb, xo + j * xstep);
    }
    if constexpr (HASI) {
      const __amdgpu_buffer_rsrc_t ib = lr_buffer(a.i, a.is, E, s, a.D);
      const unsigned io = on ? (unsigned)(row * a.is + c) * E : LR_OFF, istep = (unsigned)a.is * E;
#pragma unroll
      for (int j = 0; j < LR_TOK; ++j) ri[j] = lr_load<raw>(ib, io + j * istep);
    }
  }
  const int64_t left = s.t1 - s.t0 - row;
  const int n = left < 0 ? 0 : (left < LR_TOK ? (int)left : LR_TOK);  // tokens of this run
  float A[V], P[V], H[V], L[V], av[LR_TOK][V], uv[LR_TOK][V];
  bool small = true;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = on ? a.A[c + v] : 0.0f;
    small = small && __builtin_fabsf(A[v]) < 0.5f;
    H[v] = L[v] = 0.0f;
  }
  // plain: every token is there and |A| < 1/2 throughout the wave, as in most of a call
  auto gates = [&](auto plain) {
    constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
    for (int j = 0; j < LR_TOK; ++j) {
      float rv[V], xv[V], iv[V];
      lr_widen<T, V>(rr[j], rv);
      lr_widen<T, V>(rx[j], xv);
      if constexpr (HASI) lr_widen<T, V>(ri[j], iv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float l = A[v] * lr_sigmoid(rv[v]), d, k, u = xv[v];
        lr_decay<PLAIN>(l, d, k);
        if constexpr (HASI) u *= lr_sigmoid(iv[v]);
        if (a.normalize) u *= lr_unit(d, k);
        if (!PLAIN && j >= n) { l = 0.0f; d = 1.0f; u = 0.0f; }
        av[j][v] = d;
        uv[j][v] = u;
        L[v] += l;
        H[v] = __builtin_fmaf(d, H[v], u);
      }
    }
  };
  if (__all(small && n == LR_TOK)) gates(std::true_type()); else gates(std::false_type());
  // from the sum of the exponents: a product of 16 rounded factors would be off by 16 roundings, tile after tile
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float k;
    lr_decay<false>(L[v], P[v], k);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) maps[threadIdx.x][v] = float2{P[v], H[v]};
  __syncthreads();
  float Pb[V], Hb[V];  // the runs before this one
#pragma unroll
  for (int v = 0; v < V; ++v) { Pb[v] = 1.0f; Hb[v] = 0.0f; }
  for (int k = 0; k < run; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = maps[k * a.lanes + lane][v];
      Hb[v] = __builtin_fmaf(m.x, Hb[v], m.y);
      Pb[v] *= m.x;
    }
  }
  const bool last_run = run == runs - 1, last_tile = s.index == s.count - 1;
  float Pt[V], Ht[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Ht[v] = __builtin_fmaf(P[v], Hb[v], H[v]);
    Pt[v] = Pb[v] * P[v];
    if (last_run && on && !last_tile) lr_put_map(a.w.maps + slot * a.D + c + v, Pt[v], Ht[v]);
  }
  float h[V];
  raw rz[HASZ ? LR_TOK : 1];
  lr_enter<V, LR_FWD_BLOCK, false>(a, s, slot, s.index, c, on, lane, run, runs - 1, !last_tile, Pt, Ht, a.h0, before, base, h, [&]() {
    if constexpr (HASZ) {  // the output's gate: not needed for the map that others wait for
      const __amdgpu_buffer_rsrc_t zb = lr_buffer(a.z, a.zs, E, s, a.D);
      const unsigned zo = on ? (unsigned)(row * a.zs + c) * E : LR_OFF, zstep = (unsigned)a.zs * E;
#pragma unroll
      for (int j = 0; j < LR_TOK; ++j) rz[j] = lr_load<raw>(zb, zo + j * zstep);
    }
  });
  if (on) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (run == 0 && a.tile_states) a.tile_states[slot * a.D + c + v] = h[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = __builtin_fmaf(Pb[v], h[v], Hb[v]);
#pragma unroll
  for (int j = 0; j < LR_TOK; ++j) {
    float out[V], zv[V];
    if constexpr (HASZ) lr_widen<T, V>(rz[j], zv);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = __builtin_fmaf(av[j][v], h[v], uv[j][v]);
      out[v] = h[v];
      if constexpr (HASZ) out[v] *= lr_act(zv[v], a.act);
    }
    lr_store<raw>(yb, yo + j * a.D * E, lr_narrow<T, V>(out));
  }
  // behind a run's tokens the state stays as it is, so the run that holds the sequence's last token (or the first, of an empty one) has it
  if (a.ht && last_tile && on && (n > 0 ? s.t0 + row + n == s.t1 : run == 0 && s.t1 == s.t0)) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.ht[(int64_t)s.seq * a.D + c + v] = h[v];
  }
}

// ------------------------------------------------------------------------------------------------ gradients
template <typename T, int V, bool HASI, bool HASZ>
__global__ void __launch_bounds__(LR_BWD_BLOCK, sizeof(T) == 2 ? 4 : 2) lr_bwd_kernel(const LrArgs a) {
  typedef typename LrRaw<T, V>::type raw;
  constexpr int E = sizeof(T), TOK = LR_BWD_TOK;
  __shared__ float2 maps[LR_BWD_BLOCK][V], before[LR_BWD_BLOCK][V];
  __shared__ float base[64][V], carry[LR_BWD_BLOCK][V];
  int64_t slot;
  int cb;
  if (!lr_job<true>(a, slot, cb)) return;
  const LrTile s = lr_tile(a.q, slot);
  const int lane = threadIdx.x % a.lanes, run = threadIdx.x / a.lanes, runs = LR_BWD_BLOCK / a.lanes;
  const int c = (cb * a.lanes + lane) * V;
  const bool on = c < a.D;
  if (!s.live || s.outside) {
    if (run == 0 && on) {
#pragma unroll
      for (int v = 0; v < V; ++v) a.dA_parts[slot * a.D + c + v] = 0.0f;
    }
    if (!s.live) return;
  }
  const int row = run * TOK;
  const __amdgpu_buffer_rsrc_t dxb = lr_buffer(a.dx, a.D, E, s, a.D), drb = lr_buffer(a.dr, a.D, E, s, a.D);
  const __amdgpu_buffer_rsrc_t dib = lr_buffer(a.di, a.D, E, s, a.D), dzb = lr_buffer(a.dz, a.D, E, s, a.D);
  const unsigned yo = on ? (unsigned)(row * a.D + c) * E : LR_OFF, ystep = (unsigned)a.D * E;
  if (s.outside) {
    float zero[V];
#pragma unroll
    for (int v = 0; v < V; ++v) zero[v] = 0.0f;
    const raw none = lr_narrow<T, V>(zero);
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
      lr_store<raw>(dxb, yo + j * ystep, none);
      lr_store<raw>(drb, yo + j * ystep, none);
      if constexpr (HASI) lr_store<raw>(dib, yo + j * ystep, none);
      if constexpr (HASZ) lr_store<raw>(dzb, yo + j * ystep, none);
    }
    return;
  }
  raw rr[TOK], rx[TOK], rdy[TOK], ri[HASI ? TOK : 1], rz[HASZ ? TOK : 1];
  {
    const __amdgpu_buffer_rsrc_t rb = lr_buffer(a.r, a.rs, E, s, a.D), xb = lr_buffer(a.x, a.xs, E, s, a.D);
    const __amdgpu_buffer_rsrc_t db = lr_buffer(a.dy, a.D, E, s, a.D);
    const unsigned ro = on ? (unsigned)(row * a.rs + c) * E : LR_OFF, xo = on ? (unsigned)(row * a.xs + c) * E : LR_OFF;
    const unsigned rstep = (unsigned)a.rs * E, xstep = (unsigned)a.xs * E;
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
      rr[j] = lr_load<raw>(rb, ro + j * rstep);
      rx[j] = lr_load<raw>(xb, xo + j * xstep);
      rdy[j] = lr_load<raw>(db, yo + j * ystep);
    }
    if constexpr (HASI) {
      const __amdgpu_buffer_rsrc_t ib = lr_buffer(a.i, a.is, E, s, a.D);
      const unsigned io = on ? (unsigned)(row * a.is + c) * E : LR_OFF, istep = (unsigned)a.is * E;
#pragma unroll
      for (int j = 0; j < TOK; ++j) ri[j] = lr_load<raw>(ib, io + j * istep);
    }
    if constexpr (HASZ) {
      const __amdgpu_buffer_rsrc_t zb = lr_buffer(a.z, a.zs, E, s, a.D);
      const unsigned zo = on ? (unsigned)(row * a.zs + c) * E : LR_OFF, zstep = (unsigned)a.zs * E;
#pragma unroll
      for (int j = 0; j < TOK; ++j) rz[j] = lr_load<raw>(zb, zo + j * zstep);
    }
  }
  const int64_t left = s.t1 - s.t0 - row;
  const int n = left < 0 ? 0 : (left < TOK ? (int)left : TOK);
  float A[V], h[V], P[V], L[V], H[V], C[V], av[TOK][V], hv[TOK + 1][V];
  bool small = true;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = on ? a.A[c + v] : 0.0f;
    small = small && __builtin_fabsf(A[v]) < 0.5f;
    h[v] = on ? a.tile_states[slot * a.D + c + v] : 0.0f;
    L[v] = H[v] = C[v] = 0.0f;
    hv[0][v] = 0.0f;
  }
  const bool plain = __all(small && n == TOK);
  float dv[TOK][V];  // what reaches h from y; not kept over the wait, formed again behind it
  auto gates = [&](auto simple) {
    constexpr bool PLAIN = decltype(simple)::value;
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
      float rv[V], xv[V], iv[V], zv[V], dy[V];
      lr_widen<T, V>(rr[j], rv);
      lr_widen<T, V>(rx[j], xv);
      lr_widen<T, V>(rdy[j], dy);
      if constexpr (HASI) lr_widen<T, V>(ri[j], iv);
      if constexpr (HASZ) lr_widen<T, V>(rz[j], zv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float l = A[v] * lr_sigmoid(rv[v]), d, k, u = xv[v];
        lr_decay<PLAIN>(l, d, k);
        if constexpr (HASI) u *= lr_sigmoid(iv[v]);
        if (a.normalize) u *= lr_unit(d, k);
        if (!PLAIN && j >= n) { l = 0.0f; d = 1.0f; u = 0.0f; }
        av[j][v] = d;
        dv[j][v] = dy[v];
        if constexpr (HASZ) dv[j][v] *= lr_act(zv[v], a.act);
        H[v] = __builtin_fmaf(d, H[v], u);
        hv[j + 1][v] = H[v];  // from a state of zero
        L[v] += l;
      }
    }
  };
  if (plain) gates(std::true_type()); else gates(std::false_type());
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float k;
    lr_decay<false>(L[v], P[v], k);
  }
#pragma unroll
  for (int j = TOK - 1; j >= 0; --j) {
#pragma unroll
    for (int v = 0; v < V; ++v) C[v] = av[j][v] * (dv[j][v] + C[v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    maps[threadIdx.x][v] = float2{P[v], H[v]};
    carry[threadIdx.x][v] = C[v];
  }
  __syncthreads();
  float Pa[V], Ca[V];  // the runs behind this one
#pragma unroll
  for (int v = 0; v < V; ++v) { Pa[v] = 1.0f; Ca[v] = 0.0f; }
  for (int k = 0; k < run; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = maps[k * a.lanes + lane][v];
      h[v] = __builtin_fmaf(m.x, h[v], m.y);
    }
  }
  for (int k = runs - 1; k > run; --k) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float p = maps[k * a.lanes + lane][v].x;
      Ca[v] = __builtin_fmaf(p, Ca[v], carry[k * a.lanes + lane][v]);
      Pa[v] *= p;
    }
  }
  const bool first_tile = s.index == 0;
  const int place = s.count - 1 - s.index;
  float Pt[V], Ct[V], g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    Ct[v] = __builtin_fmaf(P[v], Ca[v], C[v]);
    Pt[v] = Pa[v] * P[v];
    if (run == 0 && on && !first_tile) lr_put_map(a.w.maps + slot * a.D + c + v, Pt[v], Ct[v]);
  }
  lr_enter<V, LR_BWD_BLOCK, true>(a, s, slot, place, c, on, lane, run, 0, !first_tile, Pt, Ct, a.dht, before, base, g, []() {});
#pragma unroll
  for (int v = 0; v < V; ++v) g[v] = __builtin_fmaf(Pa[v], g[v], Ca[v]);
  // hv[j] <- the state before token j: h under the decays so far, and what has come in since
  {
    float reach[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { hv[0][v] = h[v]; reach[v] = h[v]; }
#pragma unroll
    for (int j = 0; j < TOK; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        reach[v] *= av[j][v];
        hv[j + 1][v] += reach[v];
      }
  }
  float dA[V];
#pragma unroll
  for (int v = 0; v < V; ++v) dA[v] = 0.0f;
  auto grads = [&](auto simple) {
    constexpr bool PLAIN = decltype(simple)::value;
#pragma unroll
    for (int j = TOK - 1; j >= 0; --j) {
      float rv[V], xv[V], iv[V], zv[V], dy[V], dx[V], dr[V], di[V], dz[V];
      lr_widen<T, V>(rr[j], rv);
      lr_widen<T, V>(rx[j], xv);
      lr_widen<T, V>(rdy[j], dy);
      if constexpr (HASI) lr_widen<T, V>(ri[j], iv);
      if constexpr (HASZ) lr_widen<T, V>(rz[j], zv);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float sr = lr_sigmoid(rv[v]), l = A[v] * sr;
        const float si = HASI ? lr_sigmoid(iv[v]) : 1.0f;
        float d, k, dh = dy[v], slope = 1.0f;
        lr_decay<PLAIN>(l, d, k);
        if constexpr (HASZ) {
          dh *= lr_act(zv[v], a.act);
          if (a.act != LR_ACT_NONE) {
            const float sz = lr_sigmoid(zv[v]);
            slope = a.act == LR_ACT_SILU ? sz * __builtin_fmaf(zv[v], 1.0f - sz, 1.0f) : sz * (1.0f - sz);
          }
        }
        const float G = dh + g[v];
        float into = si, dl = d * hv[j][v];  // d h / d x, d h / d log a
        if (a.normalize) {
          const float m = lr_unit(d, k);
          into *= m;
          // a token that keeps all (m = 0) has no slope through m
          dl = __builtin_fmaf(-si * xv[v], m == 0.0f ? 0.0f : d * d * __builtin_amdgcn_rcpf(m), dl);
        }
        dl *= G;
        dx[v] = G * into;
        if constexpr (HASI) di[v] = dx[v] * xv[v] * (1.0f - si);
        dr[v] = dl * l * (1.0f - sr);
        if (PLAIN || j < n) dA[v] = __builtin_fmaf(dl, sr, dA[v]);
        if constexpr (HASZ) dz[v] = dy[v] * hv[j + 1][v] * slope;
        if (!PLAIN && j >= n) d = 1.0f;
        g[v] = d * G;
      }
      lr_store<raw>(dxb, yo + j * ystep, lr_narrow<T, V>(dx));
      lr_store<raw>(drb, yo + j * ystep, lr_narrow<T, V>(dr));
      if constexpr (HASI) lr_store<raw>(dib, yo + j * ystep, lr_narrow<T, V>(di));
      if constexpr (HASZ) lr_store<raw>(dzb, yo + j * ystep, lr_narrow<T, V>(dz));
    }
  };
  if (plain) grads(std::true_type()); else grads(std::false_type());
  if (a.dh0 && first_tile && run == 0 && on) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.dh0[(int64_t)s.seq * a.D + c + v] = g[v];
  }
  __syncthreads();  // the carries have been read
#pragma unroll
  for (int v = 0; v < V; ++v) carry[threadIdx.x][v] = dA[v];
  __syncthreads();
  if (run == 0 && on) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float sum = 0.0f;
      for (int k = 0; k < runs; ++k) sum += carry[k * a.lanes + lane][v];
      a.dA_parts[slot * a.D + c + v] = sum;
    }
  }
}

// ------------------------------------------------------------------------------------------------ one token
template <typename T>
__global__ void __launch_bounds__(256) lr_step_kernel(const T* __restrict__ x, int64_t xs, const T* __restrict__ r, int64_t rs,
                                                      const T* __restrict__ gi, int64_t is, const T* __restrict__ z, int64_t zs,
                                                      const float* __restrict__ A, const float* state, float* new_state,
                                                      T* __restrict__ y, int64_t total, int D, int act, int normalize) {
  const int64_t at = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const int64_t b = at / D;
  const int c = (int)(at % D);
  const float xv = GdrElem<T>::to_float(x[b * xs + c]), rv = GdrElem<T>::to_float(r[b * rs + c]);
  const float iv = gi ? GdrElem<T>::to_float(gi[b * is + c]) : 0.0f, zv = z ? GdrElem<T>::to_float(z[b * zs + c]) : 0.0f;
  float d, k, u = xv;
  lr_decay<false>(A[c] * lr_sigmoid(rv), d, k);
  if (gi) u *= lr_sigmoid(iv);
  if (normalize) u *= lr_unit(d, k);
  const float h = __builtin_fmaf(d, state[at], u);
  new_state[at] = h;
  y[at] = GdrElem<T>::from_float(z ? h * lr_act(zv, act) : h);
}

// ------------------------------------------------------------------------------------------------ host
// Lanes side by side over channels: as many as leave the fewest without a channel, the widest of equals (wider rows for each load).
static int lr_lanes(int D, int V) {
  const int64_t units = (D + V - 1) / V;
  int best = 64;
  int64_t least = (units + 63) / 64 * 64;
  for (int l = 32; l >= 16; l >>= 1) {
    const int64_t taken = (units + l - 1) / l * l;
    if (taken < least) { best = l; least = taken; }
  }
  return best;
}
static int lr_elem(const lampa_lr_args* a) { return a->dtype == GDR_FP32 ? 4 : 2; }
// Two channels a lane where every row of every tensor is aligned to two.
static int lr_width(const lampa_lr_args* a) {
  const uintptr_t mask = 2 * lr_elem(a) - 1;
  uintptr_t all = (uintptr_t)a->x | (uintptr_t)a->decay_gate | (uintptr_t)a->input_gate | (uintptr_t)a->gate | (uintptr_t)a->y |
                  (uintptr_t)a->dy | (uintptr_t)a->dx | (uintptr_t)a->d_decay_gate | (uintptr_t)a->d_input_gate | (uintptr_t)a->d_gate;
  int64_t odd = a->D | a->x_stride | a->decay_stride | (a->input_gate ? a->input_stride : 0) | (a->gate ? a->gate_stride : 0);
  return (all & mask) || (odd & 1) ? 1 : 2;
}
// Tokens of a tile: by D alone, so that both passes cut a call alike however their tensors lie.
static int lr_tile_tokens(int D) { return LR_FWD_BLOCK / lr_lanes(D, D % 2 ? 1 : 2) * LR_TOK; }

static int lr_check(const lampa_lr_args* a) {
  if (!a || a->n_tokens < 0 || a->n_seq < 1 || a->D < 1 || a->dtype < 0 || a->dtype > 2 || a->activation < 0 || a->activation > 2)
    return LAMPA_ERR_INVALID;
  if (!a->cu_seqlens && (a->seq_len < 0 || a->seq_len > a->n_tokens || a->seq_len * a->n_seq != a->n_tokens)) return LAMPA_ERR_INVALID;
  if (a->D > (1 << 20)) return LAMPA_ERR_UNSUPPORTED;
  return LAMPA_OK;
}
static int64_t lr_slots(const lampa_lr_args* a) {
  const int tile = lr_tile_tokens(a->D);
  if (a->cu_seqlens) return a->n_tokens / tile + a->n_seq + 1;
  return (int64_t)a->n_seq * (a->seq_len ? (a->seq_len + tile - 1) / tile : 1);
}
static bool lr_handed_out(const lampa_lr_args* a) { return (a->cu_seqlens ? a->n_tokens : a->seq_len) > lr_tile_tokens(a->D); }

struct LrLayout {
  int64_t maps, states, cu, parts, total;
};
static LrLayout lr_layout(const lampa_lr_args* a, int backward) {
  const int64_t slots = lr_slots(a);
  LrLayout l;
  l.maps = 256;
  l.states = l.maps + (lr_handed_out(a) ? lampa_align_up((slots + slots / LR_GROUP + 1) * a->D * 8, 256) : 0);
  l.cu = l.states + (lr_handed_out(a) ? lampa_align_up((slots / LR_BLOCK_TILES + 1) * a->D * 4, 256) : 0);
  l.parts = l.cu + (lr_handed_out(a) && a->cu_seqlens ? lampa_align_up(((int64_t)a->n_seq + 1) * 8, 256) : 0);
  l.total = l.parts + (backward ? slots * a->D * 4 : 0);
  return l;
}

extern "C" int64_t lampa_lr_slots(const lampa_lr_args* a) {
  const int rc = lr_check(a);
  return rc != LAMPA_OK ? rc : lr_slots(a);
}
extern "C" int64_t lampa_lr_workspace_bytes(const lampa_lr_args* a, int backward) {
  const int rc = lr_check(a);
  return rc != LAMPA_OK ? rc : lr_layout(a, backward).total;
}

static int lr_setup(const lampa_lr_args* a, int backward, LrArgs& k, int V, hipStream_t s) {
  const int lanes_of_tile = lr_lanes(a->D, a->D % 2 ? 1 : 2);
  const int tile = lr_tile_tokens(a->D);
  const int elem = lr_elem(a);
  const int64_t strides[4] = {a->x_stride, a->decay_stride, a->input_gate ? a->input_stride : a->D, a->gate ? a->gate_stride : a->D};
  for (int64_t st : strides) {
    if (st < a->D) return LAMPA_ERR_INVALID;
    if (st > (1 << 30) / ((int64_t)tile * elem)) return LAMPA_ERR_UNSUPPORTED;  // offsets inside a tile are 32 bits wide
  }
  if (a->D > (1 << 30) / ((int64_t)tile * elem)) return LAMPA_ERR_UNSUPPORTED;
  const LrLayout l = lr_layout(a, backward);
  if (!a->workspace || a->workspace_bytes < l.total) return LAMPA_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace % 8) return LAMPA_ERR_INVALID;
  char* ws = (char*)a->workspace;
  k = LrArgs{};
  k.x = a->x; k.r = a->decay_gate; k.i = a->input_gate; k.z = a->gate; k.A = a->A; k.h0 = a->h0;
  k.y = a->y; k.ht = a->ht; k.tile_states = a->tile_states;
  k.dy = a->dy; k.dht = a->dht; k.dx = a->dx; k.dr = a->d_decay_gate; k.di = a->d_input_gate; k.dz = a->d_gate;
  k.dh0 = a->dh0; k.dA_parts = (float*)(ws + l.parts);
  k.xs = a->x_stride; k.rs = a->decay_stride; k.is = a->input_stride; k.zs = a->gate_stride;
  k.slots = lr_slots(a);
  k.w = LrWords{(unsigned*)ws, (unsigned long long*)(ws + l.maps), (unsigned long long*)(ws + l.maps) + k.slots * a->D,
                 (unsigned*)(ws + l.states), (int64_t*)(ws + l.cu)};
  k.handed_out = lr_handed_out(a);
  k.q = LrSeqs{a->cu_seqlens ? (k.handed_out ? (const int64_t*)(ws + l.cu) : a->cu_seqlens) : nullptr, a->seq_len, a->n_tokens, a->n_seq, tile,
               !k.handed_out};
  k.D = a->D;
  k.lanes = lanes_of_tile;
  k.cblocks = (a->D + k.lanes * V - 1) / (k.lanes * V);
  k.act = a->activation;
  k.normalize = a->normalize;
  k.jobs = k.slots * k.cblocks;
  if (k.jobs > 0x7fffffff) return LAMPA_ERR_UNSUPPORTED;
  LAMPA_PROF(s, "start");
  if (k.handed_out) {
    const int64_t n_maps = (k.slots + k.slots / LR_GROUP + 1) * a->D, n_states = (k.slots / LR_BLOCK_TILES + 1) * a->D;
    const int64_t blocks = (n_maps + 1023) / 1024;
    hipLaunchKernelGGL(lr_init_kernel, dim3((unsigned)(blocks < 1 ? 1 : (blocks < 1024 ? blocks : 1024))), dim3(256), 0, s, k.w, n_maps,
                       n_states, a->cu_seqlens, a->n_seq, a->n_tokens);
    LAMPA_PROF(s, "lr_init_kernel");
    return lampa_launch_status();
  }
  return LAMPA_OK;
}

// Workgroups in rows of LR_GRID_ROW: a launch takes fewer than 2^32 threads along one dimension.
#define LR_GRID_ROW (1 << 22)
static dim3 lr_grid(int64_t n) {
  return dim3((unsigned)(n < LR_GRID_ROW ? n : LR_GRID_ROW), (unsigned)((n + LR_GRID_ROW - 1) / LR_GRID_ROW));
}

template <typename T, int V>
static void lr_fwd_go(const LrArgs& k, hipStream_t s) {
  const dim3 grid = lr_grid(k.jobs), block(LR_FWD_BLOCK);
#define LR_GO(I, Z) hipLaunchKernelGGL((lr_fwd_kernel<T, V, I, Z>), grid, block, 0, s, k)
  if (k.i) { if (k.z) LR_GO(true, true); else LR_GO(true, false); }
  else { if (k.z) LR_GO(false, true); else LR_GO(false, false); }
#undef LR_GO
}
template <typename T, int V>
static void lr_bwd_go(const LrArgs& k, hipStream_t s) {
  const dim3 grid = lr_grid(k.jobs), block(LR_BWD_BLOCK);
#define LR_GO(I, Z) hipLaunchKernelGGL((lr_bwd_kernel<T, V, I, Z>), grid, block, 0, s, k)
  if (k.i) { if (k.z) LR_GO(true, true); else LR_GO(true, false); }
  else { if (k.z) LR_GO(false, true); else LR_GO(false, false); }
#undef LR_GO
}

extern "C" int lampa_lr_scan_fwd(const lampa_lr_args* a, void* stream) {
  int rc = lr_check(a);
  if (rc != LAMPA_OK) return rc;
  if (!a->A || (a->n_tokens && (!a->x || !a->decay_gate || !a->y))) return LAMPA_ERR_INVALID;
  hipStream_t s = (hipStream_t)stream;
  const int V = lr_width(a);
  LrArgs k;
  rc = lr_setup(a, 0, k, V, s);
  if (rc != LAMPA_OK) return rc;
  switch (a->dtype * 2 + V - 1) {
    case GDR_BF16 * 2: lr_fwd_go<__bf16, 1>(k, s); break;
    case GDR_BF16 * 2 + 1: lr_fwd_go<__bf16, 2>(k, s); break;
    case GDR_FP16 * 2: lr_fwd_go<_Float16, 1>(k, s); break;
    case GDR_FP16 * 2 + 1: lr_fwd_go<_Float16, 2>(k, s); break;
    case GDR_FP32 * 2: lr_fwd_go<float, 1>(k, s); break;
    default: lr_fwd_go<float, 2>(k, s); break;
  }
  LAMPA_PROF(s, "lr_fwd_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_lr_scan_bwd(const lampa_lr_args* a, void* stream) {
  int rc = lr_check(a);
  if (rc != LAMPA_OK) return rc;
  if (!a->A || !a->tile_states || !a->dA || (a->h0 && !a->dh0) ||
      (a->n_tokens && (!a->x || !a->decay_gate || !a->dy || !a->dx || !a->d_decay_gate || (a->input_gate && !a->d_input_gate) ||
                       (a->gate && !a->d_gate))))
    return LAMPA_ERR_INVALID;
  hipStream_t s = (hipStream_t)stream;
  const int V = lr_width(a);
  LrArgs k;
  rc = lr_setup(a, 1, k, V, s);
  if (rc != LAMPA_OK) return rc;
  switch (a->dtype * 2 + V - 1) {
    case GDR_BF16 * 2: lr_bwd_go<__bf16, 1>(k, s); break;
    case GDR_BF16 * 2 + 1: lr_bwd_go<__bf16, 2>(k, s); break;
    case GDR_FP16 * 2: lr_bwd_go<_Float16, 1>(k, s); break;
    case GDR_FP16 * 2 + 1: lr_bwd_go<_Float16, 2>(k, s); break;
    case GDR_FP32 * 2: lr_bwd_go<float, 1>(k, s); break;
    default: lr_bwd_go<float, 2>(k, s); break;
  }
  LAMPA_PROF(s, "lr_bwd_kernel");
  rc = lampa_launch_status();
  if (rc != LAMPA_OK) return rc;
  return row_sums_launch<float>(k.dA_parts, k.slots, a->D, a->D, 0, 1, RowSumsOut<float>{{a->dA, nullptr, nullptr}, 0}, s);
}

template <typename T>
static int lr_step_go(const void* x, int64_t xs, const void* r, int64_t rs, const void* i, int64_t is, const void* z, int64_t zs,
                      const float* A, const float* state, float* new_state, void* y, int64_t total, int D, int act, int normalize,
                      hipStream_t s) {
  LAMPA_PROF(s, "start");
  hipLaunchKernelGGL((lr_step_kernel<T>), lr_grid((total + 255) / 256), dim3(256), 0, s, (const T*)x, xs, (const T*)r, rs,
                     (const T*)i, is, (const T*)z, zs, A, state, new_state, (T*)y, total, D, act, normalize);
  LAMPA_PROF(s, "lr_step_kernel");
  return lampa_launch_status();
}

extern "C" int lampa_lr_step(const void* x, int64_t x_stride, const void* decay_gate, int64_t decay_stride, const void* input_gate,
                             int64_t input_stride, const void* gate, int64_t gate_stride, const float* A, const float* state,
                             float* new_state, void* y, int64_t n, int D, int dtype, int activation, int normalize, void* stream) {
  if (!x || !decay_gate || !A || !state || !new_state || !y || n < 0 || D < 1 || activation < 0 || activation > 2) return LAMPA_ERR_INVALID;
  if (x_stride < D || decay_stride < D || (input_gate && input_stride < D) || (gate && gate_stride < D)) return LAMPA_ERR_INVALID;
  if (n > 0x7fffffffll * 256 / D) return LAMPA_ERR_UNSUPPORTED;
  if (n == 0) return LAMPA_OK;
  hipStream_t s = (hipStream_t)stream;
#define LR_STEP(T) \
  lr_step_go<T>(x, x_stride, decay_gate, decay_stride, input_gate, input_stride, gate, gate_stride, A, state, new_state, y, n * D, D, \
                activation, normalize, s)
  switch (dtype) {
    case GDR_BF16: return LR_STEP(__bf16);
    case GDR_FP16: return LR_STEP(_Float16);
    case GDR_FP32: return LR_STEP(float);
    default: return LAMPA_ERR_INVALID;
  }
#undef LR_STEP
}
