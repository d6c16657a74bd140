// gbx_delta.h -- the gated delta rule in chunks: what its forward pass and its
// gradient share.
//
//   S = a S,  e = beta (v - S^T k),  S += k e^T,  y = scale S^T q,   a = exp(gate)
//
// with S = 0 before a step where an episode begins.  A chunk of 16 steps is
// solved at once.  G_i sums the gates of its steps up to i, g_i = exp(G_i) is
// what is left of the state S0 from before it, G_ij = exp(G_i - G_j), and the
// corrections u = (e_i) solve a triangular system:
//
//   (1 + L) u = rhs,  rhs_i = beta_i (v_i - g_i S0^T k_i),  L_ij = beta_i G_ij (k_i . k_j) for j < i
//   y_i = scale (g_i S0^T q_i + sum over j <= i of G_ij (q_i . k_j) u_j)
//   S   = g_15 S0 + sum over j of G_15,j k_j u_j^T
//
// Everything is products of 16-wide tiles on the matrix cores.  A tile that
// such a product makes has four consecutive rows in each lane and a column
// for each of 16 lanes; a factor needs four consecutive places of the summed
// index in each lane, and a row (left) or a column (right) for each of 16
// lanes.  So a product is the next one's right factor as it is, and, read as
// its transpose, the next one's left factor: the state, the corrections and
// the solved system never leave the registers.
//
// Which channel a row or column stands for is free, and chosen so that a
// lane's channels lie one after the other in memory.
//
// A wavefront takes a head of an env and some columns of its state (columns do
// not depend on each other).  Episodes that begin inside a chunk, and gates
// that close, cut it into segments, solved one after the other: nothing of
// what is before a cut takes part in a product behind it, finite or not.
#pragma once
#include <type_traits>

#include "gbx_policy.h"

namespace gbx {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// exp() of a gate below this is zero in 32 bits: it clears the state as an
// episode's start does.
constexpr float kClosed = -104.0f;
constexpr float kUnitEps = 1e-6f;  // added to a squared length before its root

// d += a b, 16 x 16 x 16 in 32 bits
__device__ __forceinline__ f4 mma(f4 a, f4 b, f4 d) {
#pragma unroll
  for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], d, 0, 0, 0);
  return d;
}
__device__ __forceinline__ f4 zero4() { return f4{0.0f, 0.0f, 0.0f, 0.0f}; }

struct Lane {
  int c, g;  // place among 16 lanes (a row or column), group of 16 (four places of the other index)
  __device__ __forceinline__ int in(int j) const { return 4 * g + j; }
};

// A lane's value of the row in(j), given each row's in the lanes c.
__device__ __forceinline__ f4 across(float own, Lane l) {
  f4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __shfl(own, l.in(j), 16);
  return v;
}

// The steps of a chunk from `lo` to before `hi`.
struct Span {
  int lo, hi;
  __device__ __forceinline__ bool has(int t) const { return t >= lo && t < hi; }
};

// Rows of q or k: 4 * NT channels of step c each, tile r's place in(j) channel
// NT * in(j) + r.
template <int NT, typename T>
__device__ __forceinline__ void load_rows(const T* p, int64_t step, int channels, Span s, Lane l, f4 (&v)[NT]) {
  float x[4 * NT];
  load_row<4 * NT>(p + l.c * step + 4 * NT * l.g, s.has(l.c) ? channels - 4 * NT * l.g : 0, x);
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[r][j] = x[NT * j + r];
}
// Columns: NT channels from NT * c on of each step in(j); of q, k, v or dy.
template <int NT, typename T>
__device__ __forceinline__ void load_cols(const T* p, int64_t step, int channels, Span s, Lane l, f4 (&v)[NT]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x[NT];
    load_row<NT>(p + l.in(j) * step + NT * l.c, s.has(l.in(j)) ? channels - NT * l.c : 0, x);
#pragma unroll
    for (int r = 0; r < NT; ++r) v[r][j] = x[r];
  }
}

// 1 / length of row c, which the four groups hold a quarter each of.
template <int NT>
__device__ __forceinline__ float unit_of(const f4 (&row)[NT], bool normalize) {
  float ss = 0.0f;
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = fmaf(row[r][j], row[r][j], ss);
  ss += __shfl_xor(ss, 16, 64);
  ss += __shfl_xor(ss, 32, 64);
  return normalize ? rsqrtf(ss + kUnitEps) : 1.0f;
}

// What is left of a value after the gates between two steps.  The sums are in
// 64 bits: those of two neighbouring steps may be long and their difference short.
struct Decay {
  float all;  // over the span
  f4 in;      // from before the span to in(j)
  f4 tail;    // from in(j) to the end
  f4 pair;    // between in(j) and c, from the earlier to the later
};
// `gate`: step c's, in powers of two, zero outside of the span
__device__ __forceinline__ Decay decay_of(double gate, Lane l) {
  double sum = gate;
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    const double o = __shfl_up(sum, m, 16);
    sum += l.c >= m ? o : 0.0;
  }
  const double end = __shfl(sum, 15, 16);
  Decay d;
  d.all = exp2_fast((float)end);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double o = __shfl(sum, l.in(j), 16);
    d.in[j] = exp2_fast((float)o);
    d.tail[j] = exp2_fast((float)(end - o));
    d.pair[j] = exp2_fast((float)(l.in(j) < l.c ? sum - o : o - sum));
  }
  return d;
}

template <int LANE>
__device__ __forceinline__ float quad_lane(float v) {  // of the four lanes around
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), LANE * 0x55, 0xF, 0xF, true));
}

// The inverse of 1 + L, L strictly lower triangular; `row`: row c, places
// in(j); `col`: column c, rows in(j).  Substitution within blocks of four,
// whose rows are four neighbouring lanes, then twice
//   [A 0; M B]^-1 = [A^-1 0; -B^-1 M A^-1, B^-1],
// which for all blocks at once is T - T M T.  (The sum of L's powers would be
// fewer products, but where keys repeat, as they do while a screen stands
// still, its terms are thousands of times the result.)
struct Both {
  f4 row, col;
};
__device__ __forceinline__ Both inverse(Both L, Lane l) {
  const int b = l.c >> 2, n = l.c & 3;
  f4 ar, ac, lr, lc;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ar[j] = ac[j] = l.g == b && j == n ? 1.0f : 0.0f;
    lr[j] = l.g == b ? L.row[j] : 0.0f;
    lc[j] = l.g == b ? L.col[j] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[0], quad_lane<0>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[1], quad_lane<1>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[2], quad_lane<2>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[3], quad_lane<3>(ac[j]), ac[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[2], quad_lane<2>(ac[j]), ac[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[1], quad_lane<1>(ac[j]), ac[j]);
  f4 m8, m16;  // minus M: pairs of blocks, then of pairs
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m8[j] = b == l.g + 1 && (b & 1) ? -L.row[j] : 0.0f;
    m16[j] = b >= 2 && l.g < 2 ? -L.row[j] : 0.0f;
  }
  f4 x = mma(m8, ac, zero4());
  Both t{mma(x, ar, ar), mma(ar, x, ac)};
  x = mma(m16, t.col, zero4());
  return {mma(x, t.row, t.row), mma(t.row, x, t.col)};
}

// A head of an env, some columns of its state, and the lane's part in them.
template <int NT, int VT>
struct Unit {
  Lane l;
  int env, head, first;  // first column
  __device__ __forceinline__ int col() const { return first + VT * l.c; }
};

// State tiles: tile (r, t), place in(j): channel NT * in(j) + r, column VT * c + t.
template <int NT, int VT>
__device__ __forceinline__ void load_state(const float* p, const DeltaArgs& a, const Unit<NT, VT>& u, f4 (&s)[NT][VT]) {
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = NT * u.l.in(j) + r;
      float x[VT];
      load_row<VT>(p + (int64_t)row * a.values + u.col(), row < a.keys ? a.values - u.col() : 0, x);
#pragma unroll
      for (int t = 0; t < VT; ++t) s[r][t][j] = x[t];
    }
}
template <int NT, int VT>
__device__ __forceinline__ void store_state(float* p, const DeltaArgs& a, const Unit<NT, VT>& u, const f4 (&s)[NT][VT]) {
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = NT * u.l.in(j) + r;
      float x[VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) x[t] = s[r][t][j];
      store_row<VT>(p + (int64_t)row * a.values + u.col(), row < a.keys ? a.values - u.col() : 0, x);
    }
}
template <int NT, int VT>
__device__ __forceinline__ void clear_state(f4 (&s)[NT][VT]) {
#pragma unroll
  for (int r = 0; r < NT; ++r)
#pragma unroll
    for (int t = 0; t < VT; ++t) s[r][t] = zero4();
}

// Step c of a chunk.
struct Gates {
  int steps;      // of the chunk
  uint32_t cuts;  // steps that nothing from before reaches
  float beta;
  double gate;  // in powers of two; zero at a cut and outside
};
__device__ __forceinline__ Gates load_gates(const DeltaArgs& a, int t0, int env, int head, Lane l) {
  const int n = a.steps - t0 < kDeltaChunk ? a.steps - t0 : kDeltaChunk;
  const bool live = l.c < n;
  const int64_t t = t0 + l.c;
  const float gate = live ? a.gate[t * a.gate_step + env * a.gate_env + head] : 0.0f;
  const bool begins = live && a.resets && a.resets[t * a.envs + env];
  Gates r;
  r.steps = n;
  r.beta = live ? a.beta[t * a.beta_step + env * a.beta_env + head] : 0.0f;
  const bool cut = begins || gate < kClosed;
  r.cuts = (uint32_t)__ballot(cut) & 0xFFFFu;
  r.gate = cut ? 0.0 : (double)gate * 1.44269504088896340736;
  return r;
}
__device__ __forceinline__ int next_cut(const Gates& r, int lo) {
  const uint32_t later = r.cuts >> lo >> 1;
  return later ? lo + 1 + __builtin_ctz(later) : r.steps;
}
__device__ __forceinline__ bool cut_at(const Gates& r, int t) { return r.cuts >> t & 1u; }

// The triangular system of a span, with keys of unit length `kap` (row c) and `kin`.
struct System {
  Both T;    // inverse
  f4 plain;  // L without its betas, row c
};
template <int NT>
__device__ __forceinline__ System system_of(const f4 (&k)[NT], float kap, f4 kin, float beta, f4 bin, const Decay& d, Lane l) {
  f4 kk = zero4();
#pragma unroll
  for (int r = 0; r < NT; ++r) kk = mma(k[r], k[r], kk);
  System s;
  Both L;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float p = kk[j] * (kap * kin[j]) * d.pair[j];
    s.plain[j] = l.in(j) < l.c ? p : 0.0f;
    L.row[j] = l.in(j) < l.c ? beta * p : 0.0f;
    L.col[j] = l.in(j) > l.c ? bin[j] * p : 0.0f;
  }
  s.T = inverse(L, l);
  return s;
}

__device__ __forceinline__ bool finite4(f4 v) {
  const float z = v[0] * 0.0f + v[1] * 0.0f + v[2] * 0.0f + v[3] * 0.0f;
  return z == 0.0f;  // an infinity or NaN makes NaN
}

// f(tiles of the keys)
template <typename F>
void by_keys(int keys, F&& f) {
  if (keys <= 32) f(std::integral_constant<int, 2>{});
  else if (keys <= 64) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

}  // namespace
}  // namespace gbx
