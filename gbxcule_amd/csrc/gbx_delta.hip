// gbx_delta.hip -- the gated delta rule over whole rollouts and one step at a
// time.
#include "gbx_delta.h"

namespace gbx {
namespace {

// MAP: a piece of a rollout from zero, or from the identity, for what it makes of
// the state before it: no outputs but the state.
template <typename T, int NT, int VT, bool FULL, bool MAP>
struct Forward {
  using F = Factor<T>;
  DeltaArgs a;
  Unit<NT, VT> u;
  Steps<T, NT, FULL> q, k;
  Steps<T, VT, FULL> v;
  T* y;
  float *saved, *over;  // the states before the chunks, and u / beta of every step; may be NULL
  int64_t wide, lane;   // elements of a step of y; the lane's place in it
  const float* start;   // NULL: zeros, or the identity
  int from, upto;       // steps
  bool identity;        // columns are those of the identity, and there is no v
  f4 S[NT][VT];

  __device__ __forceinline__ Forward(const DeltaArgs& a_, const Unit<NT, VT>& u_, const float* start_, int from_, int upto_, bool identity_)
      : a(a_),
        u(u_),
        q((const T*)a.q + u.env * a.q_env + u.head / a.share * a.q_head, a.q_step, a.keys, u.l),
        k((const T*)a.k + u.env * a.k_env + u.head / a.share * a.k_head, a.k_step, a.keys, u.l),
        v((const T*)a.v + u.env * a.v_env + u.head * a.v_head + u.first, a.v_step, a.values - u.first, u.l),
        wide((int64_t)a.envs * a.heads * a.values),
        start(start_),
        from(from_),
        upto(upto_),
        identity(identity_) {
    const int64_t unit = (int64_t)u.env * a.heads + u.head, heads = (int64_t)a.envs * a.heads;
    y = (T*)a.y + unit * a.values;
    lane = 4 * u.l.g * wide + u.col();
    saved = a.saved ? a.saved + unit * a.keys * a.values : nullptr;
    over = a.saved ? a.saved + (int64_t)((a.steps + kDeltaChunk - 1) / kDeltaChunk) * heads * a.keys * a.values + unit * a.values : nullptr;
  }
  __device__ __forceinline__ void begin() {
    if (start) load_state<FULL>(start, a, u, S);
    else clear_state(S);
    if (MAP && identity) {
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) S[r][t][j] = NT * u.l.in(j) + r == u.col() + t ? 1.0f : 0.0f;
    }
  }
  __device__ __forceinline__ void values(int t0, Span s, Lane l, Raw<T> (&vc)[VT], bool keep) const {
    if (MAP && identity) {
#pragma unroll
      for (int t = 0; t < VT; ++t) vc[t] = Raw<T>{};
    } else if (keep) {
      v.template cols<true>(t0, s, l, vc);
    } else {
      v.cols(t0, s, l, vc);
    }
  }
  __device__ __forceinline__ void keep(int t0) const {
    if (!MAP && saved) store_state<FULL>(saved + (int64_t)(t0 / kDeltaChunk) * a.envs * a.heads * a.keys * a.values, a, u, S);
  }
  template <typename P>
  __device__ __forceinline__ void store(P* p, int t0, Span s, Lane l, const f4 (&v)[VT]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) x[t] = v[t][j];
      store_row<VT>((p + (t0 + j) * wide) + lane, opaque(s.has(l.in(j)) ? FULL ? VT : a.values - u.col() : 0), x);
    }
  }

  // A chunk whose system is solved.  False, and the state as it was, if a value is
  // not finite: in a product zero times infinity would reach earlier steps, too.
  // What it begins with has been loaded, and is loaded for the next one as soon
  // as it is used.
  struct First {
    Raw<T> kr[NT], qr[NT], vc[VT];
  };
  __device__ __forceinline__ void load(First& f, int t0, Lane l) const {
    const Span s{0, a.steps - t0 < kDeltaChunk ? a.steps - t0 : kDeltaChunk};
    k.template rows<true>(t0, s, l, f.kr);
    if (!MAP) q.template rows<true>(t0, s, l, f.qr);
    values(t0, s, l, f.vc, true);
  }
  __device__ __forceinline__ bool chunk(First& f, int t0, Lane l, const Solved<false>& z) {
    const Span s{0, z.steps};
    auto &kr = f.kr, &qr = f.qr;
    auto& vc = f.vc;
    Raw<T> kc[NT];
    k.template cols<true>(t0, s, l, kc);
    keep(t0);
    const f4 bin = of_rows(z.beta, l), kin = of_rows(z.kap, l), in = of_rows(z.in, l), qin = of_rows(z.qap, l) * in, tail = of_rows(z.tail, l) * kin;
    const f4 T_row = z.t[16 * l.g + l.c];
    const Fine<T> kq = F::fine(z.m[16 * l.g + l.c]);
    const float all = z.all;
    f4 E[VT], Y[VT];
    bool fine = true;
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      f4 x = zero4();
      Y[t] = zero4();
#pragma unroll
      for (int r = 0; r < NT; r += 2) {
        const auto b = two(F::fine(S[r][t]), F::fine(S[r + 1][t]));
        x = mma(two(kr[r], kr[r + 1]), b, x);
        if (!MAP) Y[t] = mma(two(qr[r], qr[r + 1]), b, Y[t]);
      }
      x = F::wide(vc[t]) - in * kin * x;
      E[t] = mma(T_row, x, zero4());
      fine = fine && finite4(bin * E[t]);
    }
    if (!__all(fine)) return false;
    load(f, t0 + kDeltaChunk < upto ? t0 + kDeltaChunk : t0, l);
    if (!MAP && over) store(over, t0, s, l, E);
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      const f4 U = bin * E[t];
      if (!MAP) Y[t] = mma(kq, F::fine(U), left_of(Y[t], qin));
      const Fine<T> x = F::fine(U * tail);
#pragma unroll
      for (int r = 0; r < NT; ++r) S[r][t] = mma(kc[r], x, S[r][t] * all);
    }
    if (!MAP) store(y, t0, s, l, Y);
    return true;
  }

  // The whole rollout span by span, and where a value is not finite step by step.
  __device__ __forceinline__ void carefully() {
    begin();
    for (int t0 = from; t0 < upto; t0 += kDeltaChunk) {
      const Lane l = again(u.l);
      const Gates gates = load_gates(a, t0, u.env, u.head, l);
      int singles = 0;  // steps before this one go one by one
      for (int lo = 0; lo < gates.steps;) {
        const Span s{lo, lo < singles ? lo + 1 : next_cut(gates, lo)};
        if (cut_at(gates, lo)) clear_state(S);
        // (a state that nothing of the chunk sees is kept as zeros: the gradient multiplies what is kept, and only then decays it)
        if (lo == 0) keep(t0);
        Raw<T> kr[NT], qr[NT], kc[NT], vc[VT];
        k.rows(t0, s, l, kr);
        q.rows(t0, s, l, qr);
        values(t0, s, l, vc, false);
        k.cols(t0, s, l, kc);
        const float beta = s.has(l.c) ? gates.beta : 0.0f;
        const f4 kk = square_of(kr);
        const float kap = unit_of(kk, a.normalize, l), qap = (a.normalize ? unit_of(square_of(qr), true, l) : 1.0f) * a.scale;
        const f4 bin = across(beta, l), kin = across(kap, l), qin = across(qap, l);
        const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
        const Both T_ = solve<false>(kk * (kap * kin) * d.pair, beta, bin, l);
        f4 E[VT], Y[VT];
        bool fine = true;
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          f4 x = zero4();
          Y[t] = zero4();
          const f4 vt = F::wide(vc[t]);
#pragma unroll
          for (int r = 0; r < NT; r += 2) {
            const auto b = two(F::fine(S[r][t]), F::fine(S[r + 1][t]));
            x = mma(two(kr[r], kr[r + 1]), b, x);
            Y[t] = mma(two(qr[r], qr[r + 1]), b, Y[t]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = s.has(l.in(j)) ? vt[j] - d.in[j] * kin[j] * x[j] : 0.0f;
          E[t] = mma(T_.row, x, zero4());
          fine = fine && finite4(bin * E[t]);
        }
        if (s.hi - s.lo > 1 && !__all(fine)) {
          singles = s.hi;
          continue;
        }
        if (!MAP && over) store(over, t0, s, l, E);
        f4 kq = product_of(kr, qr);  // row c, places in(j): q_c . k_j
#pragma unroll
        for (int j = 0; j < 4; ++j) kq[j] = l.in(j) <= l.c ? kq[j] * (qap * kin[j]) * d.pair[j] : 0.0f;
        const Fine<T> kqf = F::fine(kq);
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          f4 U;
#pragma unroll
          for (int j = 0; j < 4; ++j) U[j] = s.has(l.in(j)) ? bin[j] * E[t][j] : 0.0f;
          Y[t] = mma(kqf, F::fine(U), Y[t] * (qin * d.in));
          const Fine<T> x = F::fine(U * (d.tail * kin));
#pragma unroll
          for (int r = 0; r < NT; ++r) S[r][t] = mma(kc[r], x, S[r][t] * d.all);
        }
        if (!MAP) store(y, t0, s, l, Y);
        lo = s.hi;
      }
    }
  }
};

// A workgroup is a head of an env, or a piece of its steps, a wavefront some columns
// of its state.  MAP: of what the pieces (all but the last) make of the state
// before them: `ends` of N (the first from the rollout's own state, the others from
// zero) or, from the identity, of M (none for the first), so that a piece ends with M S + N.
template <typename T, int NT, int VT, bool FULL, bool MAP>
__global__ __launch_bounds__(512 / VT, 2) void delta_kernel(DeltaArgs a, float* ends, int identity) {
  __shared__ Solved<false> solved[kGroup];
  __shared__ int bad;
  // (a wavefront's number is the same in its lanes, which the compiler does not see)
  const int lane = threadIdx.x & 63, slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slabs = blockDim.x >> 6;
  const int64_t block = block_id(), units = (int64_t)a.envs * a.heads, unit = block % units, size = (int64_t)a.keys * a.values;
  const int piece = (int)(block / units) + (MAP ? identity : 0);
  if (piece >= a.pieces - (MAP ? 1 : 0)) return;
  int from = piece * a.piece_steps, upto = piece + 1 < a.pieces ? from + a.piece_steps : a.steps;
  const float* start = a.state ? a.state + unit * size : nullptr;
  if (MAP && piece > 0) {
    start = nullptr;
  } else if (!MAP && a.pieces > 1) {
    bool whole = false;  // not in pieces: a value is not finite that a product would spread
    for (int n = 0; n < slabs; ++n) whole = whole || a.flags[2 * (a.pieces - 1) * units + unit * slabs + n] != 0;
    if (whole && piece > 0) return;
    if (whole) upto = a.steps;
    if (piece > 0) start = a.starts + ((piece - 1) * units + unit) * size;
  }
  Forward<T, NT, VT, FULL, MAP> w(a, Unit<NT, VT>{{lane & 15, lane >> 4}, (int)(unit / a.heads), (int)(unit % a.heads), slab * 16 * VT}, start, from, upto, MAP && identity);
  if (threadIdx.x == 0) bad = 0;
  w.begin();
  typename Forward<T, NT, VT, FULL, MAP>::First ahead;
  w.load(ahead, from, w.u.l);
  bool fine = true;
  for (int t0 = from; t0 < upto && fine; t0 += kGroup * kDeltaChunk) {
    const Lane l = again(w.u.l);
    const int chunks = (upto - t0 + kDeltaChunk - 1) / kDeltaChunk;
    for (int n = slab; n < kGroup && n < chunks; n += slabs) solve_chunk(a, t0 + n * kDeltaChunk, w.u.env, w.u.head, w.q, w.k, l, solved[n]);
    __syncthreads();
    for (int n = 0; n < kGroup && n < chunks && fine; ++n) fine = w.chunk(ahead, t0 + n * kDeltaChunk, again(w.u.l), solved[n]);
    if (!fine) bad = 1;
    __syncthreads();
    fine = !bad;  // nobody sets it again before the next barrier
  }
  if (!fine) w.carefully();
  if constexpr (MAP) {
    store_state<FULL>(ends + (piece * units + unit) * size, a, w.u, w.S);
    fine = true;
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int t = 0; t < VT; ++t) fine = fine && finite4(w.S[r][t]);
    const int all = __syncthreads_and(fine);
    if (threadIdx.x == 0) a.flags[(identity * (a.pieces - 1) + piece) * units + unit] = !all;
  } else if (upto == a.steps) {
    store_state<FULL>(a.last + unit * size, a, w.u, w.S);
  }
}

// The states that pieces start from, one after the other: S = M S + N in N's place.
// A wavefront takes 16 columns; bound by a piece's M, loaded and multiplied behind the
// one before it (8,192 steps of 8 heads of 64 x 64 in 26 pieces: 61 us).  Flags, of N's and M's pieces before: of the columns after.
template <int NT, bool FULL>
__global__ __launch_bounds__(64) void delta_join_kernel(DeltaArgs a, int slabs) {
  const int lane = threadIdx.x & 63;
  const int64_t block = block_id(), units = (int64_t)a.envs * a.heads, unit = block / slabs, size = (int64_t)a.keys * a.values;
  if (unit >= units) return;
  const Unit<NT, 1> u{{lane & 15, lane >> 4}, 0, 0, (int)(block % slabs) * 16};
  const int pieces = a.pieces - 1;
  bool fine = true;
  for (int p = lane; p < pieces; p += 64) fine = fine && !a.flags[p * units + unit] && (p == 0 || !a.flags[(pieces + p) * units + unit]);
  fine = __all(fine);
  f4 S[NT][1], N[NT][1];
  load_state<FULL>(a.starts + unit * size, a, u, S);
  for (int p = 1; p < pieces && fine; ++p) {
    const float* M = a.maps + (p * units + unit) * a.keys * a.keys;
    load_state<FULL>(a.starts + (p * units + unit) * size, a, u, N);
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      const int row = NT * u.l.c + r, col = 4 * NT * u.l.g;
      Words<float, 4 * NT> x;
      if constexpr (FULL) x = load_whole<4 * NT>(M + row * a.keys + col);
      else x = load_words<4 * NT>(M + row * a.keys + col, row < a.keys ? a.keys - col : 0);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f4 m;
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = __uint_as_float(x.w[NT * j + n]);
        N[r][0] = mma(m, S[n][0], N[r][0]);
      }
    }
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      S[r][0] = N[r][0];
      fine = fine && finite4(S[r][0]);
    }
    fine = __all(fine);
    store_state<FULL>(a.starts + (p * units + unit) * size, a, u, S);
  }
  if (lane == 0) a.flags[2 * pieces * units + block] = !fine;
}

// One step: eight lanes hold 32 columns of a row of the state, eight groups of
// them the rows, R consecutive ones each; a wavefront takes 32 columns of a
// head.  With p = sum over rows of S k and w = that of S q, the state is read
// once, moved on in registers and written:
//   e = beta (v - a p),  S = a S + k e^T,  y = scale (a w + (q . k) e).
// Bound by reading and writing the state: 8,192 envs x 4 heads of 64 x 64 in 203 us,
// 5.4 TB/s (a copy to other memory reaches 4.9).  64 envs take 6.9 us, the kernel 6.1
// where one that is no more than a launch takes 3.2: a wavefront's own chain, the state's
// loads behind the gate's and the episode start's and sums over rows behind those,
// in 128 workgroups, which leave half of the compute units without one.
template <typename T, int R>
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaArgs a, int slabs, int64_t units) {
  const int lane = threadIdx.x & 63, g = lane >> 3, c = lane & 7;
  const int64_t unit = block_id() * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int env = (int)(unit / slabs / a.heads), head = (int)(unit / slabs % a.heads);
  const int col = (int)(unit % slabs) * 32 + 4 * c, wide = a.values - col, row = g * R;
  float* state = a.last + (((int64_t)env * a.heads + head) * a.keys + row) * a.values + col;
  const float gate = a.gate[env * a.gate_env + head], beta = a.beta[env * a.beta_env + head];
  const bool cut = (a.resets && a.resets[env]) || gate < kClosed;
  float k[R], q[R], v[4], S[R][4];
  load_floats<R>((const T*)a.k + env * a.k_env + head / a.share * a.k_head + row, a.keys - row, k);
  load_floats<R>((const T*)a.q + env * a.q_env + head / a.share * a.q_head + row, a.keys - row, q);
  load_floats<4>((const T*)a.v + env * a.v_env + head * a.v_head + col, wide, v);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    load_floats<4>(state + (int64_t)i * a.values, row + i < a.keys && !cut ? wide : 0, S[i]);
  }
  float p[4] = {}, w[4] = {}, kk = 0.0f, qq = 0.0f, qk = 0.0f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      p[n] = fmaf(S[i][n], k[i], p[n]);
      w[n] = fmaf(S[i][n], q[i], w[n]);
    }
    kk = fmaf(k[i], k[i], kk);
    qq = fmaf(q[i], q[i], qq);
    qk = fmaf(q[i], k[i], qk);
  }
  auto rows = [](float x) {
#pragma unroll
    for (int m = 8; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
    return x;
  };
  kk = rows(kk), qq = rows(qq), qk = rows(qk);
  const float kap = a.normalize ? rsqrtf(kk + kUnitEps) : 1.0f, qap = (a.normalize ? rsqrtf(qq + kUnitEps) : 1.0f) * a.scale;
  const float keep = cut ? 0.0f : exp2_fast(kLog2e * gate);
  float y[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float e = beta * fmaf(-keep * kap, rows(p[n]), v[n]);
    y[n] = qap * fmaf(keep, rows(w[n]), kap * qk * e);
#pragma unroll
    for (int i = 0; i < R; ++i) S[i][n] = fmaf(kap * k[i], e, keep * S[i][n]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) store_row<4>(state + (int64_t)i * a.values, row + i < a.keys ? wide : 0, S[i]);
  if (g == 0) store_row<4>((T*)a.y + ((int64_t)env * a.heads + head) * a.values + col, wide, y);
}

}  // namespace

int64_t delta_saved(const DeltaArgs& a) {
  const int64_t heads = (int64_t)a.envs * a.heads;
  return ((int64_t)(a.steps + kDeltaChunk - 1) / kDeltaChunk * a.keys + a.steps) * heads * a.values;
}
namespace {

// Few heads and many steps are cut into pieces that run side by side: what each
// makes of the state before it (two passes of the recurrence, over the values'
// and over the keys' columns), the states one after the other, and the pieces again
// from those: 8,192 steps of 8 heads of 64 x 64 in 187 us, of which the maps are 74
// and the last pass 54; one after the other 1,568.  More pieces make the passes shorter and the join longer, which
// takes about two thirds of a chunk's time a piece.
DeltaArgs in_pieces(DeltaArgs a) {
  const int64_t units = (int64_t)a.envs * a.heads, waves = units * slabs_of(a.values, 1), chunks = (a.steps + kDeltaChunk - 1) / kDeltaChunk;
  int64_t pieces = 1;
  while (pieces * waves < 2 * kManyWaves && pieces * pieces < chunks + chunks / 2) ++pieces;
  const int64_t each = ((chunks + pieces - 1) / pieces + kGroup - 1) / kGroup * kGroup;
  pieces = (chunks + each - 1) / each;
  a.pieces = 1, a.piece_steps = a.steps;
  if (pieces < 4) return a;
  a.pieces = (int)pieces, a.piece_steps = (int)each * kDeltaChunk;
  a.starts = a.work;
  a.maps = a.starts + (pieces - 1) * units * a.keys * a.values;
  a.flags = reinterpret_cast<int32_t*>(a.maps + (pieces - 1) * units * a.keys * a.keys);
  return a;
}

}  // namespace

int64_t delta_work(const DeltaArgs& args) {
  const DeltaArgs a = in_pieces(args);
  const int64_t units = (int64_t)a.envs * a.heads, pieces = a.pieces - 1;
  return pieces ? pieces * units * a.keys * (a.values + a.keys) + 2 * pieces * units + units * slabs_of(a.values, 1) : 0;
}

hipError_t launch_delta(const DeltaArgs& args, hipStream_t st) {
  const DeltaArgs a = in_pieces(args);
  DeltaArgs turned = a;  // M has as many columns as rows
  turned.values = a.keys;
  const int64_t units = (int64_t)a.envs * a.heads;
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) {
      if (a.pieces == 1) {
        by_columns<2>(a, [&](auto cols) {
          by_truth(a.keys == 16 * nt && a.values % (16 * cols) == 0, [&](auto full) {
            hipLaunchKernelGGL((delta_kernel<T, nt, cols, full, false>), wide_grid(units), dim3(64 * slabs_of(a.values, cols)), 0, st, a, nullptr, 0);
          });
        });
        return;
      }
      by_truth(a.keys == 16 * nt && a.values % 16 == 0, [&](auto full) {
        const int slabs = slabs_of(a.values, 1);
        hipLaunchKernelGGL((delta_kernel<T, nt, 1, full, true>), wide_grid((a.pieces - 1) * units), dim3(64 * slabs), 0, st, a, a.starts, 0);
        by_truth(a.keys == 16 * nt, [&](auto square) {
          hipLaunchKernelGGL((delta_kernel<T, nt, 1, square, true>), wide_grid((a.pieces - 2) * units), dim3(64 * slabs_of(a.keys, 1)), 0, st, turned, a.maps, 1);
        });
        hipLaunchKernelGGL((delta_join_kernel<nt, full>), wide_grid(units * slabs), dim3(64), 0, st, a, slabs);
        hipLaunchKernelGGL((delta_kernel<T, nt, 1, full, false>), wide_grid(a.pieces * units), dim3(64 * slabs), 0, st, a, nullptr, 0);
      });
    });
  });
  return hipGetLastError();
}

hipError_t launch_delta_step(const DeltaArgs& a, hipStream_t st) {
  const int slabs = (a.values + 31) / 32;
  const int64_t units = (int64_t)a.envs * a.heads * slabs;
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) { hipLaunchKernelGGL((delta_step_kernel<T, 2 * nt>), wide_grid((units + 3) / 4), dim3(256), 0, st, a, slabs, units); });
  });
  return hipGetLastError();
}

}  // namespace gbx
