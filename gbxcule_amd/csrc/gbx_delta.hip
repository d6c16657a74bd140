// gbx_delta.hip -- the gated delta rule over whole rollouts and one step at a
// time.
#include "gbx_delta.h"

namespace gbx {
namespace {

#ifndef MINW
#define MINW 2
#define COLS(nt) (nt == 8 ? 2 : 2)
#endif
template <typename T, int NT, int VT, bool FULL>
struct Forward {
  using F = Factor<T>;
  DeltaArgs a;
  Unit<NT, VT> u;
  Steps<T, NT, FULL> q, k;
  Steps<T, VT, FULL> v;
  T* y;
  float *saved, *over;  // the states before the chunks, and u / beta of every step; may be NULL
  int64_t wide, lane;   // elements of a step of y; the lane's place in it
  f4 S[NT][VT];

  __device__ __forceinline__ Forward(const DeltaArgs& a_, const Unit<NT, VT>& u_)
      : a(a_),
        u(u_),
        q((const T*)a.q + u.env * a.q_env + u.head / a.share * a.q_head, a.q_step, a.keys, u.l),
        k((const T*)a.k + u.env * a.k_env + u.head / a.share * a.k_head, a.k_step, a.keys, u.l),
        v((const T*)a.v + u.env * a.v_env + u.head * a.v_head + u.first, a.v_step, a.values - u.first, u.l),
        wide((int64_t)a.envs * a.heads * a.values) {
    const int64_t unit = (int64_t)u.env * a.heads + u.head, heads = (int64_t)a.envs * a.heads;
    y = (T*)a.y + unit * a.values;
    lane = 4 * u.l.g * wide + u.col();
    saved = a.saved ? a.saved + unit * a.keys * a.values : nullptr;
    over = a.saved ? a.saved + (int64_t)((a.steps + kDeltaChunk - 1) / kDeltaChunk) * heads * a.keys * a.values + unit * a.values : nullptr;
  }
  __device__ __forceinline__ int64_t place() const { return ((int64_t)u.env * a.heads + u.head) * a.keys * a.values; }
  __device__ __forceinline__ void begin() {
    if (a.state) load_state<FULL>(a.state + place(), a, u, S);
    else clear_state(S);
  }
  __device__ __forceinline__ void keep(int t0) const {
    if (saved) store_state<FULL>(saved + (int64_t)(t0 / kDeltaChunk) * a.envs * a.heads * a.keys * a.values, a, u, S);
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
  __device__ __forceinline__ bool chunk(int t0, Lane l, const Solved<false>& z) {
    const Span s{0, z.steps};
    Raw<T> kr[NT], qr[NT], kc[NT], vc[VT];
    k.template rows<true>(t0, s, l, kr);
    q.template rows<true>(t0, s, l, qr);
    v.template cols<true>(t0, s, l, vc);
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
      for (int r = 0; r < NT; ++r) {
        const auto b = F::big(S[r][t]);
        x = mma(kr[r], b, x);
        Y[t] = mma(qr[r], b, Y[t]);
      }
      x = F::wide(vc[t]) - in * kin * x;
      E[t] = mma(T_row, x, zero4());
      fine = fine && finite4(E[t]);
    }
    if (!__all(fine)) return false;
    if (over) store(over, t0, s, l, E);
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      const f4 U = bin * E[t];
      Y[t] = mma(kq, F::fine(U), Y[t] * qin);
      const Fine<T> x = F::fine(U * tail);
#pragma unroll
      for (int r = 0; r < NT; ++r) S[r][t] = mma(kc[r], x, S[r][t] * all);
    }
    store(y, t0, s, l, Y);
    return true;
  }

  // The whole rollout span by span, and where a value is not finite step by step.
  __device__ __forceinline__ void carefully() {
    begin();
    for (int t0 = 0; t0 < a.steps; t0 += kDeltaChunk) {
      const Lane l = again(u.l);
      const Gates gates = load_gates(a, t0, u.env, u.head, l);
      keep(t0);
      int singles = 0;  // steps before this one go one by one
      for (int lo = 0; lo < gates.steps;) {
        const Span s{lo, lo < singles ? lo + 1 : next_cut(gates, lo)};
        if (cut_at(gates, lo)) clear_state(S);
        Raw<T> kr[NT], qr[NT], kc[NT], vc[VT];
        k.rows(t0, s, l, kr);
        q.rows(t0, s, l, qr);
        v.cols(t0, s, l, vc);
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
          for (int r = 0; r < NT; ++r) {
            const auto b = F::big(S[r][t]);
            x = mma(kr[r], b, x);
            Y[t] = mma(qr[r], b, Y[t]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = s.has(l.in(j)) ? vt[j] - d.in[j] * kin[j] * x[j] : 0.0f;
          E[t] = mma(T_.row, x, zero4());
          fine = fine && finite4(E[t]);
        }
        if (s.hi - s.lo > 1 && !__all(fine)) {
          singles = s.hi;
          continue;
        }
        if (over) store(over, t0, s, l, E);
        f4 kq = zero4();  // row c, places in(j): q_c . k_j
#pragma unroll
        for (int r = 0; r < NT; ++r) kq = mma(kr[r], qr[r], kq);
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
        store(y, t0, s, l, Y);
        lo = s.hi;
      }
    }
  }
};

// A workgroup is a head of an env, a wavefront some columns of its state.
template <typename T, int NT, int VT, bool FULL>
__global__ __launch_bounds__(512 / VT, MINW) void delta_kernel(DeltaArgs a) {
  __shared__ Solved<false> solved[kGroup];
  __shared__ int bad;
  // (a wavefront's number is the same in its lanes, which the compiler does not see)
  const int lane = threadIdx.x & 63, slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slabs = blockDim.x >> 6;
  const int64_t unit = block_id();
  if (unit >= (int64_t)a.envs * a.heads) return;
  Forward<T, NT, VT, FULL> w(a, Unit<NT, VT>{{lane & 15, lane >> 4}, (int)(unit / a.heads), (int)(unit % a.heads), slab * 16 * VT});
  if (threadIdx.x == 0) bad = 0;
  w.begin();
  bool fine = true;
  for (int t0 = 0; t0 < a.steps && fine; t0 += kGroup * kDeltaChunk) {
    const Lane l = again(w.u.l);
    const int chunks = (a.steps - t0 + kDeltaChunk - 1) / kDeltaChunk;
    for (int n = slab; n < kGroup && n < chunks; n += slabs) solve_chunk(a, t0 + n * kDeltaChunk, w.u.env, w.u.head, w.q, w.k, l, solved[n]);
    __syncthreads();
    for (int n = 0; n < kGroup && n < chunks && fine; ++n) fine = w.chunk(t0 + n * kDeltaChunk, again(w.u.l), solved[n]);
    if (!fine) bad = 1;
    __syncthreads();
    fine = !bad;  // nobody sets it again before the next barrier
  }
  if (!fine) w.carefully();
  store_state<FULL>(a.last + w.place(), a, w.u, w.S);
}

// One step: eight lanes hold 32 columns of a row of the state, eight groups of
// them the rows, R consecutive ones each; a wavefront takes 32 columns of a
// head.  With p = sum over rows of S k and w = that of S q, the state is read
// once, moved on in registers and written:
//   e = beta (v - a p),  S = a S + k e^T,  y = scale (a w + (q . k) e).
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
  load_row<R>((const T*)a.k + env * a.k_env + head / a.share * a.k_head + row, a.keys - row, k);
  load_row<R>((const T*)a.q + env * a.q_env + head / a.share * a.q_head + row, a.keys - row, q);
  load_row<4>((const T*)a.v + env * a.v_env + head * a.v_head + col, wide, v);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    load_row<4>(state + (int64_t)i * a.values, row + i < a.keys && !cut ? wide : 0, S[i]);
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
int64_t delta_work(const DeltaArgs&) { return 0; }

hipError_t launch_delta(const DeltaArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) {
      constexpr int kCols = COLS(nt);
      const int slabs = (a.values + 16 * kCols - 1) / (16 * kCols);
      by_truth(a.keys == 16 * nt && a.values % (16 * kCols) == 0, [&](auto full) {
        hipLaunchKernelGGL((delta_kernel<T, nt, kCols, full>), wide_grid((int64_t)a.envs * a.heads), dim3(64 * slabs), 0, st, a);
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
