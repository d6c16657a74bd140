// gbx_delta_grad.hip -- gradient of the gated delta rule.
//
// A chunk (see gbx_delta.h for its forward formulas and for how tiles lie in
// registers) is walked back from D, the gradient of the state after it, and
// S0, the state before it, which the forward pass has kept.  With K, Q, U as
// matrices of the chunk's rows, A_ij = scale G_ij (q_i . k_j) for j <= i and
// T = (1 + L)^-1:
//
//   du = A^T dy + G_15 (K D),  w = T^T du,  dv = beta w,  dbeta_i = w_i . (u_i / beta_i)
//   P_ij = scale G_ij (dy_i . u_j) for j <= i,  M_ij = -beta_i G_ij (w_i . u_j) for j < i
//   dq = scale g S0 dy + P K
//   dk = -g S0 dv + M K  +  G_15 D u + P^T Q + M^T K
//   D <- g_15 D + scale sum of g_i q_i dy_i^T - sum of g_i k_i dv_i^T
//
// u_i / beta_i is v_i - g_i S0^T k_i less the sum over j of L_ij u_j / beta_i,
// which needs no division.  A gate counts in everything between an earlier
// and a later step: with "reads" the terms of dq and of dk before the gap above
// and "writes" those behind it,
//   dgate_i = <S, D> after the chunk + sum over m >= i of (q . dq + k . dk_reads - k . dk_writes)_m.
// The inner product is computed anew at the end of every chunk, so its error does not
// grow with the length of the rollout.
//
// D is needed both ways round, and registers hold one: it is turned in LDS.  S0 is
// needed with its columns summed alone, as <S, D> is taken apart into what the chunk
// wrote and what it kept, and is read so from what the forward pass kept.
#include "gbx_delta.h"

#include <algorithm>

namespace gbx {
namespace {

// The state with the summed index on its columns, channels NT * c + r: tile t,
// place in(j): column VT * in(j) + t.
template <bool FULL, int NT, int VT>
__device__ __forceinline__ void load_turned(const float* p, const DeltaArgs& a, const Unit<NT, VT>& u, int r, f4 (&s)[VT]) {
  const uint32_t at = (uint32_t)opaque((NT * u.l.c * a.values + u.first + 4 * VT * u.l.g) * 4);  // in bytes
  const float* from = (const float*)((uintptr_t)(p + r * a.values) + at);
  Words<float, 4 * VT> x;
  if constexpr (FULL) x = load_whole<4 * VT>(from);
  else x = load_words<4 * VT>(from, NT * u.l.c + r < a.keys ? a.values - u.first - 4 * VT * u.l.g : 0);
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[t][j] = __uint_as_float(x.w[VT * j + t]);
}

// The state before a span, both ways round: as the forward pass kept it,
// or nothing, read where it is used; or moved on from there, in registers.
template <int NT, int VT>
struct Kept {
  const float* p;  // NULL: zeros
};
template <int NT, int VT>
struct Moved {
  f4 S[NT][VT], St[NT][VT];
};

template <typename T, int NT, int VT, bool FULL>
struct Grad {
  using F = Factor<T>;
  DeltaArgs a;
  Unit<NT, VT> u;
  Lane l;
  Steps<T, NT, FULL> q, k;
  Steps<T, VT, FULL> v, dy;
  int t0;  // the chunk's first step
  T* dv;   // of that step
  int64_t dv_lane;
  float *tiles, *part;  // in LDS: dq and dk of the chunk's steps, this wavefront's columns' part; the lane's place
  Gates gates;
  f4 D[NT][VT];   // gradient of the state
  f4 Dt[NT][VT];  // the other way round; a chunk whose system is solved turns D in LDS

  __device__ __forceinline__ void state(const Kept<NT, VT>& from, f4 (&s)[NT][VT]) const {
    if (from.p) load_state<FULL>(from.p, a, u, s);
    else clear_state(s);
  }
  __device__ __forceinline__ void turned(const Kept<NT, VT>& from, int r, f4 (&s)[VT]) const {
    if (from.p) {
      load_turned<FULL>(from.p, a, u, r, s);
    } else {
#pragma unroll
      for (int t = 0; t < VT; ++t) s[t] = zero4();
    }
  }
  __device__ __forceinline__ void state(const Moved<NT, VT>& from, f4 (&s)[NT][VT]) const {
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int t = 0; t < VT; ++t) s[r][t] = from.S[r][t];
  }
  __device__ __forceinline__ void turned(const Moved<NT, VT>& from, int r, f4 (&s)[VT]) const {
#pragma unroll
    for (int t = 0; t < VT; ++t) s[t] = from.St[r][t];
  }

  // One step of the forward pass.
  __device__ __forceinline__ void advance(int t, Moved<NT, VT>& m) const {
    const Span s{t, t + 1};
    Raw<T> kr[NT], kc[NT], vc[VT];
    k.rows(t0, s, l, kr);
    k.cols(t0, s, l, kc);
    v.cols(t0, s, l, vc);
    const f4 bin = across(s.has(l.c) ? gates.beta : 0.0f, l), kin = across(unit_of(square_of(kr), a.normalize, l), l);
    const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      f4 x = zero4();
      const f4 vt = F::wide(vc[t]);
#pragma unroll
      for (int r = 0; r < NT; ++r) x = mma(kr[r], F::fine(m.S[r][t]), x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = s.has(l.in(j)) ? kin[j] * bin[j] * fmaf(-d.in[j] * kin[j], x[j], vt[j]) : 0.0f;
      const Fine<T> xf = F::fine(x);
#pragma unroll
      for (int r = 0; r < NT; ++r) {
        m.S[r][t] = mma(kc[r], xf, m.S[r][t] * d.all);
        m.St[r][t] = mma(xf, kc[r], m.St[r][t] * d.all);
      }
    }
  }

  // Walks a chunk back whose system is solved.  False, and nothing done, if a
  // value is not finite: in a product zero times infinity would reach steps that the
  // formulas keep from it.  Looked at is what the other products take: w, which all
  // that the system or D holds goes through, and u itself, whose first step no row
  // of the system has (its beta may be infinite, or u overflow, with u / beta finite;
  // a u / beta that is not finite makes u so for any beta).  The kept state is finite
  // where u is: where it is read, u has read it, and where it is not, it is zero.
  __device__ __forceinline__ bool chunk(const Solved<true>& z, const float* kept, const Steps<float, VT, FULL>& over, float& dgate, f4& dbeta) {
    const Span s{0, z.steps};
    const int lane = 16 * l.g + l.c;
    Raw<T> kr[NT], dyc[VT];
    Whole ec[VT], er[VT];  // u / beta
    k.template rows<true>(t0, s, l, kr);
    over.template cols<true>(t0, s, l, ec);
    over.template rows<true>(t0, s, l, er);
    dy.cols(t0, s, l, dyc);
    Raw<T> dyr[VT], kc[NT], qc[NT];
    f4 St[VT];
    dy.rows(t0, s, l, dyr);
    k.template cols<true>(t0, s, l, kc);
    q.template cols<true>(t0, s, l, qc);
    load_turned<FULL>(kept, a, u, 0, St);
    const f4 bin = of_rows(z.beta, l), kin = of_rows(z.kap, l), qin = of_rows(z.qap, l), in = of_rows(z.in, l), tail = of_rows(z.tail, l);
    const float beta = z.beta[l.c], all = z.all;
    // D goes through LDS to be read the other way round, tile (r, t) where dq's (t = 0) and dk's (t = 1) tile
    // r comes to lie afterwards.  Every other four rows lie two by two the other way, so that
    // 16 columns of four rows fall on all banks.
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) tiles[(t * NT + r) * 256 + (l.in(j) ^ (l.g & 1)) * 16 + l.c] = D[r][t][j];
    const int turned = (l.c ^ (l.c >> 2 & 1)) * 16 + 4 * l.g;
    f4 W[VT], Ut[VT], Wt[VT], bsum = zero4();  // Ut and Wt: rows c
    float whole = 0.0f;                        // <S, D> after the chunk: what it wrote, then what it kept
    {
      const f4 T_col = z.t[lane];
      const Fine<T> aq = F::fine(z.m[lane]);
      bool fine = true;
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        f4 x = zero4();
#pragma unroll
        for (int r = 0; r < NT; r += 2) x = mma(two(kr[r], kr[r + 1]), two(F::fine(D[r][t]), F::fine(D[r + 1][t])), x);
        x *= tail * kin;
        const f4 part = x * bin * ec[t].v;
        whole += (part[0] + part[1]) + (part[2] + part[3]);
        x = mma(aq, dyc[t], x);
        W[t] = mma(T_col, x, zero4());
        Wt[t] = mma(x, T_col, zero4());
        Ut[t] = er[t].v * beta;
        bsum += W[t] * ec[t].v;
        fine = fine && finite4(W[t]) && finite4(Ut[t]);
      }
      if (!__all(fine)) return false;
    }
    {  // dv, and what D takes up
      const f4 ask = a.scale * qin * in, give = -in * kin;
      float out[4][VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        const f4 v = bin * W[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j][t] = v[j];
        const auto takes = two(F::fine(ask * F::wide(dyc[t])), F::fine(give * v));
#pragma unroll
        for (int r = 0; r < NT; ++r) D[r][t] = mma(two(qc[r], kc[r]), takes, D[r][t] * all);
      }
      const int64_t v_step = (int64_t)a.envs * a.heads * a.values;
#pragma unroll
      for (int j = 0; j < 4; ++j) store_row<VT>((dv + j * v_step) + dv_lane, opaque(s.has(l.in(j)) ? FULL ? VT : a.values - u.col() : 0), out[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) dbeta[j] = row_sum(bsum[j]);
    Fine<T> Utf[VT], Wtf[VT], pf, mf, ptf, mtf;
#pragma unroll
    for (int t = 0; t < VT; ++t) Utf[t] = F::fine(Ut[t]), Wtf[t] = F::fine(Wt[t]);
    const auto Us = columns<VT>(Utf), Ws = columns<VT>(Wtf);
    const auto dys = columns<VT>(dyr);
    {
      const f4 pair = z.pair[lane];
      f4 p = mma(Us, dys, zero4()), pt = mma(dys, Us, zero4()), m = mma(Us, Ws, zero4()), mt = mma(Ws, Us, zero4());
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[j] = l.in(j) <= l.c ? left_of(p[j] * (a.scale * kin[j]), pair[j]) : 0.0f;
        pt[j] = l.in(j) < l.c ? 0.0f : left_of(pt[j] * (a.scale * qin[j]), pair[j]);
        m[j] = l.in(j) < l.c ? left_of(-m[j] * (beta * kin[j]), pair[j]) : 0.0f;
        mt[j] = l.in(j) <= l.c ? 0.0f : left_of(-mt[j] * (bin[j] * kin[j]), pair[j]);
      }
      pf = F::fine(p), ptf = F::fine(pt), mf = F::fine(m), mtf = F::fine(mt);
    }
    const auto writers = two(ptf, mtf);
    const f4 qs = a.scale * in, rs = -in * bin;
    f4 e = zero4();  // q . dq + k . dk_reads - k . dk_writes
    float held = 0.0f;
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      f4 next[VT];
      if (r + 1 < NT) load_turned<FULL>(kept, a, u, r + 1, next);
      Fine<T> sf[VT], df[VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        const f4 Dr = *reinterpret_cast<const f4*>(tiles + (t * NT + r) * 256 + turned);
        const f4 part = St[t] * Dr;
        held += (part[0] + part[1]) + (part[2] + part[3]);
        sf[t] = F::fine(St[t]), df[t] = F::fine(Dr);
        if (r + 1 < NT) St[t] = next[t];
      }
      const auto Ss = columns<VT>(sf), Ds = columns<VT>(df);
      const f4 x = mma(pf, kc[r], left_of(mma(dys, Ss, zero4()), qs));
      const f4 reads = mma(mf, kc[r], left_of(mma(Ws, Ss, zero4()), rs));
      const f4 writes = mma(writers, two(qc[r], kc[r]), left_of(mma(Us, Ds, zero4()), tail));
      e += qin * F::wide(qc[r]) * x + kin * F::wide(kc[r]) * (reads - writes);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        part[(r * 4 + j) * 64] = x[j];
        part[((NT + r) * 4 + j) * 64] = reads[j] + writes[j];
      }
    }
    whole = row_sum(whole + left_of(held, all));
    whole = from_lane(whole, l.c) + from_lane(whole, l.c + 16) + from_lane(whole, l.c + 32) + from_lane(whole, l.c + 48);
    float own = 0.0f;  // e of step c, then the sum from there to before the next cut
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float other = from_lane(row_sum(e[j]), (l.c & 12) * 4);
      own = (l.c & 3) == j ? other : own;
    }
    const uint32_t later = z.cuts >> l.c >> 1;
    const int far = later ? __builtin_ctz(later) + 1 : 16;
    float v = row_lane<kLeft + 1>(own);
    own += far > 1 ? v : 0.0f;
    v = row_lane<kLeft + 2>(own);
    own += far > 2 ? v : 0.0f;
    v = row_lane<kLeft + 4>(own);
    own += far > 4 ? v : 0.0f;
    v = row_lane<kLeft + 8>(own);
    own += far > 8 ? v : 0.0f;
    dgate = z.cuts >> l.c & 1u ? 0.0f : later ? own : own + whole;
    return true;
  }

  // Walks a span back, likewise.
  template <typename From>
  __device__ __forceinline__ bool back(Span s, const From& from, float& dgate, f4& dbeta) {
    Raw<T> kr[NT], qr[NT], kc[NT], qc[NT], dyr[VT], dyc[VT], vc[VT];
    k.rows(t0, s, l, kr);
    q.rows(t0, s, l, qr);
    v.cols(t0, s, l, vc);
    dy.cols(t0, s, l, dyc);
    const float beta = s.has(l.c) ? gates.beta : 0.0f;
    const f4 kk = square_of(kr);
    const float kap = unit_of(kk, a.normalize, l), qap = a.normalize ? unit_of(square_of(qr), true, l) : 1.0f;
    const f4 bin = across(beta, l), kin = across(kap, l), qin = across(qap, l);
    const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
    const f4 plain = kk * (kap * kin) * d.pair;
    const Both sys = solve<true>(plain, beta, bin, l);
    f4 aq = zero4();  // A^T: row c, places in(j) >= c
#pragma unroll
    for (int r = 0; r < NT; ++r) aq = mma(qr[r], kr[r], aq);
    f4 less;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      aq[j] = l.in(j) < l.c ? 0.0f : aq[j] * (kap * qin[j] * a.scale) * d.pair[j];
      less[j] = l.in(j) < l.c ? -plain[j] : 0.0f;
    }
    const Fine<T> aqf = F::fine(aq);

    f4 W[VT], over[VT];          // over: u / beta
    Fine<T> Utf[VT], Wtf[VT];    // rows c
    float whole = 0.0f;          // <S, D> after the span: what it wrote, then what it kept
    bool fine = true;
    {
      f4 S[NT][VT];
      state(from, S);
      float held = 0.0f;
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        f4 x = zero4(), rhs;
        const f4 vt = F::wide(vc[t]);
#pragma unroll
        for (int r = 0; r < NT; ++r) {
          x = mma(kr[r], F::fine(S[r][t]), x);
#pragma unroll
          for (int j = 0; j < 4; ++j) held = fmaf(S[r][t][j], D[r][t][j], held);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          over[t][j] = s.has(l.in(j)) ? fmaf(-d.in[j] * kin[j], x[j], vt[j]) : 0.0f;
          rhs[j] = s.has(l.in(j)) ? bin[j] * over[t][j] : 0.0f;
        }
        const f4 U = mma(sys.row, rhs, zero4());
        Utf[t] = F::fine(mma(rhs, sys.row, zero4()));
        over[t] = mma(less, U, over[t]);
        x = zero4();
#pragma unroll
        for (int r = 0; r < NT; ++r) x = mma(kr[r], F::fine(D[r][t]), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = s.has(l.in(j)) ? d.tail[j] * kin[j] * x[j] : 0.0f;
          whole = fmaf(x[j], U[j], whole);
        }
        x = mma(aqf, dyc[t], x);
        W[t] = mma(sys.col, x, zero4());
        Wtf[t] = F::fine(mma(x, sys.col, zero4()));
        fine = fine && finite4(U) && finite4(W[t]);
      }
      whole = fmaf(d.all, held, whole);
    }
    if (s.hi - s.lo > 1 && !__all(fine)) return false;

    dy.rows(t0, s, l, dyr);
    f4 p = zero4(), pt = zero4(), m = zero4(), mt = zero4();
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      p = mma(Utf[t], dyr[t], p);
      pt = mma(dyr[t], Utf[t], pt);
      m = mma(Utf[t], Wtf[t], m);
      mt = mma(Wtf[t], Utf[t], mt);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = l.in(j) <= l.c ? p[j] * (a.scale * kin[j]) * d.pair[j] : 0.0f;
      pt[j] = l.in(j) < l.c ? 0.0f : pt[j] * (a.scale * qin[j]) * d.pair[j];
      m[j] = l.in(j) < l.c ? -m[j] * (beta * kin[j]) * d.pair[j] : 0.0f;
      mt[j] = l.in(j) <= l.c ? 0.0f : -mt[j] * (bin[j] * kin[j]) * d.pair[j];
    }
    const Fine<T> pf = F::fine(p), ptf = F::fine(pt), mf = F::fine(m), mtf = F::fine(mt);
    // dv, dbeta, and what D takes up
    Fine<T> asks[VT], gives[VT];
    f4 bsum = zero4();
    float out[4][VT];
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      f4 x = F::wide(dyc[t]), y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bsum[j] = fmaf(W[t][j], over[t][j], bsum[j]);
        out[j][t] = bin[j] * W[t][j];
        x[j] *= a.scale * qin[j] * d.in[j];
        y[j] = -d.in[j] * kin[j] * out[j][t];
      }
      asks[t] = F::fine(x);
      gives[t] = F::fine(y);
    }
    const int64_t v_step = (int64_t)a.envs * a.heads * a.values;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      store_row<VT>((dv + j * v_step) + dv_lane, opaque(s.has(l.in(j)) ? FULL ? VT : a.values - u.col() : 0), out[j]);
      dbeta[j] = s.has(l.in(j)) ? row_sum(bsum[j]) : dbeta[j];
    }
    k.cols(t0, s, l, kc);
    q.cols(t0, s, l, qc);
    f4 e = zero4();  // q . dq + k . dk_reads - k . dk_writes
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      f4 x = zero4(), reads = zero4(), writes = zero4(), St[VT];
      turned(from, r, St);
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        const auto sf = F::fine(St[t]);
        x = mma(dyr[t], sf, x);
        reads = mma(Wtf[t], sf, reads);
        writes = mma(Utf[t], F::fine(Dt[r][t]), writes);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] *= a.scale * d.in[j];
        reads[j] *= -d.in[j] * bin[j];
        writes[j] *= d.tail[j];
      }
      x = mma(pf, kc[r], x);
      reads = mma(mf, kc[r], reads);
      writes = mma(ptf, qc[r], writes);
      writes = mma(mtf, kc[r], writes);
      const f4 qw = F::wide(qc[r]), kw = F::wide(kc[r]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = fmaf(qin[j] * qw[j], x[j], e[j]);
        e[j] = fmaf(kin[j] * kw[j], reads[j] - writes[j], e[j]);
        if (s.has(l.in(j))) {
          part[(r * 4 + j) * 64] = x[j];
          part[((NT + r) * 4 + j) * 64] = reads[j] + writes[j];
        }
      }
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        D[r][t] = mma(kc[r], gives[t], mma(qc[r], asks[t], D[r][t] * d.all));
        Dt[r][t] = mma(gives[t], kc[r], mma(asks[t], qc[r], Dt[r][t] * d.all));
      }
    }
    whole = row_sum(whole);
    whole = from_lane(whole, l.c) + from_lane(whole, l.c + 16) + from_lane(whole, l.c + 32) + from_lane(whole, l.c + 48);
    float own = 0.0f;  // e of step c, then the sum from there on
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float other = from_lane(row_sum(e[j]), (l.c & 12) * 4);
      own = (l.c & 3) == j && s.has(l.c) ? other : own;
    }
    own = sum_from(own);
    if (s.has(l.c)) dgate = cut_at(gates, l.c) ? 0.0f : whole + own;
    return true;
  }

  // The span one step at a time, each from the state moved on from `known`.
  __device__ __forceinline__ void back_singly(Span s, const Kept<NT, VT>& known, float& dgate, f4& dbeta) {
    for (int hi = s.hi; hi > s.lo; --hi) {
      Moved<NT, VT> m;
      state(known, m.S);
#pragma unroll
      for (int r = 0; r < NT; ++r) turned(known, r, m.St[r]);
      for (int t = s.lo; t < hi - 1; ++t) advance(t, m);
      back(Span{hi - 1, hi}, m, dgate, dbeta);
    }
  }
};

// The columns' parts of dq, dk, dgate and dbeta of a chunk, added in one order.
// lds: [slab][dq, dk][r][j][lane], then [slab][dgate, dbeta][step].  A thread's rows
// are loaded before the others' parts are waited for.
template <typename T, int NT, int VT, bool FULL>
struct Join {
  static constexpr int kPart = 2 * NT * 256;
  float q[NT], k[NT];  // of the thread's first turn
  __device__ __forceinline__ void load(const Grad<T, NT, VT, FULL>& w, int i, float (&q)[NT], float (&k)[NT]) const {
    const int c = i & 15, t = w.t0 + 4 * (i >> 4 & 3) + (i >> 6), rest = t < w.a.steps ? w.a.keys - NT * c : 0;
    load_floats<NT>(w.q.p + t * w.a.q_step + NT * c, rest, q);
    load_floats<NT>(w.k.p + t * w.a.k_step + NT * c, rest, k);
  }
  __device__ __forceinline__ void begin(const Grad<T, NT, VT, FULL>& w) { load(w, opaque(threadIdx.x), q, k); }
  __device__ __forceinline__ void end(const Grad<T, NT, VT, FULL>& w, int64_t unit, const float* lds, int slabs) {
    const DeltaArgs& a = w.a;
    const int t0 = w.t0, steps = a.steps - t0, first = opaque(threadIdx.x);  // (more steps than a chunk's do no harm)
    const int64_t heads = (int64_t)a.envs * a.heads;
    for (int i = first; i < 256; i += blockDim.x) {
      const int j = i >> 6, c = i & 15, t = 4 * (i >> 4 & 3) + j, rest = opaque(a.keys - NT * c);
      const bool live = t < steps;
      const int64_t row = (t0 + t) * heads + unit;
      if (i != first) load(w, i, q, k);
      auto turn = [&](const float (&x)[NT], int kind, void* to) {
        float dx[NT] = {}, ss = 0.0f, dot = 0.0f;
        for (int n = 0; n < slabs; ++n)
#pragma unroll
          for (int r = 0; r < NT; ++r) dx[r] += lds[n * kPart + ((kind * NT + r) * 4 + j) * 64 + (i & 63)];
        if (a.normalize) {  // x / length: the gradient's part along x goes
#pragma unroll
          for (int r = 0; r < NT; ++r) {
            ss = fmaf(x[r], x[r], ss);
            dot = fmaf(x[r], dx[r], dot);
          }
          const float unit_x = rsqrtf(row_sum(ss) + kUnitEps);
          dot = row_sum(dot) * (unit_x * unit_x);
#pragma unroll
          for (int r = 0; r < NT; ++r) dx[r] = unit_x * fmaf(-x[r], dot, dx[r]);
        }
        if (a.share == 1) store_row<NT>((T*)to + row * a.keys + NT * c, live ? rest : 0, dx);
        else store_row<NT>((float*)to + row * a.keys + NT * c, live ? rest : 0, dx);
      };
      turn(q, 0, a.share == 1 ? a.dq : a.work);
      turn(k, 1, a.share == 1 ? a.dk : a.work + a.steps * heads * a.keys);
      if (i < 2 * kDeltaChunk && (i & 15) < steps) {
        float x = 0.0f;
        for (int n = 0; n < slabs; ++n) x += lds[slabs * kPart + n * 2 * kDeltaChunk + i];
        (i < kDeltaChunk ? a.dgate : a.dbeta)[(t0 + (i & 15)) * heads + unit] = x;
      }
    }
  }
};

// A workgroup is a head of an env, a wavefront some columns of its state.
template <typename T, int NT, int VT, bool FULL>
__global__ __launch_bounds__(512 / VT, 2) void delta_grad_kernel(DeltaArgs a) {
  extern __shared__ float lds[];
  __shared__ Solved<true> solved[kGroup];
  __shared__ int bad;
  constexpr int kPart = 2 * NT * 256;
  const int lane = threadIdx.x & 63, slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slabs = blockDim.x >> 6;
  float* sums = lds + slabs * kPart + slab * 2 * kDeltaChunk;
  const int64_t unit = block_id(), heads = (int64_t)a.envs * a.heads, v_step = heads * a.values;
  if (unit >= heads) return;
  const int env = (int)(unit / a.heads), head = (int)(unit % a.heads);
  const Unit<NT, VT> u{{lane & 15, lane >> 4}, env, head, slab * 16 * VT};
  Grad<T, NT, VT, FULL> w{a,
                          u,
                          u.l,
                          {(const T*)a.q + env * a.q_env + head / a.share * a.q_head, a.q_step, a.keys, u.l},
                          {(const T*)a.k + env * a.k_env + head / a.share * a.k_head, a.k_step, a.keys, u.l},
                          {(const T*)a.v + env * a.v_env + head * a.v_head + u.first, a.v_step, a.values - u.first, u.l},
                          {(const T*)a.dy + env * a.dy_env + head * a.dy_head + u.first, a.dy_step, a.values - u.first, u.l},
                          0,
                          nullptr,
                          4 * u.l.g * v_step + u.col(),
                          lds + slab * kPart,
                          lds + slab * kPart + lane};
  const int chunks = (a.steps + kDeltaChunk - 1) / kDeltaChunk;
  const float* kept = a.saved + unit * a.keys * a.values;
  const int64_t state = heads * a.keys * a.values;  // of all heads
  const Steps<float, VT, FULL> over(a.saved + chunks * state + unit * a.values + u.first, v_step, a.values - u.first, u.l);
  auto at = [&](int chunk) {
    w.l = again(u.l), w.t0 = chunk * kDeltaChunk;
    w.dv = (T*)a.dv + unit * a.values + w.t0 * v_step;
  };
  auto hand_in = [&](float dgate, const f4& dbeta) {
    if (w.l.c == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[kDeltaChunk + w.l.in(j)] = dbeta[j];
    }
    if (w.l.g == 0) sums[w.l.c] = dgate;
  };
  static_assert(VT <= 2, "a tile of D for each of dq and dk");
  if (threadIdx.x == 0) bad = 0;
  clear_state(w.D);
  bool fine = true;
  for (int last = chunks; last > 0 && fine; last -= kGroup) {
    const int first = last > kGroup ? last - kGroup : 0;
    for (int n = slab; n < last - first; n += slabs) solve_chunk(a, (first + n) * kDeltaChunk, env, head, w.q, w.k, again(u.l), solved[n]);
    __syncthreads();
    for (int n = last - first - 1; n >= 0 && fine; --n) {
      at(first + n);
      f4 dbeta;
      float dgate;
      if (w.chunk(solved[n], kept + (first + n) * state, over, dgate, dbeta)) hand_in(dgate, dbeta);
      else bad = 1;
      Join<T, NT, VT, FULL> join;
      join.begin(w);
      __syncthreads();
      fine = !bad;  // nobody sets it again before the next barrier
      if (fine) join.end(w, unit, lds, slabs);
      __syncthreads();
    }
  }
  if (fine) return;
  // the whole rollout span by span, and where a value is not finite step by step
  clear_state(w.D);
  clear_state(w.Dt);
  for (int chunk = chunks - 1; chunk >= 0; --chunk) {
    at(chunk);
    w.gates = load_gates(a, w.t0, env, head, w.l);
    f4 dbeta = zero4();
    float dgate = 0.0f;
    for (int hi = w.gates.steps; hi > 0;) {
      const uint32_t before = w.gates.cuts & ((1u << hi) - 1u);
      const Span s{before ? 31 - __builtin_clz(before) : 0, hi};
      const bool cut = cut_at(w.gates, s.lo);
      const Kept<NT, VT> known{cut ? nullptr : kept + chunk * state};
      if (!w.back(s, known, dgate, dbeta)) w.back_singly(s, known, dgate, dbeta);
      if (cut) {
        clear_state(w.D);
        clear_state(w.Dt);
      }
      hi = s.lo;
    }
    hand_in(dgate, dbeta);
    Join<T, NT, VT, FULL> join;
    join.begin(w);
    __syncthreads();
    join.end(w, unit, lds, slabs);
    __syncthreads();
  }
}

// dq or dk of heads that share their rows: added in 32 bits, rounded once.  A thread
// takes four channels of a row.  Bound by reading the heads' rows.
template <typename T>
__global__ __launch_bounds__(256) void delta_share_kernel(const float* in, int64_t rows, int share, int keys, T* dq, T* dk) {
  const int pieces = (keys + 3) / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * rows * pieces; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / pieces;
    const int c = (int)(i - row * pieces) * 4;
    const float* p = in + row * share * keys + c;
    float x[4] = {};
    for (int n = 0; n < share; ++n) {
      float o[4];
      load_row<4>(p + n * keys, keys - c, o);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += o[j];
    }
    store_row<4>((row < rows ? dq + row * keys : dk + (row - rows) * keys) + c, keys - c, x);
  }
}

}  // namespace

int64_t delta_grad_work(const DeltaArgs& a) { return a.share == 1 ? 0 : 2 * (int64_t)a.steps * a.envs * a.heads * a.keys; }

hipError_t launch_delta_grad(const DeltaArgs& a, hipStream_t st) {
  hipError_t failed = hipSuccess;
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) {
      by_columns<nt == 8 ? 1 : 2>(a, [&](auto cols) {
        const int slabs = slabs_of(a.values, cols);
        const size_t shared = (size_t)slabs * (2 * 256 * nt + 2 * kDeltaChunk) * 4;
        by_truth(a.keys == 16 * nt && a.values % (16 * cols) == 0, [&](auto full) {
          auto* kernel = delta_grad_kernel<T, nt, cols, full>;
          if (shared > 48 * 1024) failed = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
          if (failed == hipSuccess) hipLaunchKernelGGL(kernel, wide_grid((int64_t)a.envs * a.heads), dim3(64 * slabs), shared, st, a);
        });
      });
    });
    if (a.share > 1 && failed == hipSuccess) {
      const int64_t rows = (int64_t)a.steps * a.envs * (a.heads / a.share), pieces = 2 * rows * ((a.keys + 3) / 4);
      hipLaunchKernelGGL((delta_share_kernel<T>), dim3((unsigned)std::min<int64_t>((pieces + 255) / 256, 1 << 16)), dim3(256), 0, st, a.work, rows, a.share, a.keys, (T*)a.dq, (T*)a.dk);
    }
  });
  return failed == hipSuccess ? hipGetLastError() : failed;
}

}  // namespace gbx
