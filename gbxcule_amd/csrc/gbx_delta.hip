// gbx_delta.hip -- the gated delta rule over whole rollouts and one step at a
// time.
#include "gbx_delta.h"

namespace gbx {
namespace {

template <typename T, int NT, int VT>
__global__ __launch_bounds__(256) void delta_kernel(DeltaArgs a, int slabs, int64_t units) {
  const int lane = threadIdx.x & 63;
  int64_t unit = block_id() * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const Unit<NT, VT> u{{lane & 15, lane >> 4}, (int)(unit / slabs / a.heads), (int)(unit / slabs % a.heads), (int)(unit % slabs) * 16 * VT};
  const Lane l = u.l;
  const int64_t place = ((int64_t)u.env * a.heads + u.head) * a.keys * a.values;  // of the state
  const T* q = (const T*)a.q + u.env * a.q_env + u.head / a.share * a.q_head;
  const T* k = (const T*)a.k + u.env * a.k_env + u.head / a.share * a.k_head;
  const T* v = (const T*)a.v + u.env * a.v_env + u.head * a.v_head + u.first;
  T* y = (T*)a.y + ((int64_t)u.env * a.heads + u.head) * a.values + u.col();
  const int64_t y_step = (int64_t)a.envs * a.heads * a.values;
  f4 S[NT][VT];
  if (a.state) load_state(a.state + place, a, u, S);
  else clear_state(S);
  for (int t0 = 0; t0 < a.steps; t0 += kDeltaChunk) {
    const Gates gates = load_gates(a, t0, u.env, u.head, l);
    if (a.saved) store_state(a.saved + (int64_t)(t0 / kDeltaChunk) * a.envs * a.heads * a.keys * a.values + place, a, u, S);
    int singles = 0;  // steps before this one go one by one
    for (int lo = 0; lo < gates.steps;) {
      const Span s{lo, lo < singles ? lo + 1 : next_cut(gates, lo)};
      if (cut_at(gates, lo)) clear_state(S);
      f4 kr[NT], qr[NT];
      load_rows(k + (int64_t)t0 * a.k_step, a.k_step, a.keys, s, l, kr);
      load_rows(q + (int64_t)t0 * a.q_step, a.q_step, a.keys, s, l, qr);
      const float beta = s.has(l.c) ? gates.beta : 0.0f;
      const float kap = unit_of(kr, a.normalize), qap = unit_of(qr, a.normalize) * a.scale;
      const f4 bin = across(beta, l), kin = across(kap, l), qin = across(qap, l);
      const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
      const System sys = system_of(kr, kap, kin, beta, bin, d, l);
      f4 vc[VT], U[VT];
      load_cols(v + (int64_t)t0 * a.v_step, a.v_step, a.values - u.first, s, l, vc);
      bool fine = true;
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        f4 rhs = zero4();
#pragma unroll
        for (int r = 0; r < NT; ++r) rhs = mma(kr[r], S[r][t], rhs);
#pragma unroll
        for (int j = 0; j < 4; ++j) rhs[j] = s.has(l.in(j)) ? bin[j] * fmaf(-d.in[j] * kin[j], rhs[j], vc[t][j]) : 0.0f;
        U[t] = mma(sys.T.row, rhs, zero4());
        fine = fine && finite4(U[t]);
      }
      if (s.hi - s.lo > 1 && !__all(fine)) {
        // in a product zero times infinity would reach earlier steps, too
        singles = s.hi;
        continue;
      }
      f4 kq = zero4();  // row c, places in(j): q_c . k_j
#pragma unroll
      for (int r = 0; r < NT; ++r) kq = mma(kr[r], qr[r], kq);
#pragma unroll
      for (int j = 0; j < 4; ++j) kq[j] = l.in(j) <= l.c ? kq[j] * (qap * kin[j]) * d.pair[j] : 0.0f;
      float out[4][VT];
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        f4 Y = zero4();
#pragma unroll
        for (int r = 0; r < NT; ++r) Y = mma(qr[r], S[r][t], Y);
#pragma unroll
        for (int j = 0; j < 4; ++j) Y[j] *= qin[j] * d.in[j];
        Y = mma(kq, U[t], Y);
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j][t] = Y[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) store_row<VT>(y + (t0 + l.in(j)) * y_step, s.has(l.in(j)) ? a.values - u.col() : 0, out[j]);
      f4 kc[NT];
      load_cols(k + (int64_t)t0 * a.k_step, a.k_step, a.keys, s, l, kc);
#pragma unroll
      for (int t = 0; t < VT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) U[t][j] *= d.tail[j] * kin[j];
#pragma unroll
        for (int r = 0; r < NT; ++r) S[r][t] = mma(kc[r], U[t], S[r][t] * d.all);
      }
      lo = s.hi;
    }
  }
  store_state(a.last + place, a, u, S);
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

int64_t delta_work(const DeltaArgs&) { return 0; }

hipError_t launch_delta(const DeltaArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) {
      constexpr int kCols = nt == 8 ? 2 : 4;
      const int slabs = (a.values + 16 * kCols - 1) / (16 * kCols);
      const int64_t units = (int64_t)a.envs * a.heads * slabs;
      hipLaunchKernelGGL((delta_kernel<T, nt, kCols>), wide_grid((units + 3) / 4), dim3(256), 0, st, a, slabs, units);
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
