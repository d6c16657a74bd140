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
// The inner product is computed anew at the end of every span, so its error does not
// grow with the length of the rollout.
#include "gbx_delta.h"

#include <algorithm>

namespace gbx {
namespace {

// The state with the summed index on its columns: tile (t, r), place in(j):
// column VT * in(j) + t, channel NT * c + r.
template <int NT, int VT>
__device__ __forceinline__ void load_turned(const float* p, const DeltaArgs& a, const Unit<NT, VT>& u, f4 (&s)[VT][NT]) {
  const int col = u.first + 4 * VT * u.l.g;
#pragma unroll
  for (int r = 0; r < NT; ++r) {
    const int row = NT * u.l.c + r;
    float x[4 * VT];
    load_row<4 * VT>(p + (int64_t)row * a.values + col, row < a.keys ? a.values - col : 0, x);
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[t][r][j] = x[VT * j + t];
  }
}

template <typename T, int NT, int VT>
struct Grad {
  static constexpr int kKeys = 16 * NT;
  DeltaArgs a;
  Unit<NT, VT> u;
  Lane l;
  const T *q, *k, *v, *dy;  // of the chunk's first step
  T* dv;
  Gates gates;
  f4 D[NT][VT], Dt[VT][NT];  // gradient of the state, both ways round
  f4 S[NT][VT], St[VT][NT];  // the state before the span

  __device__ __forceinline__ void start(const float* saved, bool cut) {
    if (cut) {
      clear_state(S);
      clear_state(St);
    } else {
      load_state(saved, a, u, S);
      load_turned(saved, a, u, St);
    }
  }
  // One step of the forward pass.
  __device__ __forceinline__ void advance(int t0) {
    const Span s{t0, t0 + 1};
    f4 kr[NT], kc[NT], vc[VT];
    load_rows(k, a.k_step, a.keys, s, l, kr);
    load_cols(k, a.k_step, a.keys, s, l, kc);
    load_cols(v, a.v_step, a.values - u.first, s, l, vc);
    const f4 bin = across(s.has(l.c) ? gates.beta : 0.0f, l), kin = across(unit_of(kr, a.normalize), l);
    const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      f4 x = zero4();
#pragma unroll
      for (int r = 0; r < NT; ++r) x = mma(kr[r], S[r][t], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = s.has(l.in(j)) ? kin[j] * bin[j] * fmaf(-d.in[j] * kin[j], x[j], vc[t][j]) : 0.0f;
#pragma unroll
      for (int r = 0; r < NT; ++r) {
        S[r][t] = mma(kc[r], x, S[r][t] * d.all);
        St[t][r] = mma(x, kc[r], St[t][r] * d.all);
      }
    }
  }

  // Walks a span back.  False, and nothing done, if a value is not finite: in a
  // product zero times infinity would reach steps that the formulas keep from it.
  __device__ __forceinline__ bool back(Span s, f4 (&dq)[NT], f4 (&dk)[NT], float& dgate, f4& dbeta) {
    f4 kr[NT], qr[NT], kc[NT], qc[NT], dyr[VT], dyc[VT], vc[VT];
    load_rows(k, a.k_step, a.keys, s, l, kr);
    load_rows(q, a.q_step, a.keys, s, l, qr);
    const float beta = s.has(l.c) ? gates.beta : 0.0f;
    const float kap = unit_of(kr, a.normalize), qap = unit_of(qr, a.normalize);
    const f4 bin = across(beta, l), kin = across(kap, l), qin = across(qap, l);
    const Decay d = decay_of(s.has(l.c) ? gates.gate : 0.0, l);
    const System sys = system_of(kr, kap, kin, beta, bin, d, l);
    load_cols(v, a.v_step, a.values - u.first, s, l, vc);
    load_cols(dy, a.dy_step, a.values - u.first, s, l, dyc);
    load_rows(dy, a.dy_step, a.values - u.first, s, l, dyr);
    f4 aq = zero4();  // A^T: row c, places in(j) >= c
#pragma unroll
    for (int r = 0; r < NT; ++r) aq = mma(qr[r], kr[r], aq);
#pragma unroll
    for (int j = 0; j < 4; ++j) aq[j] = l.in(j) >= l.c ? aq[j] * (kap * qin[j] * a.scale) * d.pair[j] : 0.0f;

    f4 U[VT], Ut[VT], W[VT], Wt[VT], over[VT];  // over: u / beta
    float whole = 0.0f;                         // the part of <S, D> that the span wrote
    bool fine = true;
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      f4 x = zero4(), rhs, plain;
#pragma unroll
      for (int r = 0; r < NT; ++r) x = mma(kr[r], S[r][t], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        over[t][j] = s.has(l.in(j)) ? fmaf(-d.in[j] * kin[j], x[j], vc[t][j]) : 0.0f;
        rhs[j] = s.has(l.in(j)) ? bin[j] * over[t][j] : 0.0f;
        plain[j] = -sys.plain[j];
      }
      U[t] = mma(sys.T.row, rhs, zero4());
      Ut[t] = mma(rhs, sys.T.row, zero4());
      over[t] = mma(plain, U[t], over[t]);
      x = zero4();
#pragma unroll
      for (int r = 0; r < NT; ++r) x = mma(kr[r], D[r][t], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = s.has(l.in(j)) ? d.tail[j] * kin[j] * x[j] : 0.0f;
        whole = fmaf(x[j], U[t][j], whole);
      }
      x = mma(aq, dyc[t], x);
      W[t] = mma(sys.T.col, x, zero4());
      Wt[t] = mma(x, sys.T.col, zero4());
      fine = fine && finite4(U[t]) && finite4(W[t]);
    }
    if (s.hi - s.lo > 1 && !__all(fine)) return false;

    f4 p = zero4(), pt = zero4(), m = zero4(), mt = zero4();
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      p = mma(Ut[t], dyr[t], p);
      pt = mma(dyr[t], Ut[t], pt);
      m = mma(Ut[t], Wt[t], m);
      mt = mma(Wt[t], Ut[t], mt);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      p[j] = l.in(j) <= l.c ? p[j] * (a.scale * kin[j]) * d.pair[j] : 0.0f;
      pt[j] = l.in(j) >= l.c ? pt[j] * (a.scale * qin[j]) * d.pair[j] : 0.0f;
      m[j] = l.in(j) < l.c ? -m[j] * (beta * kin[j]) * d.pair[j] : 0.0f;
      mt[j] = l.in(j) > l.c ? -mt[j] * (bin[j] * kin[j]) * d.pair[j] : 0.0f;
    }
    // dv, dbeta, and what D takes up
    f4 asks[VT], gives[VT], bsum = zero4();
    float out[4][VT];
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      Wt[t] *= beta;  // dv's rows
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bsum[j] = fmaf(W[t][j], over[t][j], bsum[j]);
        out[j][t] = bin[j] * W[t][j];
        asks[t][j] = a.scale * qin[j] * d.in[j] * dyc[t][j];
        gives[t][j] = -d.in[j] * kin[j] * out[j][t];
      }
    }
    const int64_t v_step = (int64_t)a.envs * a.heads * a.values;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      store_row<VT>(dv + l.in(j) * v_step, s.has(l.in(j)) ? a.values - u.col() : 0, out[j]);
#pragma unroll
      for (int n = 1; n < 16; n <<= 1) bsum[j] += __shfl_xor(bsum[j], n, 16);
      dbeta[j] = s.has(l.in(j)) ? bsum[j] : dbeta[j];
    }
    load_cols(k, a.k_step, a.keys, s, l, kc);
    load_cols(q, a.q_step, a.keys, s, l, qc);
    f4 e = zero4();  // q . dq + k . dk_reads - k . dk_writes
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      f4 x = zero4(), reads = zero4(), writes = zero4();
#pragma unroll
      for (int t = 0; t < VT; ++t) {
        x = mma(dyr[t], St[t][r], x);
        reads = mma(Wt[t], St[t][r], reads);
        writes = mma(Ut[t], Dt[t][r], writes);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] *= a.scale * d.in[j];
        reads[j] *= -d.in[j];
        writes[j] *= d.tail[j];
      }
      x = mma(p, kc[r], x);
      reads = mma(m, kc[r], reads);
      writes = mma(pt, qc[r], writes);
      writes = mma(mt, kc[r], writes);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = fmaf(qin[j] * qc[r][j], x[j], e[j]);
        e[j] = fmaf(kin[j] * kc[r][j], reads[j] - writes[j], e[j]);
        dq[r][j] = s.has(l.in(j)) ? x[j] : dq[r][j];
        dk[r][j] = s.has(l.in(j)) ? reads[j] + writes[j] : dk[r][j];
      }
    }
    float held = 0.0f;
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int t = 0; t < VT; ++t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) held = fmaf(S[r][t][j], D[r][t][j], held);
        D[r][t] = mma(kc[r], gives[t], mma(qc[r], asks[t], D[r][t] * d.all));
        Dt[t][r] = mma(gives[t], kc[r], mma(asks[t], qc[r], Dt[t][r] * d.all));
      }
    whole = fmaf(d.all, held, whole);
#pragma unroll
    for (int n = 1; n < 64; n <<= 1) whole += __shfl_xor(whole, n, 64);
    float own = 0.0f;  // e of step c, then the sum from there on
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int n = 1; n < 16; n <<= 1) e[j] += __shfl_xor(e[j], n, 16);
      const float other = __shfl(e[j], l.c / 4 * 16, 64);
      own = (l.c & 3) == j && s.has(l.c) ? other : own;
    }
#pragma unroll
    for (int n = 1; n < 16; n <<= 1) {
      const float later = __shfl_down(own, n, 16);
      own += l.c + n < 16 ? later : 0.0f;
    }
    if (s.has(l.c)) dgate = cut_at(gates, l.c) ? 0.0f : whole + own;
    return true;
  }
};

// A workgroup is a head of an env, a wavefront some columns of its state.  The
// columns' parts of dq, dk, dgate and dbeta are added in LDS, in one order.
template <typename T, int NT, int VT>
__global__ __launch_bounds__(512 / VT) void delta_grad_kernel(DeltaArgs a) {
  extern __shared__ float lds[];
  constexpr int kKeys = 16 * NT, kPart = 2 * kDeltaChunk * kKeys;
  const int lane = threadIdx.x & 63, slab = threadIdx.x >> 6, slabs = blockDim.x >> 6;
  float* sums = lds + slabs * kPart;  // [slab][dgate, dbeta][step]
  Grad<T, NT, VT> w;
  w.a = a;
  const int64_t unit = block_id();
  if (unit >= (int64_t)a.envs * a.heads) return;
  w.u = {{lane & 15, lane >> 4}, (int)(unit / a.heads), (int)(unit % a.heads), slab * 16 * VT};
  w.l = w.u.l;
  const Lane l = w.l;
  const int env = w.u.env, head = w.u.head;
  const T* q = (const T*)a.q + env * a.q_env + head / a.share * a.q_head;
  const T* k = (const T*)a.k + env * a.k_env + head / a.share * a.k_head;
  const T* v = (const T*)a.v + env * a.v_env + head * a.v_head + w.u.first;
  const T* dy = (const T*)a.dy + env * a.dy_env + head * a.dy_head + w.u.first;
  T* dv = (T*)a.dv + unit * a.values + w.u.col();
  const int64_t heads = (int64_t)a.envs * a.heads;
  clear_state(w.D);
  clear_state(w.Dt);
  for (int t0 = (a.steps - 1) / kDeltaChunk * kDeltaChunk; t0 >= 0; t0 -= kDeltaChunk) {
    w.gates = load_gates(a, t0, env, head, l);
    w.q = q + t0 * a.q_step, w.k = k + t0 * a.k_step, w.v = v + t0 * a.v_step, w.dy = dy + t0 * a.dy_step;
    w.dv = dv + t0 * heads * a.values;
    const float* saved = a.saved + ((int64_t)(t0 / kDeltaChunk) * heads + unit) * a.keys * a.values;
    f4 dq[NT], dk[NT], dbeta = zero4();
    float dgate = 0.0f;
#pragma unroll
    for (int r = 0; r < NT; ++r) dq[r] = dk[r] = zero4();
    int singles = kDeltaChunk;  // steps from this one on go one by one
    for (int hi = w.gates.steps; hi > 0;) {
      const uint32_t before = w.gates.cuts & ((1u << hi) - 1u);
      const int from = before ? 31 - __builtin_clz(before) : 0;  // where the state is known
      const int lo = hi > singles ? hi - 1 : from;
      w.start(saved, cut_at(w.gates, from));
      for (int t = from; t < lo; ++t) w.advance(t);
      if (!w.back({lo, hi}, dq, dk, dgate, dbeta)) {
        singles = lo;
        continue;
      }
      if (cut_at(w.gates, lo)) {
        clear_state(w.D);
        clear_state(w.Dt);
      }
      hi = lo;
    }
    float* part = lds + slab * kPart;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[NT];
#pragma unroll
      for (int r = 0; r < NT; ++r) x[r] = dq[r][j];
      store_row<NT>(part + l.in(j) * kKeys + NT * l.c, NT, x);
#pragma unroll
      for (int r = 0; r < NT; ++r) x[r] = dk[r][j];
      store_row<NT>(part + (kDeltaChunk + l.in(j)) * kKeys + NT * l.c, NT, x);
      if (l.c == 0) sums[(slab * 2 + 1) * kDeltaChunk + l.in(j)] = dbeta[j];
    }
    if (l.g == 0) sums[slab * 2 * kDeltaChunk + l.c] = dgate;
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += blockDim.x) {
      const int t = i >> 4, c = i & 15, rest = a.keys - NT * c;
      const bool live = t < w.gates.steps;
      const int64_t row = (t0 + t) * heads + unit;
      auto turn = [&](const T* p, int64_t step, int kind, void* to) {
        float x[NT], dx[NT] = {}, ss = 0.0f, dot = 0.0f;
        load_row<NT>(p + t * step + NT * c, live ? rest : 0, x);
        for (int n = 0; n < slabs; ++n)
#pragma unroll
          for (int r = 0; r < NT; ++r) dx[r] += lds[n * kPart + (kind * kDeltaChunk + t) * kKeys + NT * c + r];
        if (a.normalize) {  // x / length: the gradient's part along x goes
#pragma unroll
          for (int r = 0; r < NT; ++r) {
            ss = fmaf(x[r], x[r], ss);
            dot = fmaf(x[r], dx[r], dot);
          }
#pragma unroll
          for (int n = 1; n < 16; n <<= 1) {
            ss += __shfl_xor(ss, n, 16);
            dot += __shfl_xor(dot, n, 16);
          }
          const float unit_x = rsqrtf(ss + kUnitEps);
          dot *= unit_x * unit_x;
#pragma unroll
          for (int r = 0; r < NT; ++r) dx[r] = unit_x * fmaf(-x[r], dot, dx[r]);
        }
        if (a.share == 1) store_row<NT>((T*)to + row * a.keys + NT * c, live ? rest : 0, dx);
        else store_row<NT>((float*)to + row * a.keys + NT * c, live ? rest : 0, dx);
      };
      turn(w.q, a.q_step, 0, a.share == 1 ? a.dq : a.work);
      turn(w.k, a.k_step, 1, a.share == 1 ? a.dk : a.work + a.steps * heads * a.keys);
      if (i < 2 * kDeltaChunk && c < w.gates.steps) {
        float x = 0.0f;
        for (int n = 0; n < slabs; ++n) x += sums[n * 2 * kDeltaChunk + i];
        (t == 0 ? a.dgate : a.dbeta)[(t0 + c) * heads + unit] = x;
      }
    }
    __syncthreads();
  }
}

// dq or dk of heads that share their rows: added in 32 bits, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void delta_share_kernel(const float* in, int64_t count, int share, int keys, T* dq, T* dk) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * count; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / keys;
    const float* p = in + row * share * keys + i % keys;
    float x = 0.0f;
    for (int n = 0; n < share; ++n) x += p[(int64_t)n * keys];
    (i < count ? dq[i] : dk[i - count]) = (T)x;
  }
}

}  // namespace

int64_t delta_grad_work(const DeltaArgs& a) { return a.share == 1 ? 0 : 2 * (int64_t)a.steps * a.envs * a.heads * a.keys; }

hipError_t launch_delta_grad(const DeltaArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_keys(a.keys, [&](auto nt) {
      constexpr int kCols = nt == 8 ? 1 : 2;
      const int slabs = (a.values + 16 * kCols - 1) / (16 * kCols);
      const size_t shared = (size_t)slabs * (2 * kDeltaChunk * 16 * nt + 2 * kDeltaChunk) * 4;
      auto* kernel = delta_grad_kernel<T, nt, kCols>;
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
      hipLaunchKernelGGL(kernel, wide_grid((int64_t)a.envs * a.heads), dim3(64 * slabs), shared, st, a);
    });
    if (a.share > 1) {
      const int64_t count = (int64_t)a.steps * a.envs * (a.heads / a.share) * a.keys;
      hipLaunchKernelGGL((delta_share_kernel<T>), dim3((unsigned)std::min<int64_t>((2 * count + 255) / 256, 1 << 16)), dim3(256), 0, st, a.work, count, a.share, a.keys, (T*)a.dq, (T*)a.dk);
    }
  });
  return hipGetLastError();
}

}  // namespace gbx
