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
//   (solved for u / beta, which the gradient wants: rhs / beta, and beta_j in L for beta_i)
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
// not depend on each other), a workgroup all of them: what does not depend on the
// state, the solved system above all, its wavefronts make for each other.  A gate
// that closes and an episode's start are a zero decay.  That is the formulas as
// long as all is finite; where a value is not, zero times it would reach steps that it
// must not, and the workgroup does its rollout again in segments between the
// cuts, and step by step where a segment has such a value: nothing of what is
// before a cut takes part in a product behind it.
//
// What bounds it: a chunk follows the one before, and of the three parts of every
// 32-bit factor 24 bits of work come for each 8 that a matrix instruction
// takes.  At 128 steps x 1,024 envs x 4 heads of 64 x 64 the forward pass takes
// 289 us (moving 0.94 GB with what it keeps for the gradient, 190 us) and the
// gradient 753 (1.1 GB, 230 us): 2,460 vector instructions a wavefront and chunk,
// 175 of them matrix ones, and two wavefronts a SIMD to hide that each waits 64% of its time.
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

__device__ __forceinline__ f4 zero4() { return f4{0.0f, 0.0f, 0.0f, 0.0f}; }

// What a decay leaves of a sum: of none nothing, though the sum be infinite (of finite
// values from before an episode, say, as large as memory may hold that nothing has written).
__device__ __forceinline__ float left_of(float x, float decay) { return decay == 0.0f ? 0.0f : x * decay; }
__device__ __forceinline__ f4 left_of(f4 x, f4 decay) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = left_of(x[j], decay[j]);
  return x;
}

// Factors of a product, four places of the summed index a lane.
//
// Whole: 32 bits, on the 32-bit matrix instructions, which sum 4 places in twice
// the time that the 16-bit ones take for 32.  Parts: a sum of N bfloat16
// values, each what the ones before leave; an input's bfloat16 is one part, a
// float16 exactly two.  A product of two sums is their terms' products, added in
// 32 bits, two of them in an instruction that sums 32 places.
// Three parts hold a 32-bit value whole; two lose its last eight bits, which brought
// the learner's recurrence from 1,400 to 1,020 us and its results from 3e-7 to 4e-6.
constexpr int kParts = 3;
struct Whole {
  f4 v;
};
typedef uint32_t w2 __attribute__((ext_vector_type(2)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
template <int N>
struct Parts {
  w2 p[N];
};
// two bfloat16 in a word, and back
__device__ __forceinline__ uint32_t narrow2(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x, y}, b2));
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ f4 wide(w2 w) { return f4{low(w[0]), high(w[0]), low(w[1]), high(w[1])}; }
template <int N>
__device__ __forceinline__ Parts<N> parts_of(f4 x) {
  Parts<N> r;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    r.p[n] = w2{narrow2(x[0], x[1]), narrow2(x[2], x[3])};
    if (n + 1 < N) x -= wide(r.p[n]);
  }
  return r;
}

// d += a b, 16 x 16 x 16
__device__ __forceinline__ f4 mma(f4 a, f4 b, f4 d) {
#pragma unroll
  for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], d, 0, 0, 0);
  return d;
}
__device__ __forceinline__ f4 mma(Whole a, Whole b, f4 d) { return mma(a.v, b.v, d); }
// (All 16-bit products are of this one shape.  A product of 16 places and one of 32 that
// follow each other through the same sum lose terms: nothing waits between them, neither
// the card nor, by code of the compiler's, the program; half of 131,072 sums of small whole
// numbers were wrong, and none with 16 cycles in between.  Products of 32 places and the 32-bit
// ones of 4, in turn through one sum or one the factor of the other, were all exact.)
__device__ __forceinline__ f4 two_terms(w2 a, w2 b, w2 a2, w2 b2, f4 d) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, w4{a[0], a[1], a2[0], a2[1]}), __builtin_bit_cast(b8, w4{b[0], b[1], b2[0], b2[1]}), d, 0, 0, 0);
}
__device__ __forceinline__ f4 one_term(w2 a, w2 b, f4 d) { return two_terms(a, b, a, w2{0u, 0u}, d); }
// Terms whose places add up to more than a whole value's last, kParts - 1, are below its
// rounding and left out, but where an instruction has room for one.
template <int A, int B>
__device__ __forceinline__ f4 mma(const Parts<A>& a, const Parts<B>& b, f4 d) {
  if constexpr (A > B) {
    if constexpr (B == 1) return two_terms(a.p[0], b.p[0], a.p[1], b.p[0], one_term(a.p[2], b.p[0], d));
    else return two_terms(a.p[0], b.p[0], a.p[0], b.p[1], two_terms(a.p[1], b.p[0], a.p[1], b.p[1], two_terms(a.p[2], b.p[0], a.p[2], b.p[1], d)));
  } else if constexpr (A == 1) {
    if constexpr (B == 1) return one_term(a.p[0], b.p[0], d);
    else return two_terms(a.p[0], b.p[0], a.p[0], b.p[1], one_term(a.p[0], b.p[2], d));
  } else if constexpr (B == 2) {
    return two_terms(a.p[0], b.p[0], a.p[1], b.p[0], two_terms(a.p[0], b.p[1], a.p[1], b.p[1], d));
  } else if constexpr (A == 2) {
    return two_terms(a.p[0], b.p[0], a.p[1], b.p[0], two_terms(a.p[0], b.p[1], a.p[1], b.p[1], two_terms(a.p[0], b.p[2], a.p[1], b.p[2], d)));
  } else {
    return two_terms(a.p[0], b.p[0], a.p[0], b.p[1], two_terms(a.p[1], b.p[0], a.p[1], b.p[1], two_terms(a.p[2], b.p[0], a.p[0], b.p[2], d)));
  }
}

// Two tiles that follow each other in the sum: an instruction takes a term of both,
// with no place left empty.
struct WholeTwo {
  f4 v[2];
};
template <int N>
struct PartsTwo {
  w4 p[N];
};
__device__ __forceinline__ WholeTwo two(Whole a, Whole b) { return {{a.v, b.v}}; }
template <int N>
__device__ __forceinline__ PartsTwo<N> two(const Parts<N>& a, const Parts<N>& b) {
  PartsTwo<N> r;
#pragma unroll
  for (int n = 0; n < N; ++n) r.p[n] = w4{a.p[n][0], a.p[n][1], b.p[n][0], b.p[n][1]};
  return r;
}
__device__ __forceinline__ f4 mma(const WholeTwo& a, const WholeTwo& b, f4 d) { return mma(a.v[0], b.v[0], mma(a.v[1], b.v[1], d)); }
template <int A, int B>
__device__ __forceinline__ f4 mma(const PartsTwo<A>& a, const PartsTwo<B>& b, f4 d) {
#pragma unroll
  for (int n = kParts - 1; n >= 0; --n)  // the small terms first
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j)
        if (i + j == n) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a.p[i]), __builtin_bit_cast(b8, b.p[j]), d, 0, 0, 0);
  return d;
}

// Inputs in words as they lie in memory.
template <typename T, int COUNT>
struct Words {
  static constexpr int kWords = (COUNT * (int)sizeof(T) + 3) / 4;
  uint32_t w[kWords];
};
// A value of which the compiler does not know that it is the same every time:
// what is made from it inside a loop is made there, not before.  (Hundreds of
// masks and addresses of rows that may end inside a tile, kept through a loop over
// chunks, leave no registers.)
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// COUNT elements.
template <int COUNT, typename T>
__device__ __forceinline__ Words<T, COUNT> load_whole(const T* p) {
  Words<T, COUNT> r{};
  __builtin_memcpy(r.w, p, COUNT * sizeof(T));
  return r;
}
// Zeros where `has` does not hold.
template <int COUNT, typename T>
__device__ __forceinline__ void mask(Words<T, COUNT>& r, bool has) {
#pragma unroll
  for (int i = 0; i < r.kWords; ++i) r.w[i] = has ? r.w[i] : 0u;
}
// COUNT elements, zero from `valid` on, in pieces of up to 8.  A piece that ends
// inside is loaded element by element, its last one again and again: without
// conditions of their own the loads go out together.  (Zeros and loads meet in whole
// words: where they met in 16-bit elements, each took a register.)
template <int COUNT, typename T>
__device__ __forceinline__ Words<T, COUNT> load_words(const T* p, int valid) {
  constexpr int kPiece = COUNT < 8 ? COUNT : 8, kWords = Words<T, kPiece>::kWords;
  static_assert(COUNT % kPiece == 0, "whole pieces");
  Words<T, COUNT> r{};
  valid = opaque(valid);
#pragma unroll
  for (int n = 0; n < COUNT; n += kPiece) {
    uint32_t* to = r.w + n / kPiece * kWords;
    const int rest = valid - n;
    if (rest >= kPiece) {
      __builtin_memcpy(to, p + n, kPiece * sizeof(T));
    } else if (rest > 0) {
      T x[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) x[i] = p[n + (i < rest ? i : rest - 1)];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        if constexpr (sizeof(T) == 4) to[i] = i < rest ? __builtin_bit_cast(uint32_t, x[i]) : 0u;
        else to[i / 2] |= i < rest ? (uint32_t)__builtin_bit_cast(uint16_t, x[i]) << (16 * (i & 1)) : 0u;
      }
    }
  }
  return r;
}
// the same as floats
template <int COUNT, typename T>
__device__ __forceinline__ void load_floats(const T* p, int valid, float (&v)[COUNT]) {
  const Words<T, COUNT> x = load_words<COUNT>(p, valid);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(x.w[i]);
    else v[i] = (float)__builtin_bit_cast(T, (uint16_t)(x.w[i / 2] >> (16 * (i & 1))));
  }
}
// elements I and J of 16 bits as one word
template <int I, int J>
__device__ __forceinline__ uint32_t pick(const uint32_t* p, const uint32_t* q) {
  return __builtin_amdgcn_perm(q[J / 2], p[I / 2], ((J & 1) ? 0x07060000u : 0x05040000u) | ((I & 1) ? 0x0302u : 0x0100u));
}

// How the products take the inputs, of type T, and values computed from them.
template <typename T>
struct Factor {
  using Raw = Parts<1>;
  using Fine = Parts<kParts>;
  // elements I, J, K and L of four rows of words
  template <int I, int J, int K, int L>
  static __device__ __forceinline__ Raw raw(const uint32_t* x, const uint32_t* y, const uint32_t* z, const uint32_t* v) {
    return {{w2{pick<I, J>(x, y), pick<K, L>(z, v)}}};
  }
  static __device__ __forceinline__ f4 wide(const Raw& x) { return gbx::wide(x.p[0]); }
  static __device__ __forceinline__ Fine fine(f4 x) { return parts_of<kParts>(x); }
};
template <>
struct Factor<_Float16> {
  using Raw = Parts<2>;
  using Fine = Parts<kParts>;
  static __device__ __forceinline__ float half(const uint32_t* x, int i) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(x[i / 2] >> (16 * (i & 1)))); }
  template <int I, int J, int K, int L>
  static __device__ __forceinline__ Raw raw(const uint32_t* x, const uint32_t* y, const uint32_t* z, const uint32_t* v) {
    return parts_of<2>(f4{half(x, I), half(y, J), half(z, K), half(v, L)});
  }
  static __device__ __forceinline__ f4 wide(const Raw& x) { return gbx::wide(x.p[0]) + gbx::wide(x.p[1]); }
  static __device__ __forceinline__ Fine fine(f4 x) { return parts_of<kParts>(x); }
};
template <>
struct Factor<float> {
  using Raw = Whole;
  using Fine = Whole;
  template <int I, int J, int K, int L>
  static __device__ __forceinline__ Raw raw(const uint32_t* x, const uint32_t* y, const uint32_t* z, const uint32_t* v) {
    return {f4{__uint_as_float(x[I]), __uint_as_float(y[J]), __uint_as_float(z[K]), __uint_as_float(v[L])}};
  }
  static __device__ __forceinline__ f4 wide(const Raw& x) { return x.v; }
  static __device__ __forceinline__ Fine fine(f4 x) { return {x}; }
};
// The tiles of a sum over a wavefront's VT tiles of columns.
template <int VT, typename R>
__device__ __forceinline__ auto columns(const R (&x)[VT]) {
  if constexpr (VT == 2) return two(x[0], x[1]);
  else return x[0];
}
template <typename T>
using Raw = typename Factor<T>::Raw;
template <typename T>
using Fine = typename Factor<T>::Fine;

struct Lane {
  int c, g;  // place among 16 lanes (a row or column), group of 16 (four places of the other index)
  __device__ __forceinline__ int in(int j) const { return 4 * g + j; }
};
__device__ __forceinline__ Lane again(Lane l) { return {opaque(l.c), opaque(l.g)}; }

// Another of the 16 lanes' value, zero past their ends.
template <int CONTROL>
__device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xF, 0xF, true));
}
template <int CONTROL>
__device__ __forceinline__ double row_lane(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CONTROL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CONTROL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kQuad = 0x55, kLeft = 0x100, kRight = 0x110, kTurn = 0x120, kOf = 0x150;  // times a lane; by n lanes; lane n's
// sum over the 16 lanes, in all of them
__device__ __forceinline__ float row_sum(float v) {
  v += row_lane<kTurn + 8>(v);
  v += row_lane<kTurn + 4>(v);
  v += row_lane<kTurn + 2>(v);
  return v + row_lane<kTurn + 1>(v);
}
// sums over the lanes up to this one, and from this one on
template <typename V>
__device__ __forceinline__ V sum_up_to(V v) {
  v += row_lane<kRight + 1>(v);
  v += row_lane<kRight + 2>(v);
  v += row_lane<kRight + 4>(v);
  return v + row_lane<kRight + 8>(v);
}
__device__ __forceinline__ float sum_from(float v) {
  v += row_lane<kLeft + 1>(v);
  v += row_lane<kLeft + 2>(v);
  v += row_lane<kLeft + 4>(v);
  return v + row_lane<kLeft + 8>(v);
}
__device__ __forceinline__ float from_lane(float v, int lane) { return __int_as_float(__builtin_amdgcn_ds_bpermute(4 * lane, __float_as_int(v))); }

// A lane's value of the row in(j), given each row's in the lanes c.
__device__ __forceinline__ f4 across(float own, Lane l) {
  f4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = from_lane(own, 20 * l.g + j);
  return v;
}

// The steps of a chunk from `lo` to before `hi`.
struct Span {
  int lo, hi;
  __device__ __forceinline__ bool has(int t) const { return t >= lo && t < hi; }
};

// f(std::integral_constant) for 0 to N - 1
template <int N, typename F, int I = 0>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, F, I + 1>((F&&)f);
  }
}

// A tensor's steps of one head of an env, read as rows (4 * NT channels of step
// c each, tile r's place in(j) channel NT * in(j) + r) or as columns (NT channels
// from NT * c on of each step in(j)).
//
// FULL: there are as many channels as the tiles have.  Steps outside of the span
// then read the span's first: loads without branches, which all go out
// together.  They come out as zeros, or, where nothing is made of them, as they are (KEEP).
template <typename T, int NT, bool FULL>
struct Steps {
  const T* p;  // of the first step, the same in all lanes
  int64_t step, row, col;
  int channels;
  __device__ __forceinline__ Steps(const T* p_, int64_t step_, int channels_, Lane l)
      : p(p_), step(step_), row(l.c * step_ + 4 * NT * l.g), col(4 * l.g * step_ + NT * l.c), channels(channels_) {}
  template <bool KEEP = false>
  __device__ __forceinline__ void rows(int t0, Span s, Lane l, Raw<T> (&v)[NT]) const {
    Words<T, 4 * NT> x;
    const bool has = s.has(l.c);
    if constexpr (FULL) {
      x = load_whole<4 * NT>(p + t0 * step + (has ? row : s.lo * step + 4 * NT * l.g));
      if constexpr (!KEEP) mask(x, has);
    } else {
      x = load_words<4 * NT>(p + t0 * step + row, has ? channels - 4 * NT * l.g : 0);
    }
    each<NT>([&](auto r) { v[r] = Factor<T>::template raw<r, NT + r, 2 * NT + r, 3 * NT + r>(x.w, x.w, x.w, x.w); });
  }
  template <bool KEEP = false>
  __device__ __forceinline__ void cols(int t0, Span s, Lane l, Raw<T> (&v)[NT]) const {
    Words<T, NT> x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool has = s.has(l.in(j));
      if constexpr (FULL) {
        x[j] = load_whole<NT>(p + t0 * step + (has ? j * step + col : s.lo * step + NT * l.c));
        if constexpr (!KEEP) mask(x[j], has);
      } else {
        x[j] = load_words<NT>(p + (t0 + j) * step + col, has ? channels - NT * l.c : 0);
      }
    }
    each<NT>([&](auto r) { v[r] = Factor<T>::template raw<r, r, r, r>(x[0].w, x[1].w, x[2].w, x[3].w); });
  }
};

// Inner products of the rows with each other: row c, places in(j), or the other way round.
template <int NT, typename R>
__device__ __forceinline__ f4 product_of(const R (&row)[NT], const R (&col)[NT]) {
  f4 x = zero4();
#pragma unroll
  for (int r = 0; r < NT; r += 2) x = mma(two(row[r], row[r + 1]), two(col[r], col[r + 1]), x);
  return x;
}
template <int NT, typename R>
__device__ __forceinline__ f4 square_of(const R (&row)[NT]) {
  return product_of(row, row);
}
// 1 / length of row c, from the diagonal.
__device__ __forceinline__ float unit_of(f4 square, bool normalize, Lane l) {
  float ss = square[0];
#pragma unroll
  for (int j = 1; j < 4; ++j) ss = (l.c & 3) == j ? square[j] : ss;
  ss = from_lane(ss, (l.c & 12) * 4 + l.c);
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
  const double sum = sum_up_to(gate), end = row_lane<kOf + 15>(sum);
  const uint64_t bits = __builtin_bit_cast(uint64_t, sum);
  Decay d;
  d.all = exp2_fast((float)end);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (20 * l.g + j), (int)(uint32_t)bits);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (20 * l.g + j), (int)(uint32_t)(bits >> 32));
    const double o = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    d.in[j] = exp2_fast((float)o);
    d.tail[j] = exp2_fast((float)(end - o));
    const float apart = (float)(sum - o);
    d.pair[j] = exp2_fast(l.in(j) < l.c ? apart : -apart);
  }
  return d;
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
  const int b = l.c >> 2;
  f4 ar, ac, lr, lc;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ar[j] = ac[j] = l.in(j) == l.c ? 1.0f : 0.0f;
    lr[j] = l.g == b ? L.row[j] : 0.0f;
    lc[j] = l.g == b ? L.col[j] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[0], row_lane<0 * kQuad>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[1], row_lane<1 * kQuad>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ar[j] = fmaf(-lr[2], row_lane<2 * kQuad>(ar[j]), ar[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[3], row_lane<3 * kQuad>(ac[j]), ac[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[2], row_lane<2 * kQuad>(ac[j]), ac[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) ac[j] = fmaf(-lc[1], row_lane<1 * kQuad>(ac[j]), ac[j]);
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
// f(r, j, address, columns that there are): p is the same in all lanes.
template <bool FULL, int NT, int VT, typename P, typename F>
__device__ __forceinline__ void each_row(P* p, const DeltaArgs& a, const Unit<NT, VT>& u, F&& f) {
  const int rows = opaque(a.keys - 4 * NT * u.l.g), wide = opaque(a.values - u.col());
  const uint32_t at = (uint32_t)opaque((4 * NT * u.l.g * a.values + u.col()) * 4);  // in bytes
  each<NT * 4>([&](auto n) {
    constexpr int r = n / 4, j = n % 4, row = NT * j + r;
    f(r, j, (P*)((uintptr_t)(p + row * a.values) + at), FULL ? VT : row < rows ? wide : 0);
  });
}
template <bool FULL, int NT, int VT>
__device__ __forceinline__ void load_state(const float* p, const DeltaArgs& a, const Unit<NT, VT>& u, f4 (&s)[NT][VT]) {
  each_row<FULL>(p, a, u, [&](int r, int j, const float* at, int wide) {
    Words<float, VT> x;
    if constexpr (FULL) x = load_whole<VT>(at);
    else x = load_words<VT>(at, wide);
#pragma unroll
    for (int t = 0; t < VT; ++t) s[r][t][j] = __uint_as_float(x.w[t]);
  });
}
template <bool FULL, int NT, int VT>
__device__ __forceinline__ void store_state(float* p, const DeltaArgs& a, const Unit<NT, VT>& u, const f4 (&s)[NT][VT]) {
  each_row<FULL>(p, a, u, [&](int r, int j, float* at, int wide) {
    float x[VT];
#pragma unroll
    for (int t = 0; t < VT; ++t) x[t] = s[r][t][j];
    store_row<VT>(at, wide, x);
  });
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

// The inverse of the triangular system, from the keys' inner products times what is
// left between their steps (`p`, both ways round).  Forward it is solved for u /
// beta, so that the gradient finds that without a division:
//   (1 + P beta) (u / beta) = v - g S0^T k;  the gradient solves (1 + beta P)^T.
template <bool GRAD>
__device__ __forceinline__ Both solve(f4 p, float beta, f4 bin, Lane l) {
  Both L;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    L.row[j] = l.in(j) < l.c ? p[j] * (GRAD ? beta : bin[j]) : 0.0f;
    L.col[j] = l.in(j) <= l.c ? 0.0f : p[j] * (GRAD ? bin[j] : beta);
  }
  return inverse(L, l);
}

// What a chunk's products need that does not depend on the state, made by one
// wavefront for all of a workgroup's: kGroup chunks at a time, side by side.
constexpr int kGroup = 4;
constexpr int kManyWaves = 1024;  // one for each SIMD
template <bool GRAD>
struct Solved {
  f4 t[64];                   // solve()'s rows; GRAD: columns
  f4 m[64];                   // scale G_ij (q_i . k_j), row i; GRAD: row j
  f4 pair[GRAD ? 64 : 1];     // what is left between two steps, zero across a cut
  double sums[16];
  float beta[16], kap[16], qap[16], in[16], tail[16];  // 1 / lengths; qap times the scale, but for GRAD
  float all;
  uint32_t cuts;
  int steps, pad;
};
__device__ __forceinline__ f4 of_rows(const float* p, Lane l) { return *reinterpret_cast<const f4*>(p + 4 * l.g); }

// Cuts are gates that let nothing through, which is the same as long as
// everything in the chunk is finite; where it is not, so is T or the result.
template <bool GRAD, typename T, int NT, bool FULL>
__device__ __forceinline__ void solve_chunk(const DeltaArgs& a, int t0, int env, int head, const Steps<T, NT, FULL>& q, const Steps<T, NT, FULL>& k, Lane l, Solved<GRAD>& z) {
  const Gates gates = load_gates(a, t0, env, head, l);
  const Span s{0, gates.steps};
  Raw<T> kr[NT], qr[NT];
  k.rows(t0, s, l, kr);
  q.rows(t0, s, l, qr);
  const f4 kk = square_of(kr);
  const float kap = unit_of(kk, a.normalize, l);
  const float qap = (a.normalize ? unit_of(square_of(qr), true, l) : 1.0f) * (GRAD ? 1.0f : a.scale);
  const f4 kq = GRAD ? product_of(qr, kr) : product_of(kr, qr);
  const double sum = sum_up_to(gates.gate), end = row_lane<kOf + 15>(sum);
  const uint32_t upto = (2u << l.c) - 1u;  // bits of the steps up to c
  if (l.g == 0) {
    z.sums[l.c] = sum;
    z.beta[l.c] = gates.beta, z.kap[l.c] = kap, z.qap[l.c] = qap;
    z.in[l.c] = gates.cuts & upto ? 0.0f : exp2_fast((float)sum);
    z.tail[l.c] = gates.cuts & ~upto ? 0.0f : exp2_fast((float)(end - sum));
    if (l.c == 0) z.all = gates.cuts ? 0.0f : exp2_fast((float)end), z.cuts = gates.cuts, z.steps = gates.steps;
  }
  const int lane = 16 * l.g + l.c;
  const f4 bin = of_rows(z.beta, l), kin = of_rows(z.kap, l), qin = of_rows(z.qap, l);
  f4 p, m, pair;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float apart = (float)(sum - z.sums[l.in(j)]);
    const bool same = ((upto ^ ((2u << l.in(j)) - 1u)) & gates.cuts) == 0u;
    pair[j] = same ? exp2_fast(l.in(j) < l.c ? apart : -apart) : 0.0f;
    p[j] = left_of(kk[j] * (kap * kin[j]), pair[j]);
    if constexpr (GRAD) m[j] = l.in(j) < l.c ? 0.0f : left_of(kq[j] * (kap * qin[j] * a.scale), pair[j]);
    else m[j] = l.in(j) <= l.c ? left_of(kq[j] * (qap * kin[j]), pair[j]) : 0.0f;
  }
  const Both t = solve<GRAD>(p, gates.beta, bin, l);
  z.t[lane] = GRAD ? t.col : t.row;
  z.m[lane] = m;
  if constexpr (GRAD) z.pair[lane] = pair;
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
// f(tiles of columns a wavefront takes): two share what does not depend on the
// columns, but registers do for no more with 128 keys, and a few heads need all the
// wavefronts that they can make.
constexpr int slabs_of(int values, int cols) { return (values + 16 * cols - 1) / (16 * cols); }
template <int MOST, typename F>
void by_columns(const DeltaArgs& a, F&& f) {
  if (MOST > 1 && (int64_t)a.envs * a.heads * slabs_of(a.values, 2) >= kManyWaves) f(std::integral_constant<int, MOST>{});
  else f(std::integral_constant<int, 1>{});
}
template <typename F>
void by_truth(bool yes, F&& f) {
  if (yes) f(std::true_type{});
  else f(std::false_type{});
}

}  // namespace
}  // namespace gbx
