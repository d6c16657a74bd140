// gbx_sample.hip -- actions drawn from logits with given random numbers.
//
// With m the row's largest logit, w_i = exp((x_i - m) / temperature), and the
// actions from the likeliest on, the lowest index first among equals, a row keeps
// its first top_k, of those the fewest that hold top_p of their weight, and of
// those all with w_i >= min_p; at least one.  All three cuts are a beginning of
// that order, so what stays is "all larger logits than some value, and the first
// few of its equals".  The action is then the first index at which the running
// sum of the kept weights, by index, passes uniform * their sum, and logp the
// logarithm of its share.
//
// Weights and sums are in 64 bits: a random number or a cut falls between two
// actions whose border a 32-bit sum of a few thousand weights misses by up to
// 1e-4 of a weight, and a policy's update divides by the probability that the
// action was drawn with.
#include "gbx_policy.h"

#include <type_traits>

namespace gbx {
namespace {

// A row's options, with what keeps one action alone as top_k = 1.
struct Cuts {
  double heat, p, least;  // heat 0: the largest logit
  int k;                  // 0: all
};
__device__ __forceinline__ Cuts cuts_of(const SampleArgs& a, int64_t row) {
  Cuts c;
  c.heat = a.temperatures ? (double)a.temperatures[row] : a.temperature;
  c.p = a.top_ps ? (double)a.top_ps[row] : a.top_p;
  c.least = a.min_ps ? (double)a.min_ps[row] : a.min_p;
  c.k = a.top_ks ? a.top_ks[row] : a.top_k;
  if (!(c.heat > 0.0)) c.heat = 0.0;
  if (c.heat == 0.0 || !(c.p > 0.0) || !(c.least <= 1.0)) c.k = 1;
  if (c.k < 0 || c.k >= a.actions) c.k = 0;
  if (c.k == 1 || c.p >= 1.0) c.p = 1.0;
  if (c.k == 1) c.least = 0.0;
  return c;
}
// NaN stands for an action that is not allowed, as -infinity does.
template <typename T>
__device__ __forceinline__ float logit(T x) {
  const float v = (float)x;
  return v == v ? v : -INFINITY;
}
__device__ __forceinline__ double weight_of(float x, float most, double heat) {
  if (x == -INFINITY) return 0.0;
  if (x == most) return 1.0;
  if (most == INFINITY || heat == 0.0) return 0.0;
  return exp(((double)x - (double)most) / heat);
}
__device__ __forceinline__ void write(const SampleArgs& a, int64_t row, int action, double share) {
  a.action[row] = action;
  a.logp[row] = (float)log(share);
}
// a row without an action that is allowed
__device__ __forceinline__ void write_none(const SampleArgs& a, int64_t row) {
  a.action[row] = -1;
  a.logp[row] = __builtin_nanf("");
}

// Up to 64 actions: L lanes hold a row, one action each, and compare each with each.
template <typename T, int L>
__global__ __launch_bounds__(256) void sample_few_kernel(SampleArgs a) {
  const int i = threadIdx.x % L, base = (threadIdx.x & 63) / L * L;
  const int64_t row = block_id() * (256 / L) + threadIdx.x / L;
  if (row >= a.rows) return;
  const float x = i < a.actions ? logit(((const T*)a.logits)[row * a.stride + i]) : -INFINITY;
  float most = x;
#pragma unroll
  for (int m = 1; m < L; m <<= 1) most = fmaxf(most, __shfl_xor(most, m, L));
  if (most == -INFINITY) {
    if (i == 0) write_none(a, row);
    return;
  }
  const Cuts c = cuts_of(a, row);
  double w = weight_of(x, most, c.heat);
  if (c.k || c.p < 1.0) {
    int rank = 0;
    for (int n = 1; n < L; ++n) {
      const int j = (i + n) % L;
      const float o = __shfl(x, j, L);
      rank += o > x || (o == x && j < i);
    }
    if (c.k && rank >= c.k) w = 0.0;
    if (c.p < 1.0) {
      double before = 0.0, all = w;
      for (int n = 1; n < L; ++n) {
        const int j = (i + n) % L;
        const double o = __shfl(w, j, L);
        all += o;
        before += __shfl(rank, j, L) < rank ? o : 0.0;
      }
      if (rank > 0 && !(before < c.p * all)) w = 0.0;
    }
  }
  if (!(w >= c.least)) w = 0.0;
  double run = w;
#pragma unroll
  for (int m = 1; m < L; m <<= 1) {
    const double o = __shfl_up(run, m, L);
    run += i >= m ? o : 0.0;
  }
  const double all = __shfl(run, L - 1, L);
  constexpr uint64_t kRow = L == 64 ? ~0ull : (1ull << L) - 1;
  const uint64_t kept = __ballot(w > 0.0) >> base & kRow;
  const uint64_t past = __ballot(w > 0.0 && run > (double)a.uniform[row] * all) >> base & kRow;
  if (i == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(kept))) write(a, row, i, w / all);
}

// ---- longer rows: a workgroup each

// The workgroup's wavefronts, and one place of LDS for each.
template <int THREADS>
struct Group {
  static constexpr int kWaves = THREADS / 64;
  double* lds;  // kWaves
  template <typename V, typename F>
  __device__ __forceinline__ V all(V v, F&& f) const {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = f(v, __shfl_xor(v, m, 64));
    if constexpr (kWaves > 1) {
      V* at = reinterpret_cast<V*>(lds);
      __syncthreads();  // the last use has been read
      if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
      __syncthreads();
      v = at[0];
#pragma unroll
      for (int n = 1; n < kWaves; ++n) v = f(v, at[n]);
    }
    return v;
  }
  // sum of the threads before this one, and of all
  template <typename V>
  __device__ __forceinline__ V before(V v, V& total) const {
    const int lane = threadIdx.x & 63;
    V run = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const V o = __shfl_up(run, m, 64);
      run += lane >= m ? o : V(0);
    }
    V first = V(0);
    total = __shfl(run, 63, 64);
    if constexpr (kWaves > 1) {
      V* at = reinterpret_cast<V*>(lds);
      __syncthreads();
      if (lane == 0) at[threadIdx.x >> 6] = total;
      __syncthreads();
      total = V(0);
#pragma unroll
      for (int n = 0; n < kWaves; ++n) {
        first += n < (int)(threadIdx.x >> 6) ? at[n] : V(0);
        total += at[n];
      }
    }
    run = __shfl_up(run, 1, 64);
    return first + (lane ? run : V(0));
  }
};

// A logit as a whole number of the same order, in the bits that its type fills.
template <typename T>
constexpr int kKeyBits = sizeof(T) == 4 ? 32 : std::is_same<T, _Float16>::value ? 19 : 16;
template <typename T>
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
  return (b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) >> (32 - kKeyBits<T>);
}

// HELD consecutive logits a thread stay in registers (0: rows of any length,
// read again at each turn).  Cuts are found by halving the range of keys, one
// count or sum over the row a bit.
template <typename T, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ double lds[THREADS / 64];
  __shared__ int choice[2];
  const Group<THREADS> group{lds};
  const int64_t row = block_id();
  if (row >= a.rows) return;
  const T* logits = (const T*)a.logits + row * a.stride;
  const int each = HELD ? HELD : (a.actions + THREADS - 1) / THREADS, first = threadIdx.x * each;
  float held[HELD ? HELD : 1];
  if constexpr (HELD > 0) {
    load_row<HELD>(logits + first, a.actions - first, held);
#pragma unroll
    for (int e = 0; e < HELD; ++e) held[e] = first + e < a.actions ? logit(held[e]) : -INFINITY;
  }
  auto over = [&](auto&& f) {  // f(place, logit) of this thread's
    if constexpr (HELD > 0) {
#pragma unroll
      for (int e = 0; e < HELD; ++e) f(e, held[e]);
    } else {
      for (int e = 0; e < each && first + e < a.actions; ++e) f(e, logit(logits[first + e]));
    }
  };
  auto add = [](auto p, auto q) { return p + q; };
  float most = -INFINITY;
  over([&](int, float x) { most = fmaxf(most, x); });
  most = group.all(most, [](float p, float q) { return fmaxf(p, q); });
  if (most == -INFINITY) {
    if (threadIdx.x == 0) write_none(a, row);
    return;
  }
  const Cuts c = cuts_of(a, row);
  double weights[HELD ? HELD : 1];
  if constexpr (HELD > 0) {
#pragma unroll
    for (int e = 0; e < HELD; ++e) weights[e] = weight_of(held[e], most, c.heat);
  }
  auto weight = [&](int e, float x) {
    if constexpr (HELD > 0) return weights[e];
    else return weight_of(x, most, c.heat);
  };
  // what stays: keys above `edge`, and the first `equals` of those at it
  uint32_t edge = 0;
  int equals = a.actions;
  auto count_from = [&](uint32_t t) {
    int n = 0;
    over([&](int, float x) { n += key_of<T>(x) >= t; });
    return group.all(n, add);
  };
  auto mass_from = [&](uint32_t t) {
    double n = 0.0;
    over([&](int e, float x) { n += key_of<T>(x) >= t ? weight(e, x) : 0.0; });
    return group.all(n, add);
  };
  if (c.k) {
    for (int bit = kKeyBits<T> - 1; bit >= 0; --bit)
      if (count_from(edge | 1u << bit) >= c.k) edge |= 1u << bit;
    equals = c.k - count_from(edge + 1u);
  }
  if (c.p < 1.0) {
    // the logit at an edge: weights of equals are equal
    auto at_edge = [&](uint32_t t, double& w) {
      w = 0.0;
      int n = 0;
      over([&](int e, float x) {
        if (key_of<T>(x) == t) {
          w = weight(e, x);
          ++n;
        }
      });
      w = group.all(w, [](double p, double q) { return p > q ? p : q; });
      return group.all(n, add);
    };
    double w;
    const int there = at_edge(edge, w);
    if (equals > there) equals = there;
    const double above = mass_from(edge + 1u), need = c.p * (above + equals * w);
    if (above >= need) {  // the edge goes up
      uint32_t t = 0;
      for (int bit = kKeyBits<T> - 1; bit >= 0; --bit)
        if (mass_from(t | 1u << bit) >= need) t |= 1u << bit;
      edge = t;
      equals = at_edge(edge, w);
    }
    const double over_edge = mass_from(edge + 1u);
    int fewest = 0;  // equals that come before what is needed is there
    for (int bit = 20; bit >= 0; --bit)
      if (fewest + (1 << bit) <= equals && over_edge + (fewest + (1 << bit) - 1) * w < need) fewest += 1 << bit;
    equals = fewest < 1 ? 1 : fewest;
  }
  int mine = 0, there;
  over([&](int, float x) { mine += key_of<T>(x) == edge; });
  int rank = group.before(mine, there);
  auto kept = [&](int e, float x, int& rank) {
    const uint32_t key = key_of<T>(x);
    const double w = weight(e, x);
    const bool stays = key > edge || (key == edge && rank < equals);
    rank += key == edge;
    return stays && w >= c.least ? w : 0.0;
  };
  double sum = 0.0, all;
  {
    int r = rank;
    over([&](int e, float x) { sum += kept(e, x, r); });
  }
  const double start = group.before(sum, all);
  if (threadIdx.x < 2) choice[threadIdx.x] = threadIdx.x ? -1 : a.actions;
  __syncthreads();
  const double target = (double)a.uniform[row] * all;
  {
    double run = start;
    int r = rank, past = a.actions, last = -1;
    over([&](int e, float x) {
      const double w = kept(e, x, r);
      run += w;
      if (w > 0.0) {
        last = first + e;
        if (past == a.actions && run > target) past = first + e;
      }
    });
    if (past < a.actions) atomicMin(&choice[0], past);
    if (last >= 0) atomicMax(&choice[1], last);
  }
  __syncthreads();
  const int action = choice[0] < a.actions ? choice[0] : choice[1];
  over([&](int e, float x) {
    if (first + e == action) write(a, row, action, weight(e, x) / all);
  });
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    auto few = [&](auto lanes) { hipLaunchKernelGGL((sample_few_kernel<T, lanes>), wide_grid((a.rows + 256 / lanes - 1) / (256 / lanes)), dim3(256), 0, st, a); };
    auto many = [&](auto threads, auto held) { hipLaunchKernelGGL((sample_kernel<T, threads, held>), wide_grid(a.rows), dim3(threads), 0, st, a); };
    using std::integral_constant;
    if (a.actions <= 8) few(integral_constant<int, 8>{});
    else if (a.actions <= 16) few(integral_constant<int, 16>{});
    else if (a.actions <= 32) few(integral_constant<int, 32>{});
    else if (a.actions <= 64) few(integral_constant<int, 64>{});
    else if (a.actions <= 512) many(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else if (a.actions <= 2048) many(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else if (a.actions <= 16384) many(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
    else many(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
  });
  return hipGetLastError();
}

}  // namespace gbx
