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
  if (c.k == 1) c.p = 1.0, c.least = 0.0;  // before k becomes `all`, as it does where there is one action
  if (c.k < 0 || c.k >= a.actions) c.k = 0;
  if (c.p >= 1.0) c.p = 1.0;
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

// What lane n of the next L lanes holds (n counts from lane i where rows share a
// wavefront; with a row a wavefront it is the same lane for all, read as a scalar).
template <int L>
__device__ __forceinline__ int turn_of(int i, int n) { return L == 64 ? n : (i + n) % L; }
template <int L>
__device__ __forceinline__ int held_by(int v, int j) {
  if constexpr (L == 64) return __builtin_amdgcn_readlane(v, j);
  else return __shfl(v, j, L);
}
template <int L>
__device__ __forceinline__ float held_by(float v, int j) { return __int_as_float(held_by<L>(__float_as_int(v), j)); }
template <int L>
__device__ __forceinline__ double held_by(double v, int j) {
  return __hiloint2double(held_by<L>(__double2hiint(v), j), held_by<L>(__double2loint(v), j));
}

// Draws from up to 64 logits in the order of their indexes: L lanes hold one each
// (-infinity where there are fewer) and compare each with each.  `full`: the weight
// of the whole row; negative: that of these.
template <int L>
__device__ __forceinline__ void draw_few(const SampleArgs& a, int64_t row, const Cuts& c, float x, float most, int index, double full) {
  const int i = threadIdx.x % L, base = (threadIdx.x & 63) / L * L;
  double w = weight_of(x, most, c.heat);
  if (c.k || c.p < 1.0) {
    int rank = 0;
#pragma unroll 8
    for (int n = 0; n < L; ++n) {
      const int j = turn_of<L>(i, n);
      const float o = held_by<L>(x, j);
      rank += o > x || (o == x && j < i);
    }
    if (c.k && rank >= c.k) w = 0.0;
    if (c.p < 1.0) {
      double before = 0.0, all = 0.0;
#pragma unroll 8
      for (int n = 0; n < L; ++n) {
        const int j = turn_of<L>(i, n);
        const double o = held_by<L>(w, j);
        all += o;
        before += held_by<L>(rank, j) < rank ? o : 0.0;
      }
      if (rank > 0 && !(before < c.p * (c.k || full < 0.0 ? all : full))) w = 0.0;
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
  if (i == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(kept))) write(a, row, index, w / all);
}

// Up to 64 actions: L lanes a row.  Bound by a launch at 64 x 8 (6.4 us).  131,072 x
// 8 with every option its own a row takes 12.8 us, of which reading 8 MB is 2: every lane
// goes over its row's others by exchanges, so the sums for ranks and shares, in 64 bits,
// are made eight times, and the logarithm and the division for one lane in eight.
template <typename T, int L>
__global__ __launch_bounds__(256) void sample_few_kernel(SampleArgs a) {
  const int i = threadIdx.x % L;
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
  draw_few<L>(a, row, cuts_of(a, row), x, most, i, -1.0);
}

// ---- longer rows: a workgroup each

// Sums over a workgroup, in one order.  Two halves of LDS in turn: what one
// call writes is not what the call before may still read.
template <int THREADS>
struct Group {
  static constexpr int kWaves = THREADS / 64;
  double* lds;  // 2 * kWaves
  int turn;
  template <typename V>
  __device__ __forceinline__ const V* share(V v) {
    V* at = reinterpret_cast<V*>(lds + (turn ^= kWaves));
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    return at;
  }
  template <typename V, typename F>
  __device__ __forceinline__ V all(V v, F&& f) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = f(v, __shfl_xor(v, m, 64));
    if constexpr (kWaves > 1) {
      const V* at = share(v);
      v = at[0];
#pragma unroll
      for (int n = 1; n < kWaves; ++n) v = f(v, at[n]);
    }
    return v;
  }
  template <typename V>
  __device__ __forceinline__ V sum(V v) {
    return all(v, [](V p, V q) { return p + q; });
  }
  // sum of the threads before this one, and of all
  template <typename V>
  __device__ __forceinline__ V before(V v, V& total) {
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
      const V* at = share(total);
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
  // threads for which it holds
  __device__ __forceinline__ int count(bool yes) {
    int n = __builtin_popcountll(__ballot(yes));
    if constexpr (kWaves > 1) {
      const int* at = share(n);
      n = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) n += at[w];
    }
    return n;
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

// Draws from the row's logits, or from those of them that can stay, which
// over(f) hands to f(logit, weight, index) thread by thread in the order of
// their indexes.  `full`: the weight of all.  Cuts are found by halving the range
// of keys, one count or sum over the row a bit.
template <typename T, int THREADS, typename Over>
__device__ __forceinline__ void draw(const SampleArgs& a, int64_t row, const Cuts& c, double full, Group<THREADS>& group, int* choice, Over&& over) {
  // what stays: keys above `edge`, and the first `equals` of those at it
  uint32_t edge = 0;
  int equals = a.actions;
  auto count_from = [&](uint32_t t) {
    int n = 0;
    over([&](float x, double, int) { n += key_of<T>(x) >= t; });
    return group.sum(n);
  };
  auto mass_from = [&](uint32_t t) {
    double n = 0.0;
    over([&](float x, double w, int) { n += key_of<T>(x) >= t ? w : 0.0; });
    return group.sum(n);
  };
  if (c.k) {
    for (int bit = kKeyBits<T> - 1; bit >= 0; --bit)
      if (count_from(edge | 1u << bit) >= c.k) edge |= 1u << bit;
    equals = c.k - count_from(edge + 1u);
  }
  if (c.p < 1.0) {
    auto at_edge = [&](uint32_t t, double& weight) {  // equals have equal weights
      weight = 0.0;
      int n = 0;
      over([&](float x, double w, int) {
        if (key_of<T>(x) == t) {
          weight = w;
          ++n;
        }
      });
      weight = group.all(weight, [](double p, double q) { return p > q ? p : q; });
      return group.sum(n);
    };
    double w;
    const int there = at_edge(edge, w);
    if (equals > there) equals = there;
    const double above = mass_from(edge + 1u), need = c.p * (c.k ? above + equals * w : full);
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
  over([&](float x, double, int) { mine += key_of<T>(x) == edge; });
  const int rank = group.before(mine, there);
  auto kept = [&](float x, double w, int& r) {
    const uint32_t key = key_of<T>(x);
    const bool stays = key > edge || (key == edge && r < equals);
    r += key == edge;
    return stays && w >= c.least ? w : 0.0;
  };
  double sum = 0.0, all;
  int r = rank;
  over([&](float x, double w, int) { sum += kept(x, w, r); });
  if (threadIdx.x < 2) choice[threadIdx.x] = threadIdx.x ? -1 : a.actions;
  double run = group.before(sum, all);
  if constexpr (THREADS == 64) __syncthreads();
  const double target = (double)a.uniform[row] * all;
  int past = a.actions, last = -1;
  r = rank;
  over([&](float x, double w, int index) {
    w = kept(x, w, r);
    run += w;
    if (w > 0.0) {
      last = index;
      if (past == a.actions && run > target) past = index;
    }
  });
  if (past < a.actions) atomicMin(&choice[0], past);
  if (last >= 0) atomicMax(&choice[1], last);
  __syncthreads();
  const int action = choice[0] < a.actions ? choice[0] : choice[1];
  over([&](float, double w, int index) {
    if (index == action) write(a, row, action, w / all);
  });
}

// HELD consecutive logits a thread stay in registers (0: rows of any length, read
// again at each turn), and with KEEP their weights.
//
// The search for a cut goes over the row once a bit, so where few logits can stay
// they are put together first, one a thread: those from the k-th largest of the
// threads' own largest on hold the k largest of the row; and those that weigh
// less than (1 - p) / actions of the row are together less than what top_p leaves
// out.  512 x 32,768 in 16 bits, top_k 50, top_p 0.95: 20 us, where reading the
// row once is 7; the rest are the 20 turns of a workgroup's counts, each a barrier
// that two workgroups a compute unit cannot hide.
template <typename T, int THREADS, int HELD, bool KEEP>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ double lds[2 * THREADS / 64];
  __shared__ float some[THREADS];
  __shared__ int places[THREADS], order[THREADS], found, choice[2];
  Group<THREADS> group{lds, 0};
  const int64_t row = block_id();
  if (row >= a.rows) return;
  const T* logits = (const T*)a.logits + row * a.stride;
  // (whole vectors of 8 a thread)
  const int each = HELD ? HELD : ((a.actions + THREADS - 1) / THREADS + 7) & ~7, first = threadIdx.x * each;
  auto eight = [&](int e, float (&x)[8]) {
    load_row<8>(logits + e, a.actions - e, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = e + i < a.actions ? logit(x[i]) : -INFINITY;
  };
  float held[HELD ? HELD : 1];
  double weights[KEEP ? HELD : 1];
  // f(logit, index) in any order: what is not held is read in whole lines, four
  // vectors a thread under way together
  auto logits_of = [&](auto&& f) {
    if constexpr (HELD > 0) {
#pragma unroll
      for (int e = 0; e < HELD; ++e) f(held[e], first + e);
    } else {
      constexpr int kStep = THREADS * 8;
      int e = threadIdx.x * 8;
      for (; e + 3 * kStep + 8 <= a.actions; e += 4 * kStep) {
        float x[4][8];
#pragma unroll
        for (int n = 0; n < 4; ++n) load_row<8>(logits + e + n * kStep, 8, x[n]);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int i = 0; i < 8; ++i) f(logit(x[n][i]), e + n * kStep + i);
      }
      for (; e < a.actions; e += kStep) {
        float x[8];
        eight(e, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) f(x[i], e + i);
      }
    }
  };
  float most = -INFINITY;
  if constexpr (HELD > 0) {
#pragma unroll
    for (int e = 0; e < HELD; e += 8) {
      float x[8];
      eight(first + e, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) held[e + i] = x[i];
    }
  }
  logits_of([&](float x, int) { most = fmaxf(most, x); });
  if (threadIdx.x == 0) found = 0;
  const uint32_t own = key_of<T>(most);
  most = group.all(most, [](float p, float q) { return fmaxf(p, q); });
  if (most == -INFINITY) {
    if (threadIdx.x == 0) write_none(a, row);
    return;
  }
  const Cuts c = cuts_of(a, row);
  auto over = [&](auto&& f) {  // f(logit, weight, index), in order
    if constexpr (KEEP) {
#pragma unroll
      for (int e = 0; e < HELD; ++e) f(held[e], weights[e], first + e);
    } else {
      for (int e = first; e < first + each && e < a.actions; e += 8) {
        float x[8];
        eight(e, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) f(x[i], weight_of(x[i], most, c.heat), e + i);
      }
    }
  };
  auto any = [&](auto&& f) {  // the same in any order
    if constexpr (KEEP) over(f);
    else logits_of([&](float x, int index) { f(x, weight_of(x, most, c.heat), index); });
  };
  // Draws from the logits that each_of(f) hands to f, if there are no more of
  // them than threads.  They come as they come, and are ordered by their indexes.
  auto from_some = [&](double full, auto&& each_of) {
    each_of([&](float x, int index) {
      const int at = atomicAdd(&found, 1);
      if (at < THREADS) {
        some[at] = x;
        places[at] = index;
      }
    });
    __syncthreads();
    const int count = found;
    if (count > THREADS) return false;
    const bool live = (int)threadIdx.x < count;
    float x = live ? some[threadIdx.x] : -INFINITY;
    int index = live ? places[threadIdx.x] : a.actions;
    if (live) {
      int rank = 0;
#pragma unroll 8
      for (int n = 0; n < count; ++n) rank += places[n] < index;
      order[rank] = threadIdx.x;
    }
    __syncthreads();
    if (live) {
      const int from = order[threadIdx.x];
      x = some[from];
      index = places[from];
    }
    if (count <= 64) {
      if (threadIdx.x < 64) draw_few<64>(a, row, c, x, most, index, full);
      return true;
    }
    const double w = weight_of(x, most, c.heat);
    draw<T>(a, row, c, full, group, choice, [&](auto&& f) { f(x, w, index); });
    return true;
  };
  if (c.k && c.k <= THREADS) {
    uint32_t from = 0;
    for (int bit = kKeyBits<T> - 1; bit >= 0; --bit)
      if (group.count(own >= (from | 1u << bit)) >= c.k) from |= 1u << bit;
    if (from_some(0.0, [&](auto&& f) {
          logits_of([&](float x, int index) {
            if (key_of<T>(x) >= from && x > -INFINITY) f(x, index);
          });
        }))
      return;
  }
  if constexpr (KEEP) {
#pragma unroll
    for (int e = 0; e < HELD; ++e) weights[e] = weight_of(held[e], most, c.heat);
  }
  double full = 0.0;
  if (!c.k && (c.p < 1.0 || c.least > 0.0)) {
    double least = c.least;
    if (c.p < 1.0) {
      any([&](float, double w, int) { full += w; });
      full = group.sum(full);
      least = fmax(least, (1.0 - c.p) * full / a.actions * (1.0 - 1e-9));
    }
    if (from_some(full, [&](auto&& f) {
          any([&](float x, double w, int index) {
            if (w >= least && w > 0.0) f(x, index);
          });
        }))
      return;
  }
  draw<T>(a, row, c, full, group, choice, over);
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    auto few = [&](auto lanes) { hipLaunchKernelGGL((sample_few_kernel<T, lanes>), wide_grid((a.rows + 256 / lanes - 1) / (256 / lanes)), dim3(256), 0, st, a); };
    auto many = [&](auto threads, auto held) { hipLaunchKernelGGL((sample_kernel<T, threads, held, (held > 0)>), wide_grid(a.rows), dim3(threads), 0, st, a); };
    // With one top_k for all, every row finds few logits to draw from, and only
    // their weights are needed: a long row is then read twice in whole lines and
    // not held (512 x 32,768 in 16 bits, top_k 50: 20 us, held 70).  Other cuts
    // may leave the whole row to search, with a weight for each turn, and hold it
    // (the same with top_p alone: 248 us, read again at each turn 893).  A top_k of
    // each row's own takes the held form, 35 us: a row's may be 0.
    const bool cut = !a.top_ks && a.top_k > 0 && a.top_k <= 512;
    using std::integral_constant;
    if (a.actions <= 8) few(integral_constant<int, 8>{});
    else if (a.actions <= 16) few(integral_constant<int, 16>{});
    else if (a.actions <= 32) few(integral_constant<int, 32>{});
    else if (a.actions <= 64) few(integral_constant<int, 64>{});
    else if (a.actions <= 512) many(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else if (a.actions <= 2048) many(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else if (a.actions <= 8192) many(integral_constant<int, 512>{}, integral_constant<int, 16>{});
    else if (a.actions <= 32768 && !cut) many(integral_constant<int, 512>{}, integral_constant<int, 64>{});
    else if (a.actions <= 32768) many(integral_constant<int, 512>{}, integral_constant<int, 0>{});
    else many(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
  });
  return hipGetLastError();
}

}  // namespace gbx
