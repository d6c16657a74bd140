// gbx_conv.hip -- short causal convolution along the steps of each env and
// channel, its gradient and its single step.
//
//   pre[t] = bias + sum over j < width of weight[width - 1 - j] * x[t - j],   y = silu(pre) or pre
//
// where x[t - j] counts only if no episode begins in (t - j, t], and steps
// before the first one come from the carried state.  A lane walks along the
// steps with the last width - 1 inputs of 8 channels in registers, so each
// input is read once; the kernels are bound by memory.
#include <algorithm>

#include "gbx_policy.h"

namespace gbx {
namespace {

constexpr int kThreads = 256;
constexpr int kMinSteps = 16;  // of a piece of the steps: its lead-in of up to 3 is read twice
// Lanes that keep the memory busy, times the channels of each: rows of fewer
// are cut along the steps.
constexpr int64_t kBusy = 256 * 2048 * 8;

// Shape of the launch: a workgroup is `lanes` groups of V neighbouring channels
// by 256 / lanes rows; a row is one env and one piece of the steps.
struct Shape {
  int groups, shift, chunk, chunks;  // groups of channels; log2 of lanes in a row; steps of a piece, pieces
  uint32_t rows;                     // below 2^28: only rows of few lanes are cut
};
Shape shape_of(int steps, int envs, int dim, int v) {
  Shape s;
  s.groups = (dim + v - 1) / v;
  s.shift = 0;
  while (s.shift < 6 && (1 << s.shift) < s.groups) ++s.shift;
  const int64_t want = std::max<int64_t>(1, kBusy / ((int64_t)envs * s.groups * v));
  s.chunk = (int)std::max<int64_t>(kMinSteps, (steps + want - 1) / want);
  s.chunks = (steps + s.chunk - 1) / s.chunk;
  s.rows = (uint32_t)((int64_t)envs * s.chunks);
  return s;
}

// Neighbouring channels of a row, as they lie.  WHOLE: every group has V; where
// the channels are no multiple of V the last group begins V before the end and
// shares some with the group before it.  Both compute and write the same
// values there (one lane with part of a group would load and store element by
// element: 1,023 channels forward and backward 699 us).
template <typename T, int V>
struct Packed {
  T v[V];
};
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void fetch_row(const T* p, int n, Packed<T, V>& r) {
  if (WHOLE || n >= V) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = k < n ? p[k] : (T)0.0f;
  }
}

// The inputs before step t0 of one env and V channels, oldest first, zero where
// an episode begins between them and step t0 - 1; `age`: steps since the
// episode began, no more than W.
template <int W, int V, typename T>
__device__ __forceinline__ void lead_in(const ConvArgs& a, int env, int t0, int c, float (&win)[W - 1][V], int& age) {
  const int n = a.dim - c;
  age = W;
#pragma unroll
  for (int i = 0; i < W - 1; ++i) {
    const int t = t0 - (W - 1) + i;
    if (t < 0) {
      if (a.state) load_row<V>((const T*)a.state + ((int64_t)env * (W - 1) + (t + W - 1)) * a.dim + c, n, win[i]);
      else {
#pragma unroll
        for (int k = 0; k < V; ++k) win[i][k] = 0.0f;
      }
    } else {
      load_row<V>((const T*)a.x + (int64_t)t * a.x_step + (int64_t)env * a.x_env + c, n, win[i]);
    }
  }
  if (a.resets) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      const int t = t0 - (W - 1) + i;
      const bool begins = t >= 0 && a.resets[(int64_t)t * a.envs + env];
      age = begins ? 0 : min(age + 1, W);
#pragma unroll
      for (int j = 0; j < i; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) win[j][k] = begins ? 0.0f : win[j][k];
    }
  }
}

// the weights of neighbouring channels lie together
template <int W, int V>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int c, float (&w)[W][V], float (&bias)[V]) {
  float row[W * V];
  load_row<W * V>(a.weight + (int64_t)c * W, (a.dim - c) * W, row);
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][k] = row[k * W + j];
  if (a.bias) {
    load_row<V>(a.bias + c, a.dim - c, bias);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) bias[k] = 0.0f;
  }
}

// Where an episode begins in some lane, that lane's older inputs become zero.
// A branch that most wavefronts skip: selections would cost each step as much
// as the products do.
template <int N, int V>
__device__ __forceinline__ void forget(bool begins, float (&win)[N][V]) {
  if (__ballot(begins)) {
    asm volatile("");
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) win[j][k] = begins ? 0.0f : win[j][k];
  }
}
template <int W, int V>
__device__ __forceinline__ float convolve(const float (&w)[W][V], const float (&win)[W - 1][V], float in, float bias, int k) {
  float pre = bias;
#pragma unroll
  for (int j = 0; j < W - 1; ++j) pre = fmaf(w[j][k], win[j][k], pre);
  return fmaf(w[W - 1][k], in, pre);
}
template <int W, int V>
__device__ __forceinline__ void move_on(float (&win)[W - 1][V], float in, int k) {
#pragma unroll
  for (int j = 0; j + 1 < W - 1; ++j) win[j][k] = win[j + 1][k];
  win[W - 2][k] = in;
}

constexpr int kForward = 8, kBackward = 4;  // channels of a lane: 16 or 8 bytes of a 16-bit type

// First channel of a group.
template <int V, bool WHOLE>
__device__ __forceinline__ int channel_of(int group, int dim) {
  return WHOLE && group * V > dim - V ? dim - V : group * V;
}

// A row's place: its first channel group's lane, env and piece of the steps.
// WIDE: a wavefront is one row, and what depends on the row alone is scalar.
template <bool WIDE>
__device__ __forceinline__ uint32_t row_of(const Shape& s) {
  const int in = threadIdx.x >> s.shift;
  return blockIdx.x * (kThreads >> s.shift) + (WIDE ? __builtin_amdgcn_readfirstlane(in) : in);
}

// Bound by memory: 128 steps x 1,024 envs x 1,024 channels in bf16 with episodes
// that begin in one step of a hundred move 537 MB in 113 us (4.7 TB/s; a copy
// reaches 4.9), 4 steps of 131,072 envs x 512 with a carried state 1.88 GB in 366
// us (5.1).  Pieces of the steps are long where there are many rows (the lead-in is
// read twice) and no shorter than 16 steps where there are few.
template <typename T, int W, bool WHOLE, bool WIDE>
__global__ __launch_bounds__(kThreads) void conv_kernel(ConvArgs a, Shape s) {
  constexpr int V = kForward, kAhead = 4;  // steps whose loads are in flight while four others are worked on
  const int lanes = 1 << s.shift;
  const int group = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
  const uint32_t row = row_of<WIDE>(s);
  if (group >= s.groups || row >= s.rows) return;
  const int env = (int)(row % (uint32_t)a.envs), part = (int)(row / (uint32_t)a.envs);
  const int c = channel_of<V, WHOLE>(group, a.dim), n = a.dim - c;
  const int t0 = part * s.chunk, t1 = min(t0 + s.chunk, a.steps);
  const T* x = (const T*)a.x + (int64_t)t0 * a.x_step + (int64_t)env * a.x_env;
  const uint8_t* resets = a.resets + (int64_t)t0 * a.envs + env;
  T* y = (T*)a.y + ((int64_t)t0 * a.envs + env) * a.dim;
  Packed<T, V> next[kAhead];
  uint8_t next_begins[kAhead];
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int on = t + i + 1 < t1;  // the last row is loaded again past the end
      fetch_row<WHOLE>(x + c, n, next[i]);
      x += on ? a.x_step : 0;
      next_begins[i] = 0;
      if (a.resets) {
        next_begins[i] = *resets;
        resets += on ? a.envs : 0;
      }
    }
  };
  fetch(t0);
  float w[W][V], bias[V], win[W - 1][V];
  int age;
  load_weights<W>(a, c, w, bias);
  lead_in<W, V, T>(a, env, t0, c, win, age);
  for (int t = t0; t < t1; t += kAhead) {
    Packed<T, V> in[kAhead];
    bool begins[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      in[i] = next[i];
      begins[i] = (WIDE ? __builtin_amdgcn_readfirstlane((int)next_begins[i]) : (int)next_begins[i]) != 0;
    }
    if (t + kAhead < t1) fetch(t + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t + i >= t1) break;
      forget(begins[i], win);
      float out[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = (float)in[i].v[k], pre = convolve<W, V>(w, win, v, bias[k], k);
        out[k] = a.silu ? pre * sigmoid(pre) : pre;
        move_on<W, V>(win, v, k);
      }
      store_row<V>(y + c, WHOLE ? V : n, out);
      y += (int64_t)a.envs * a.dim;
    }
  }
  if (t1 == a.steps) {
    T* last = (T*)a.last + (int64_t)env * (W - 1) * a.dim + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<V>(last + (int64_t)j * a.dim, n, win[j]);
  }
}

// With d[t] = dy[t] * silu'(pre[t]), pre computed again from x:
//   dx[t] = sum over j of weight[width - 1 - j] * d[t + j], as far as the episode goes,
//   dweight[width - 1 - j] = sum of d[t] * x[t - j],   dbias = sum of d[t].
// The lane walks forward and keeps width sums of dx under way, as it keeps the
// inputs; a piece of the steps goes width - 1 steps past its end to finish
// its own.  dweight and dbias of a workgroup's rows are added in LDS and
// written as one row of partial sums.
//
// 128 steps x 1,024 envs x 1,024 channels in bf16 move 805 MB in 191 us (4.2
// TB/s): memory and the vector units (127 us of issue) take turns, with 4
// channels in a lane.  The partial sums grow with the rows: where an env has few
// steps they and their sum are much of the work (4 steps of 131,072 envs x 512
// channels: 336 MB of them beside 1.6 GB, forward and backward 1,321 us, 2.2
// times what their own bytes take).
// 8 channels a lane took the same time with half the wavefronts, and more
// wavefronts by launch bounds spill (427 us).
template <typename T, int W, bool WHOLE, bool WIDE>
__global__ __launch_bounds__(kThreads) void conv_grad_kernel(ConvArgs a, Shape s) {
  constexpr int V = kBackward, kAhead = 4;
  __shared__ float tile[kThreads][V];
  const int lanes = 1 << s.shift;
  const int group = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
  const uint32_t row = row_of<WIDE>(s);
  const int c = channel_of<V, WHOLE>(group, a.dim), n = a.dim - c;
  float dw[W][V], db[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    db[k] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][k] = 0.0f;
  }
  if (group < s.groups && row < s.rows) {
    const int env = (int)(row % (uint32_t)a.envs), part = (int)(row / (uint32_t)a.envs);
    const int t0 = part * s.chunk, t1 = min(t0 + s.chunk, a.steps);
    const T* x = (const T*)a.x + (int64_t)t0 * a.x_step + (int64_t)env * a.x_env;
    const T* dy = (const T*)a.dy + (int64_t)t0 * a.dy_step + (int64_t)env * a.dy_env;
    const uint8_t* resets = a.resets + (int64_t)t0 * a.envs + env;
    T* dx = (T*)a.dx + ((int64_t)t0 * a.envs + env) * a.dim;
    Packed<T, V> next_x[kAhead], next_d[kAhead];
    uint8_t next_begins[kAhead];
    auto fetch = [&](int t) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int on = t + i + 1 < a.steps;
        fetch_row<WHOLE>(x + c, n, next_x[i]);
        x += on ? a.x_step : 0;
        fetch_row<WHOLE>(dy + c, n, next_d[i]);
        dy += on ? a.dy_step : 0;
        next_begins[i] = 0;
        if (a.resets) {
          next_begins[i] = *resets;
          resets += on ? a.envs : 0;
        }
      }
    };
    fetch(t0);
    float w[W][V], bias[V], win[W - 1][V], acc[W][V];  // acc[i]: dx of step t - (W - 1) + i
    int age;
    load_weights<W>(a, c, w, bias);
    lead_in<W, V, T>(a, env, t0, c, win, age);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[j][k] = 0.0f;
    const int end = t1 + W - 1;
    for (int t = t0; t < end; t += kAhead) {
      Packed<T, V> xs[kAhead], ds[kAhead];
      bool begins[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        xs[i] = next_x[i];
        ds[i] = next_d[i];
        begins[i] = (WIDE ? __builtin_amdgcn_readfirstlane((int)next_begins[i]) : (int)next_begins[i]) != 0;
      }
      if (t + kAhead < end) fetch(t + kAhead);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int ti = t + i;
        if (ti >= end) break;
        forget(begins[i], win);
        age = begins[i] ? 0 : min(age + 1, W);
        float d[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float v = (float)xs[i].v[k];
          d[k] = (float)ds[i].v[k];
          if (a.silu) {
            const float pre = convolve<W, V>(w, win, v, bias[k], k), sig = sigmoid(pre);
            d[k] *= sig * fmaf(pre, 1.0f - sig, 1.0f);
          }
        }
        if (ti < t1) {
#pragma unroll
          for (int k = 0; k < V; ++k) {
            db[k] += d[k];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) dw[j][k] = fmaf(d[k], win[j][k], dw[j][k]);
            dw[W - 1][k] = fmaf(d[k], (float)xs[i].v[k], dw[W - 1][k]);
          }
        }
        // acc moves one step on; its last slot begins with this step.  Steps
        // before the episode's first get nothing, and nothing comes from past the end.
        const bool any = ti < a.steps;
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int k = 0; k < V; ++k) acc[j][k] = acc[j + 1][k];
        if (__ballot(age < W - 1 || !any)) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) acc[j][k] = any && W - 1 - j <= age ? fmaf(w[j][k], d[k], acc[j][k]) : acc[j][k];
        } else {
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) acc[j][k] = fmaf(w[j][k], d[k], acc[j][k]);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          acc[W - 1][k] = w[W - 1][k] * d[k];
          move_on<W, V>(win, (float)xs[i].v[k], k);
        }
        if (ti - (W - 1) >= t0) {
          store_row<V>(dx + c, WHOLE ? V : n, acc[0]);
          dx += (int64_t)a.envs * a.dim;
        }
      }
    }
  }
  // one row of partial sums a workgroup: [dim][width], then the bias [dim]
  float* part = a.work + (int64_t)blockIdx.x * (W + 1) * a.dim;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) tile[threadIdx.x][k] = j < W ? dw[j < W ? j : 0][k] : db[k];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * V; i += kThreads) {
      const int ch = channel_of<V, WHOLE>(blockIdx.y * lanes + i / V, a.dim) + i % V;
      float v = 0.0f;
      for (int r = 0; r < (kThreads >> s.shift); ++r) v += tile[(r << s.shift) + i / V][i % V];
      if (blockIdx.y * lanes + i / V < s.groups && ch < a.dim) part[j < W ? ch * W + j : a.dim * W + ch] = v;
    }
  }
}

// One step of every env: reads the state once and writes it moved on.  Bound by
// memory: 16,384 envs x 512 channels in bf16 move 134 MB in 25 us (5.3 TB/s).
// Rows that end inside a piece are taken element by element there (a lapped
// piece would read a state that its neighbour may have moved on): 2.8 TB/s.
template <typename T, int W, int EACH, bool WHOLE>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(ConvArgs a) {
  constexpr int V = kForward;
  const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V, n = a.dim - c;
  const int64_t env0 = first_env<EACH>();
  if (env0 >= a.envs || n <= 0) return;
  Packed<T, V> in[EACH], past[EACH][W - 1];
  uint8_t begins[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int64_t env = least(env0 + e * blockDim.y, a.envs - 1);
    const T* state = (const T*)a.last + env * (W - 1) * a.dim + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) fetch_row<WHOLE>(state + (int64_t)j * a.dim, n, past[e][j]);
    fetch_row<WHOLE>((const T*)a.x + env * a.x_env + c, n, in[e]);
    begins[e] = a.resets ? a.resets[env] : 0;
  }
  float w[W][V], bias[V];
  load_weights<W>(a, c, w, bias);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int64_t env = env0 + e * blockDim.y;
    if (env >= a.envs) break;
    T* state = (T*)a.last + env * (W - 1) * a.dim + c;
    float win[W - 1][V], x[V], out[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j][k] = begins[e] ? 0.0f : (float)past[e][j].v[k];
      x[k] = (float)in[e].v[k];
      const float pre = convolve<W, V>(w, win, x[k], bias[k], k);
      out[k] = a.silu ? pre * sigmoid(pre) : pre;
    }
    store_row<V>((T*)a.y + env * a.dim + c, WHOLE ? V : n, out);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<V>(state + (int64_t)j * a.dim, WHOLE ? V : n, j + 1 < W - 1 ? win[j + 1 < W - 1 ? j + 1 : 0] : x);
  }
}

template <typename F>
void by_width(int width, F&& f) {
  if (width == 2) f(std::integral_constant<int, 2>{});
  else if (width == 3) f(std::integral_constant<int, 3>{});
  else f(std::integral_constant<int, 4>{});
}
dim3 grid_of(const Shape& s) {
  const int per = kThreads >> s.shift;
  return dim3((unsigned)((s.rows + per - 1) / per), (unsigned)((s.groups + (1 << s.shift) - 1) >> s.shift));
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, hipStream_t st) {
  const Shape s = shape_of(a.steps, a.envs, a.dim, kForward);
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_width(a.width, [&](auto w) {
      if (a.dim < kForward) hipLaunchKernelGGL((conv_kernel<T, w, false, false>), grid_of(s), dim3(kThreads), 0, st, a, s);
      else if (s.shift == 6) hipLaunchKernelGGL((conv_kernel<T, w, true, true>), grid_of(s), dim3(kThreads), 0, st, a, s);
      else hipLaunchKernelGGL((conv_kernel<T, w, true, false>), grid_of(s), dim3(kThreads), 0, st, a, s);
    });
  });
  return hipGetLastError();
}

// the workgroups' partial sums
int64_t conv_grad_work(int steps, int envs, int dim, int width) {
  return (int64_t)grid_of(shape_of(steps, envs, dim, kBackward)).x * (width + 1) * dim;
}

hipError_t launch_conv_grad(const ConvArgs& a, hipStream_t st) {
  const Shape s = shape_of(a.steps, a.envs, a.dim, kBackward);
  const dim3 grid = grid_of(s);
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_width(a.width, [&](auto w) {
      if (a.dim < kBackward) hipLaunchKernelGGL((conv_grad_kernel<T, w, false, false>), grid, dim3(kThreads), 0, st, a, s);
      else if (s.shift == 6) hipLaunchKernelGGL((conv_grad_kernel<T, w, true, true>), grid, dim3(kThreads), 0, st, a, s);
      else hipLaunchKernelGGL((conv_grad_kernel<T, w, true, false>), grid, dim3(kThreads), 0, st, a, s);
    });
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_column_sum(a.work, (int)grid.x, SumOutputs{{a.dweight, a.dbias}, {a.dim * a.width, a.dim}}, st);
}

hipError_t launch_conv_step(const ConvArgs& a, hipStream_t st) {
  const StepShape s = step_shape((a.dim + kForward - 1) / kForward, a.envs);
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_width(a.width, [&](auto w) {
      const bool whole = a.dim % kForward == 0;
      if (s.each == 4 && whole) hipLaunchKernelGGL((conv_step_kernel<T, w, 4, true>), s.grid(), s.block(), 0, st, a);
      else if (s.each == 4) hipLaunchKernelGGL((conv_step_kernel<T, w, 4, false>), s.grid(), s.block(), 0, st, a);
      else if (whole) hipLaunchKernelGGL((conv_step_kernel<T, w, 1, true>), s.grid(), s.block(), 0, st, a);
      else hipLaunchKernelGGL((conv_step_kernel<T, w, 1, false>), s.grid(), s.block(), 0, st, a);
    });
  });
  return hipGetLastError();
}

}  // namespace gbx
