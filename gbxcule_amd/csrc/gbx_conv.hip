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

constexpr int kThreads = 256, kVec = 8;
constexpr int kMinSteps = 16;  // of a piece of the steps: its lead-in of up to 7 is read twice
// Lanes that keep the memory busy: 2,048 for each of 256 CUs.  Rows of fewer
// lanes are cut along the steps.
constexpr int64_t kBusyLanes = 256 * 2048;

// Shape of the launch: a workgroup is `lanes` pieces of 8 channels by
// 256 / lanes rows; a row is one env and one piece of the steps.
struct Shape {
  int pieces, shift, chunk, chunks;  // 8-channel pieces; log2 of lanes in a row; steps of a piece, pieces
  int64_t rows;
};
Shape shape_of(int steps, int envs, int dim) {
  Shape s;
  s.pieces = (dim + kVec - 1) / kVec;
  s.shift = 0;
  while (s.shift < 5 && (1 << s.shift) < s.pieces) ++s.shift;
  const int64_t lanes = (int64_t)envs * s.pieces;
  const int64_t want = std::max<int64_t>(1, kBusyLanes / lanes);
  s.chunk = (int)std::max<int64_t>(kMinSteps, (steps + want - 1) / want);
  s.chunks = (steps + s.chunk - 1) / s.chunk;
  s.rows = (int64_t)envs * s.chunks;
  return s;
}

// The inputs before step t0 of one env and 8 channels, oldest first, zero
// where an episode begins between them and step t0 - 1.
template <int W, typename T>
__device__ __forceinline__ void lead_in(const ConvArgs& a, int env, int t0, int c, float (&win)[W - 1][kVec], int& age) {
  const int n = a.dim - c;
  age = W;  // steps since the episode began, no more than W
#pragma unroll
  for (int i = 0; i < W - 1; ++i) {
    const int t = t0 - (W - 1) + i;
    if (t < 0) {
      if (a.state) load_row<kVec>((const T*)a.state + ((int64_t)env * (W - 1) + (t + W - 1)) * a.dim + c, n, win[i]);
      else {
#pragma unroll
        for (int k = 0; k < kVec; ++k) win[i][k] = 0.0f;
      }
    } else {
      load_row<kVec>((const T*)a.x + (int64_t)t * a.x_step + (int64_t)env * a.x_env + c, n, win[i]);
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
        for (int k = 0; k < kVec; ++k) win[j][k] = begins ? 0.0f : win[j][k];
    }
  }
}

// the weights of 8 channels lie together
template <int W>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int c, float (&w)[W][kVec], float (&bias)[kVec]) {
  float row[W * kVec];
  load_row<W * kVec>(a.weight + (int64_t)c * W, (a.dim - c) * W, row);
#pragma unroll
  for (int k = 0; k < kVec; ++k)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][k] = row[k * W + j];
  if (a.bias) {
    load_row<kVec>(a.bias + c, a.dim - c, bias);
  } else {
#pragma unroll
    for (int k = 0; k < kVec; ++k) bias[k] = 0.0f;
  }
}

template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_kernel(ConvArgs a, Shape s) {
  const int lanes = 1 << s.shift;
  const int piece = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
  const int64_t row = (int64_t)blockIdx.x * (kThreads >> s.shift) + (threadIdx.x >> s.shift);
  if (piece >= s.pieces || row >= s.rows) return;
  const int env = (int)(row % a.envs), part = (int)(row / a.envs);
  const int c = piece * kVec, n = a.dim - c;
  const int t0 = part * s.chunk, t1 = min(t0 + s.chunk, a.steps);
  float w[W][kVec], bias[kVec], win[W - 1][kVec];
  int age;
  load_weights<W>(a, c, w, bias);
  lead_in<W, T>(a, env, t0, c, win, age);
  const T* x = (const T*)a.x + (int64_t)env * a.x_env + c;
  T* y = (T*)a.y + (int64_t)env * a.dim + c;
  constexpr int kAhead = 4;  // steps whose loads are in flight together
  for (int t = t0; t < t1; t += kAhead) {
    float in[kAhead][kVec];
    bool begins[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int ti = min(t + i, t1 - 1);
      load_row<kVec>(x + (int64_t)ti * a.x_step, n, in[i]);
      begins[i] = a.resets && a.resets[(int64_t)ti * a.envs + env];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (t + i >= t1) break;
      float out[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        float pre = bias[k];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          win[j][k] = begins[i] ? 0.0f : win[j][k];
          pre = fmaf(w[j][k], win[j][k], pre);
        }
        pre = fmaf(w[W - 1][k], in[i][k], pre);
        out[k] = a.silu ? pre * sigmoid(pre) : pre;
#pragma unroll
        for (int j = 0; j + 1 < W - 1; ++j) win[j][k] = win[j + 1][k];
        win[W - 2][k] = in[i][k];
      }
      store_row<kVec>(y + (int64_t)(t + i) * a.envs * a.dim, n, out);
    }
  }
  if (t1 == a.steps) {
    T* last = (T*)a.last + (int64_t)env * (W - 1) * a.dim + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<kVec>(last + (int64_t)j * a.dim, n, win[j]);
  }
}

// With d[t] = dy[t] * silu'(pre[t]), pre computed again from x:
//   dx[t] = sum over j of weight[width - 1 - j] * d[t + j], as far as the episode goes,
//   dweight[width - 1 - j] = sum of d[t] * x[t - j],   dbias = sum of d[t].
// The lane walks forward and keeps width sums of dx under way, as it keeps the
// inputs; a piece of the steps goes width - 1 steps past its end to finish
// its own.  dweight and dbias of a workgroup's rows are added in LDS and
// written as one row of partial sums.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_grad_kernel(ConvArgs a, Shape s) {
  __shared__ float tile[kThreads][kVec];
  const int lanes = 1 << s.shift;
  const int piece = blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
  const int64_t row = (int64_t)blockIdx.x * (kThreads >> s.shift) + (threadIdx.x >> s.shift);
  const int c = piece * kVec, n = a.dim - c;
  float dw[W][kVec], db[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    db[k] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][k] = 0.0f;
  }
  if (piece < s.pieces && row < s.rows) {
    const int env = (int)(row % a.envs), part = (int)(row / a.envs);
    const int t0 = part * s.chunk, t1 = min(t0 + s.chunk, a.steps);
    float w[W][kVec], bias[kVec], win[W - 1][kVec], acc[W][kVec];  // acc[i]: dx of step t - (W - 1) + i
    int age;
    load_weights<W>(a, c, w, bias);
    lead_in<W, T>(a, env, t0, c, win, age);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int k = 0; k < kVec; ++k) acc[j][k] = 0.0f;
    const T* x = (const T*)a.x + (int64_t)env * a.x_env + c;
    const T* dy = (const T*)a.dy + (int64_t)env * a.dy_env + c;
    T* dx = (T*)a.dx + (int64_t)env * a.dim + c;
    constexpr int kAhead = 4;
    for (int t = t0; t < t1 + W - 1; t += kAhead) {
      float in[kAhead][kVec], d[kAhead][kVec];
      bool begins[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int ti = min(t + i, a.steps - 1);
        load_row<kVec>(x + (int64_t)ti * a.x_step, n, in[i]);
        load_row<kVec>(dy + (int64_t)ti * a.dy_step, n, d[i]);
        begins[i] = a.resets && a.resets[(int64_t)ti * a.envs + env];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int ti = t + i;
        if (ti >= t1 + W - 1) break;
        age = begins[i] ? 0 : min(age + 1, W);
        const bool mine = ti < t1, any = ti < a.steps;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          float pre = bias[k], dk = any ? d[i][k] : 0.0f;
#pragma unroll
          for (int j = 0; j < W - 1; ++j) {
            win[j][k] = begins[i] ? 0.0f : win[j][k];
            pre = fmaf(w[j][k], win[j][k], pre);
          }
          pre = fmaf(w[W - 1][k], in[i][k], pre);
          if (a.silu) {
            const float sig = sigmoid(pre);
            dk *= sig * fmaf(pre, 1.0f - sig, 1.0f);
          }
          // acc moves one step on; its last slot begins with this step
#pragma unroll
          for (int j = 0; j < W - 1; ++j) acc[j][k] = W - 1 - j <= age ? fmaf(w[j][k], dk, acc[j + 1][k]) : acc[j + 1][k];
          acc[W - 1][k] = w[W - 1][k] * dk;
          const float own = mine ? dk : 0.0f;
          db[k] += own;
#pragma unroll
          for (int j = 0; j < W - 1; ++j) dw[j][k] = fmaf(own, win[j][k], dw[j][k]);
          dw[W - 1][k] = fmaf(own, in[i][k], dw[W - 1][k]);
#pragma unroll
          for (int j = 0; j + 1 < W - 1; ++j) win[j][k] = win[j + 1][k];
          win[W - 2][k] = in[i][k];
        }
        const int done = ti - (W - 1);
        if (done >= t0 && done < t1) store_row<kVec>(dx + (int64_t)done * a.envs * a.dim, n, acc[0]);
      }
    }
  }
  // one row of partial sums a workgroup: [dim][width], then the bias [dim]
  float* part = a.work + (int64_t)blockIdx.x * (W + 1) * a.dim;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVec; ++k) tile[threadIdx.x][k] = j < W ? dw[j < W ? j : 0][k] : db[k];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * kVec; i += kThreads) {
      const int ch = blockIdx.y * lanes * kVec + i;
      float v = 0.0f;
      for (int r = 0; r < (kThreads >> s.shift); ++r) v += tile[(r << s.shift) + i / kVec][i % kVec];
      if (ch < a.dim) part[j < W ? ch * W + j : a.dim * W + ch] = v;
    }
  }
}

// One step of every env: reads the state once and writes it moved on.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(ConvArgs a, int pieces) {
  const int64_t i = block_id() * kThreads + threadIdx.x;
  const int64_t env = i / pieces;
  const int c = (int)(i % pieces) * kVec, n = a.dim - c;
  if (env >= a.envs) return;
  const bool begins = a.resets && a.resets[env];
  T* state = (T*)a.last + env * (W - 1) * a.dim + c;
  float w[W][kVec], bias[kVec], win[W - 1][kVec], in[kVec], out[kVec];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) load_row<kVec>(state + (int64_t)j * a.dim, n, win[j]);
  load_row<kVec>((const T*)a.x + env * a.x_env + c, n, in);
  load_weights<W>(a, c, w, bias);
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    float pre = bias[k];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      win[j][k] = begins ? 0.0f : win[j][k];
      pre = fmaf(w[j][k], win[j][k], pre);
    }
    pre = fmaf(w[W - 1][k], in[k], pre);
    out[k] = a.silu ? pre * sigmoid(pre) : pre;
  }
  store_row<kVec>((T*)a.y + env * a.dim + c, n, out);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store_row<kVec>(state + (int64_t)j * a.dim, n, j + 1 < W - 1 ? win[j + 1 < W - 1 ? j + 1 : 0] : in);
}

template <typename F>
void by_width(int width, F&& f) {
  if (width == 2) f(std::integral_constant<int, 2>{});
  else if (width == 3) f(std::integral_constant<int, 3>{});
  else f(std::integral_constant<int, 4>{});
}
dim3 grid_of(const Shape& s) {
  const int per = kThreads >> s.shift;
  return dim3((unsigned)((s.rows + per - 1) / per), (unsigned)((s.pieces + (1 << s.shift) - 1) >> s.shift));
}

}  // namespace

hipError_t launch_conv(const ConvArgs& a, hipStream_t st) {
  const Shape s = shape_of(a.steps, a.envs, a.dim);
  by_element(a.elem, [&](auto t) {
    by_width(a.width, [&](auto w) { hipLaunchKernelGGL((conv_kernel<decltype(t), w>), grid_of(s), dim3(kThreads), 0, st, a, s); });
  });
  return hipGetLastError();
}

// the workgroups' partial sums
int64_t conv_grad_work(int steps, int envs, int dim, int width) {
  return (int64_t)grid_of(shape_of(steps, envs, dim)).x * (width + 1) * dim;
}

hipError_t launch_conv_grad(const ConvArgs& a, hipStream_t st) {
  const Shape s = shape_of(a.steps, a.envs, a.dim);
  const dim3 grid = grid_of(s);
  by_element(a.elem, [&](auto t) {
    by_width(a.width, [&](auto w) { hipLaunchKernelGGL((conv_grad_kernel<decltype(t), w>), grid, dim3(kThreads), 0, st, a, s); });
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_column_sum(a.work, (int)grid.x, SumOutputs{{a.dweight, a.dbias}, {a.dim * a.width, a.dim}}, st);
}

hipError_t launch_conv_step(const ConvArgs& a, hipStream_t st) {
  const int pieces = (a.dim + kVec - 1) / kVec;
  const dim3 grid = wide_grid(((int64_t)a.envs * pieces + kThreads - 1) / kThreads);
  by_element(a.elem, [&](auto t) {
    by_width(a.width, [&](auto w) { hipLaunchKernelGGL((conv_step_kernel<decltype(t), w>), grid, dim3(kThreads), 0, st, a, pieces); });
  });
  return hipGetLastError();
}

}  // namespace gbx
