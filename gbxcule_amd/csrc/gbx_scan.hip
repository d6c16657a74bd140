// gbx_scan.hip -- selective state space scan along the steps of each env, its
// gradient and its single step.  For every channel d with `states` states s:
//
//   delta = softplus(dt + bias)                        (or dt + bias as it is)
//   h[s]  = exp(delta * A[d][s]) * h[s] + delta * x * B[s]     (h = 0 first where an episode begins)
//   y     = (sum over s of C[s] * h[s] + skip * x) * silu(z)
//
// A state costs one exponential and six other operations a step for 8/16
// bytes of 16-bit input and output, so the kernels are bound by the vector
// units, not by memory.  States, step sizes and sums are 32-bit throughout.
#include <algorithm>

#include "gbx_policy.h"

namespace gbx {
namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;  // wavefronts of a forward workgroup

// log(1 + e^v).  log1p(e) for small e as log(u) * e / (u - 1) with u = 1 + e
// rounded: the rounding error of u cancels (Goldberg, "What every computer
// scientist should know about floating-point arithmetic", theorem 4).
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_fast(-kLog2e * fabsf(v));
  const float u = 1.0f + e;
  const float log1p = u == 1.0f ? e : __builtin_amdgcn_logf(u) * kLn2 * (e * rcp_fast(u - 1.0f));
  return fmaxf(v, 0.0f) + log1p;
}

template <int SP, typename T>
struct RowBits {  // SP elements of a row as the dwords that a scalar load takes
  static constexpr int kWords = SP * (int)sizeof(T) / 4;
  uint32_t w[kWords];
};
template <typename T>
__device__ __forceinline__ float unpack(const uint32_t* w, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
  else if constexpr (__is_same(T, __bf16)) return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
}
typedef const uint32_t __attribute__((address_space(4))) * ScalarPtr;
template <int SP, typename T>
__device__ __forceinline__ void load_scalar(const T* p, RowBits<SP, T>& r) {
  ScalarPtr q = (ScalarPtr)(uintptr_t)p;
#pragma unroll
  for (int i = 0; i < RowBits<SP, T>::kWords; ++i) r.w[i] = q[i];
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// How the steps are divided.  A wavefront takes 64 channels (of one group) of
// one env and one piece of the steps.
struct Pieces {
  int blocks, blocks_per_group;  // channel blocks of a wavefront
  int chunk, chunks;             // steps of a piece, pieces
};

// Up to 16 pieces are joined by FULL itself, each going over those before its
// own: as a launch between, join_kernel is another 4 us and the host's time for
// it (forward of 77 steps of 37 envs x 200 channels x 8 states in 5 pieces 21.5
// -> 18.8 us, 128 of 16 x 512 x 16 in 8 28.6 -> 24.5, 256 of them in 16 37.0 ->
// 34.4, but 512 of 8 x 512 x 16 in 32 36.8 -> 39.0).  The gradient's kernel has
// no registers left for it.
constexpr int kFewPieces = 16;
// What a piece ends with, from the state it starts with (or the gradient,
// against the steps): `end` from zero and its decay.  An episode that begins
// inside lets nothing through: its sum of step sizes is given as infinity.  A
// start of zero adds nothing, also where the growth over a piece (rates or step
// sizes of the other sign) passes 32 bits.
__device__ __forceinline__ float through_piece(float from, float sum, float decay, float end) {
  return sum == __builtin_inff() || from == 0.0f ? end : fmaf(from, exp2_fast(sum * decay), end);
}

enum { FULL, ENDS, BACK };  // what scan_kernel computes

// A lane is a channel and holds its states; B and C are the same for all lanes
// of a wavefront and come through scalar registers: SCALAR loads them as
// dwords (rows that start on 4 bytes and hold exactly SP states), else each
// lane loads one element and the wavefront reads lanes.
//
// FULL: y and the last state.  Where there are too few rows to fill the chip
// the steps are cut: ENDS computes, for each piece, the state that it ends
// with when it starts from zero and the sum of its step sizes, whose decay
// carries any start state across the piece (h_end = exp(A * sum) * h_start +
// ends); join_kernel runs over them where they are many; FULL then starts each
// piece from its own state.  BACK is ENDS for the gradient, against the steps: the
// gradient of the state before a piece when nothing flows into its end.
//
// Bound by the vector units: a state takes an exponential and four products a
// step in FULL, three in ENDS; with what a channel needs once a step, the loop of
// FULL has 8 vector instructions a state step, an eighth of them exponentials.
// 128 steps x 1,024 envs x 512 channels x 16 states (1.07 G state steps, 1.07 GB
// with the states for the gradient, half of it those) take 318 us, 3.4 T state
// steps/s; as whole calls 330 us, 276 without those states, whose stores are half
// hidden.  16,384 steps of one env x 1,024 channels x 16 states take 77 us in
// FULL, 58 in ENDS.
//
// States are padded to 8, 16 or 32 (by_states), and a group's last wavefront to 64
// channels.  Without SCALAR two lane reads come to each state step: 128 steps x
// 512 envs x 512 channels x 16 states 149 us, 12 states 185, 24 states 328, 32
// states 285; 1,000 channels whose 16-bit rows of B start on odd elements 340 us,
// 992 whose do not 266.  128 steps x 1,024 envs x 128 channels in one or two groups
// 99 us, in 4 of 32 channels 145, in 8 of 16 251.
// All states in a lane: no sum across lanes, and delta, softplus and the gate
// once a channel.  More wavefronts by launch bounds are slower (8 a SIMD: 823
// us, 6: 590).
template <typename T, int SP, int WHAT, bool SCALAR>
__global__ __launch_bounds__(kWave* kWaves) void scan_kernel(ScanArgs a, Pieces p, float* ends, float* sums) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = block_id() * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = wave / p.blocks;
  const int block = (int)(wave % p.blocks);
  const int env = (int)(item % a.envs), piece = (int)(item / a.envs);
  if (piece >= p.chunks) return;
  const int group = block / p.blocks_per_group, per_group = a.dim / a.groups;
  const int in_group = (block % p.blocks_per_group) * kWave + lane;
  const bool live = in_group < per_group;
  const int d = group * per_group + min(in_group, per_group - 1);
  const int t0 = piece * p.chunk, t1 = min(t0 + p.chunk, a.steps), count = t1 - t0;
  const bool gated = a.z != nullptr;
  const int states = SCALAR ? SP : a.states;

  float decay[SP], h[SP];  // A in powers of two; the states, or their gradient
#pragma unroll
  for (int s = 0; s < SP; ++s) {
    decay[s] = s < states ? a.a[(int64_t)d * states + s] * kLog2e : 0.0f;
    h[s] = 0.0f;
  }
  const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.skip ? a.skip[d] : 0.0f;
  if constexpr (WHAT == FULL) {
    if (p.chunks > kFewPieces) {
#pragma unroll
      for (int s = 0; s < SP; ++s)
        if (s < states) h[s] = ends[((int64_t)item * states + s) * a.dim + d];
    } else {
      if (a.state) {
#pragma unroll
        for (int s = 0; s < SP; ++s)
          if (s < states) h[s] = a.state[((int64_t)env * a.dim + d) * states + s];
      }
      for (int j = 0; j < piece; ++j) {
        const int64_t of = (int64_t)j * a.envs + env;
        const float sum = sums[of * a.dim + d];
#pragma unroll
        for (int s = 0; s < SP; ++s)
          if (s < states) h[s] = through_piece(h[s], sum, decay[s], ends[(of * states + s) * a.dim + d]);
      }
    }
  }

  // Rows of the current step: uniform addresses that move from step to step
  // (against the steps for BACK), to which a lane adds its channel.
  const int64_t from = WHAT == BACK ? t1 - 1 : t0, to = WHAT == BACK ? -1 : 1;
  const uint32_t at = (uint32_t)d * sizeof(T);
  const int64_t x_step = WHAT == BACK ? a.dy_step : a.x_step, x_env = WHAT == BACK ? a.dy_env : a.x_env;
  const T* x = (const T*)(WHAT == BACK ? a.dy : a.x) + from * x_step + env * x_env;
  const T* dt = (const T*)a.dt + from * a.dt_step + env * a.dt_env;
  const T* z = (const T*)a.z + from * a.z_step + env * a.z_env;
  const T* b = (const T*)a.b + from * a.b_step + env * a.b_env + group * a.b_group;
  const T* c = (const T*)a.c + from * a.c_step + env * a.c_env + group * a.c_group;
  const uint8_t* resets = a.resets + from * a.envs + env;
  T* y = (T*)a.y + ((int64_t)t0 * a.envs + env) * a.dim;
  float* saved = a.saved + ((int64_t)(t0 / kSegment) * a.envs + env) * a.dim * states;
  auto of_lane = [&](const T* row) { return *(const T*)((const char*)row + at); };

  constexpr int kAhead = 4;  // steps whose loads are in flight together
  T xs[kAhead], dts[kAhead], zs[kAhead], bcs[kAhead];
  uint8_t rs[kAhead];
  const T* row_bc = lane >= 32 ? c : b;  // without SCALAR: lanes hold B, then C
  const int64_t row_bc_step = lane >= 32 ? to * a.c_step : to * a.b_step;
  auto fetch = [&](int k0) {
    // the last row is loaded again past the end
    const auto rows = [&](auto&& load) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) load(i, k0 + i + 1 < count ? to : 0);
    };
    rows([&](int i, int64_t on) {
      xs[i] = of_lane(x);
      x += on * x_step;
      dts[i] = of_lane(dt);
      dt += on * a.dt_step;
    });
    if (gated && WHAT != ENDS)
      rows([&](int i, int64_t on) {
        zs[i] = of_lane(z);
        z += on * a.z_step;
      });
    if (a.resets)
      rows([&](int i, int64_t on) {
        rs[i] = *resets;
        resets += on * a.envs;
      });
    if constexpr (!SCALAR)
      rows([&](int i, int64_t on) {
        bcs[i] = (lane & 31) < states ? row_bc[lane & 31] : (T)0.0f;
        row_bc += on ? row_bc_step : 0;
      });
  };
  RowBits<SP, T> rb, rc;
  if constexpr (SCALAR) {
    if constexpr (WHAT != BACK) load_scalar(b, rb);
    if constexpr (WHAT != ENDS) load_scalar(c, rc);
  }
  auto store_states = [&](float* to, const float(&v)[SP]) {
    if (states == SP) {  // 16 bytes at a time
#pragma unroll
      for (int s = 0; s < SP; s += 4) *reinterpret_cast<float4*>(to + s) = float4{v[s], v[s + 1], v[s + 2], v[s + 3]};
    } else {
#pragma unroll
      for (int s = 0; s < SP; ++s)
        if (s < states) to[s] = v[s];
    }
  };
  auto clear = [&]() {
    // a branch, the same for all lanes: without the barrier it becomes a
    // selection of every state at every step
    asm volatile("");
#pragma unroll
    for (int s = 0; s < SP; ++s) h[s] = 0.0f;
  };
  float sum = 0.0f;
  bool began = false;
  fetch(0);
  auto four = [&](int k0, auto whole) {
    float xv[kAhead], dtv[kAhead], zv[kAhead], bcv[kAhead];
    bool begins[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      xv[i] = (float)xs[i];
      dtv[i] = (float)dts[i];
      zv[i] = gated && WHAT != ENDS ? (float)zs[i] : 0.0f;
      if constexpr (!SCALAR) bcv[i] = (float)bcs[i];
      begins[i] = a.resets && __builtin_amdgcn_readfirstlane((int)rs[i]) != 0;
    }
    if (k0 + kAhead < count) fetch(k0 + kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (!whole && k0 + i >= count) break;
      float delta = dtv[i] + bias;
      if (a.softplus) delta = softplus(delta);
      float bv[SP], cv[SP];
      if constexpr (SCALAR) {
        // this step's rows have arrived: unpack them, then ask for the next
        // step's (the last ones again past the end)
        const bool more = k0 + i + 1 < count;
        if constexpr (WHAT != BACK) {
#pragma unroll
          for (int s = 0; s < SP; ++s) bv[s] = unpack<T>(rb.w, s);
          b += more ? to * a.b_step : 0;
          load_scalar(b, rb);
        }
        if constexpr (WHAT != ENDS) {
#pragma unroll
          for (int s = 0; s < SP; ++s) cv[s] = unpack<T>(rc.w, s);
          c += more ? to * a.c_step : 0;
          load_scalar(c, rc);
        }
      } else {
#pragma unroll
        for (int s = 0; s < SP; ++s) {
          if constexpr (WHAT != BACK) bv[s] = lane_value(bcv[i], s);
          if constexpr (WHAT != ENDS) cv[s] = lane_value(bcv[i], 32 + s);
        }
      }
      if constexpr (WHAT == BACK) {
        const float dv = gated ? xv[i] * zv[i] * sigmoid(zv[i]) : xv[i];
#pragma unroll
        for (int s = 0; s < SP; ++s) h[s] = fmaf(cv[s], dv, h[s]) * exp2_fast(delta * decay[s]);
        if (begins[i]) clear();
        sum += delta;
        began = began || begins[i];
      } else {
        if (begins[i]) clear();
        if constexpr (WHAT == FULL) {
          if (a.saved && (k0 + i) % kSegment == 0) {  // pieces begin at multiples of kSegment
            if (live) {
#pragma unroll
              for (int s = 0; s < SP; ++s)
                if (s < states) saved[(int64_t)s * a.dim + d] = h[s];
            }
            saved += (int64_t)a.envs * states * a.dim;
          }
        }
        const float u = delta * xv[i];
#pragma unroll
        for (int s = 0; s < SP; ++s) h[s] = fmaf(h[s], exp2_fast(delta * decay[s]), u * bv[s]);
        if constexpr (WHAT == FULL) {
          float part[2] = {skip * xv[i], 0.0f};
#pragma unroll
          for (int s = 0; s < SP; ++s) part[s & 1] = fmaf(h[s], cv[s], part[s & 1]);
          float out = part[0] + part[1];
          if (gated) out *= zv[i] * sigmoid(zv[i]);
          if (live) *(T*)((char*)y + at) = (T)out;
          y += (int64_t)a.envs * a.dim;
        } else {
          sum += delta;
          began = began || begins[i];
        }
      }
    }
  };
  // (an exit after each of the four would keep copies of the states for it:
  // 377 us where this took 325)
  int k0 = 0;
  for (; k0 + kAhead <= count; k0 += kAhead) four(k0, std::true_type{});
  if (k0 < count) four(k0, std::false_type{});
  if (!live) return;
  if constexpr (WHAT == FULL) {
    if (t1 == a.steps) store_states(a.last + ((int64_t)env * a.dim + d) * states, h);
  } else {
#pragma unroll
    for (int s = 0; s < SP; ++s)
      if (s < states) ends[((int64_t)item * states + s) * a.dim + d] = h[s];
    sums[(int64_t)item * a.dim + d] = began ? __builtin_inff() : sum;
  }
}

// Runs over the pieces, first to last (BACKWARD: last to first), and leaves in
// `ends` what each piece starts from.  A lane is one env, state and channel, and
// waits for its loads, 16 pieces at a time.
template <bool BACKWARD>
__global__ __launch_bounds__(256) void join_kernel(ScanArgs a, int chunks, float* ends, const float* sums) {
  const int64_t i = block_id() * 256 + threadIdx.x, each = (int64_t)a.envs * a.states * a.dim;
  if (i >= each) return;
  const int d = (int)(i % a.dim), s = (int)(i / a.dim % a.states), env = (int)(i / a.dim / a.states);
  const float decay = a.a[(int64_t)d * a.states + s] * kLog2e;
  float h = !BACKWARD && a.state ? a.state[((int64_t)env * a.dim + d) * a.states + s] : 0.0f;
  constexpr int kAhead = 16;  // pieces whose loads are in flight together
  for (int k0 = 0; k0 < chunks; k0 += kAhead) {
    float e[kAhead], sum[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = min(k0 + k, chunks - 1), piece = BACKWARD ? chunks - 1 - j : j;
      e[k] = ends[piece * each + i];
      sum[k] = sums[((int64_t)piece * a.envs + env) * a.dim + d];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (k0 + k >= chunks) break;
      const int piece = BACKWARD ? chunks - 1 - k0 - k : k0 + k;
      ends[piece * each + i] = h;
      h = through_piece(h, sum[k], decay, e[k]);
    }
  }
}

// The same for many pieces.  A workgroup is 64 channels of one env and state by
// 16 runs of up to 16 pieces: each lane composes its run, the runs are joined
// through LDS, and the lane goes through its run again from what comes before
// it.  256 pieces of 1,024 channels x 16 states take 13 us (join_kernel 27), 64
// of 512 channels as long as there, but 32 pieces of 16 envs 40 us longer.
constexpr int kRuns = 16, kRun = 16, kManyPieces = 64;
template <bool BACKWARD>
__global__ __launch_bounds__(kWave* kRuns) void join_runs_kernel(ScanArgs a, int chunks, float* ends, const float* sums) {
  __shared__ float last[kRuns][kWave], through[kRuns][kWave];  // of a run: its end from zero; what it lets through
  const int lane = threadIdx.x % kWave, run = threadIdx.x / kWave, blocks = (a.dim + kWave - 1) / kWave;
  const int64_t row = block_id() / blocks;  // env and state
  if (row >= (int64_t)a.envs * a.states) return;
  const int d0 = (int)(block_id() % blocks) * kWave + lane, d = min(d0, a.dim - 1);
  const int s = (int)(row % a.states), env = (int)(row / a.states);
  const float decay = a.a[(int64_t)d * a.states + s] * kLog2e;
  float h = !BACKWARD && a.state ? a.state[((int64_t)env * a.dim + d) * a.states + s] : 0.0f;
  // (as through_piece: an episode that begins in a piece lets nothing through,
  // whatever lies before, and zero adds nothing)
  constexpr float kNothing = -1.0f;
  const auto pass = [&](float from, float by, float end) { return by < 0.0f || from == 0.0f ? end : fmaf(from, by, end); };
  for (int first = 0; first < chunks; first += kRuns * kRun) {
    const int count = min(kRuns * kRun, chunks - first), per = (count + kRuns - 1) / kRuns;
    const int mine = max(0, min(per, count - run * per));
    const auto piece_of = [&](int k) {
      const int j = first + run * per + min(k, mine - 1);
      return (int64_t)(BACKWARD ? chunks - 1 - j : j) * a.envs + env;
    };
    float e[kRun], by[kRun], end = 0.0f, all = 1.0f;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      e[k] = by[k] = 0.0f;
      if (mine > 0) {
        e[k] = ends[(piece_of(k) * a.states + s) * a.dim + d];
        by[k] = sums[piece_of(k) * a.dim + d];
      }
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k) by[k] = by[k] == __builtin_inff() ? kNothing : exp2_fast(by[k] * decay);
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (k >= mine) break;
      end = pass(end, by[k], e[k]);
      all = by[k] < 0.0f || all < 0.0f ? kNothing : all * by[k];
    }
    last[run][lane] = end;
    through[run][lane] = all;
    __syncthreads();
    float start = h;
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      start = r == run ? h : start;
      h = pass(h, through[r][lane], last[r][lane]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (k >= mine) break;
      if (d0 < a.dim) ends[(piece_of(k) * a.states + s) * a.dim + d] = start;
      start = pass(start, by[k], e[k]);
    }
  }
}

// Gradient.  With d = dy * silu(z) and g the gradient of the state,
//   g = C d + a' g' (a', g': the next step's),  dC = sum over channels of d h,  dB = sum over channels of g delta x,
//   through = sum over s of g B,  by = g a h_before,
//   dA = sum over steps and envs of by delta,  ddelta = through x + sum over s of by A,  dx = through delta + skip d.
//
// A wavefront takes CH channels (16 lanes along channels, C of them in each
// lane) and all states (4 lanes, Q states in each): 8 states of channels a
// lane, so that both sums, over states within 4 lanes and over channels, are
// cheap.  It walks the steps backwards in segments of kSegment: from the saved
// state before the segment it computes the segment's states again into
// registers, then goes back through them.  What a channel needs at a step
// (delta, x, d) and the rows of B and C are converted once into LDS.  The
// wavefronts of a workgroup take neighbouring channels of the same steps and
// add their dB and dC in LDS at the end of a segment.
//
// Bound by the vector units, which are active three quarters of the time: about
// 25 instructions a state step, one and a half of them exponentials.  128 steps x 1,024
// envs x 512 channels x 16 states in bf16: 1,008 us, 1.07 T state steps/s.  8
// elements a lane and 8 steps a segment fill the registers of two wavefronts a
// SIMD; three spill (2,284 us).
constexpr int kGradWaves = 4;  // wavefronts of a workgroup at most
template <int SP>
struct GradShape {
  static constexpr int Q = SP / 4, C = 8 / Q, CH = 16 * C;
  // Last steps of a segment whose decays stay in registers from the way forward
  // to the way back; the others' are computed twice.  16 states 1,397 us with
  // none, 1,371 with 2, 1,360 with 4, 1,838 with 8, which spill; 8 states 886,
  // 877, 987, 1,472 (forward and backward of the rollout above).
  static constexpr int kKept = SP == 8 ? 2 : 4;
  struct Lds {
    float delta[kSegment][CH], x[kSegment][CH], d[kSegment][CH];
    float through[kSegment][CH], by[kSegment][CH], plain[kSegment][CH];  // sums over states
    float b[kSegment][SP], c[kSegment][SP];
    float cross[2][kSegment][2 * SP];  // dB, dC; two segments in turn
  };
};

__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float(__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// sum over the 4 lanes that share channels
__device__ __forceinline__ float quad_sum(float v) { return add_dpp<0x4E>(add_dpp<0xB1>(v)); }  // lanes 1 0 3 2, 2 3 0 1
// lanes 0-31: a summed over the two halves of the wavefront; lanes 32-63: b
__device__ __forceinline__ float fold_halves(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// even rows of 16 lanes: a summed over the row and its odd neighbour; odd rows: b
__device__ __forceinline__ float fold_rows(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T, int SP>
__global__ __launch_bounds__(kWave* kGradWaves, 2) void scan_grad_kernel(ScanArgs a, Pieces p, int slots, const float* carried, float* cross_out, float* sums_out) {
  using S = GradShape<SP>;
  constexpr int Q = S::Q, C = S::C, CH = S::CH, kOnce = kSegment - S::kKept, kApart = kWave / CH, kPairs = kSegment / kApart;
  extern __shared__ __align__(16) char lds[];
  typename S::Lds* all = reinterpret_cast<typename S::Lds*>(lds);
  const int lane = threadIdx.x & 63, which = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / kWave;
  typename S::Lds& m = all[which];
  const int block = blockIdx.x % p.blocks, slot = blockIdx.x / p.blocks;
  const int group = block / p.blocks_per_group, per_group = a.dim / a.groups, first_d = group * per_group;
  const int base = (block % p.blocks_per_group * waves + which) * CH;  // of the wavefront's channels in the group
  const int cg = lane >> 2, sg = lane & 3;                             // the lane's channels cg * C.., states sg * Q..
  // one channel a lane where a step's values are prepared and finished
  const int own = lane % CH, own_i = lane / CH, own_d = first_d + min(base + own, per_group - 1);
  const bool own_live = base + own < per_group, gated = a.z != nullptr;
  const float bias = a.bias ? a.bias[own_d] : 0.0f, skip = a.skip ? a.skip[own_d] : 0.0f;

  // A in powers of two.  Lanes past the last channel or state hold its rate, so
  // that a step of infinite size makes a zero of their decay too; with a rate of
  // zero it would be NaN, and sums over lanes with it.
  float A[C][Q], dA[C][Q], dskip = 0.0f, dbias = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int ch = min(base + cg * C + c, per_group - 1);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int s = min(sg * Q + q, a.states - 1);
      A[c][q] = a.a[(int64_t)(first_d + ch) * a.states + s] * kLog2e;
      dA[c][q] = 0.0f;
    }
  }
  int turn = 0;
  for (int64_t item = slot; item < (int64_t)p.chunks * a.envs; item += slots) {
    const int env = (int)(item % a.envs), piece = (int)(item / a.envs);
    const int t0 = piece * p.chunk, t1 = min(t0 + p.chunk, a.steps);
    float g[C][Q];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int ch = base + cg * C + c, s = sg * Q + q;
        g[c][q] = p.chunks > 1 && ch < per_group && s < a.states ? carried[(item * a.states + s) * a.dim + first_d + ch] : 0.0f;
      }
    // a lane's part of the addresses; the steps' part is the same for all
    const T* xp = (const T*)a.x + env * a.x_env + own_i * a.x_step + own_d;
    const T* dtp = (const T*)a.dt + env * a.dt_env + own_i * a.dt_step + own_d;
    const T* zp = (const T*)a.z + env * a.z_env + own_i * a.z_step + own_d;
    const T* dyp = (const T*)a.dy + env * a.dy_env + own_i * a.dy_step + own_d;
    const int row_i = lane / SP, row_s = lane % SP;
    const T* bp = (const T*)a.b + env * a.b_env + group * a.b_group + row_i * a.b_step + row_s;
    const T* cp = (const T*)a.c + env * a.c_env + group * a.c_group + row_i * a.c_step + row_s;
    const int64_t out_step = (int64_t)a.envs * a.dim, out = (int64_t)env * a.dim + own_i * out_step + own_d;

    // A segment's inputs as they lie in memory; the next segment's are on
    // their way while this one is worked on.
    constexpr int kRows = kWave / SP, kRowLoads = kSegment / kRows;
    struct Inputs {
      T x[kPairs], dt[kPairs], dy[kPairs], z[kPairs], b[kRowLoads], c[kRowLoads];
      uint8_t begins;
      float before[C][Q];
    } in, next;
    auto fetch = [&](int seg, Inputs& to) {
      const int live_steps = min(kSegment, a.steps - seg);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int64_t t = seg + k * kApart;
        to.x[k] = to.dt[k] = to.dy[k] = to.z[k] = (T)0.0f;
        if (own_i + k * kApart < live_steps) {
          to.x[k] = xp[t * a.x_step];
          to.dt[k] = dtp[t * a.dt_step];
          to.dy[k] = dyp[t * a.dy_step];
          if (gated) to.z[k] = zp[t * a.z_step];
        }
      }
#pragma unroll
      for (int k = 0; k < kRowLoads; ++k) {
        const int64_t t = seg + k * kRows;
        to.b[k] = to.c[k] = (T)0.0f;
        if (row_i + k * kRows < live_steps && row_s < a.states) {
          to.b[k] = bp[t * a.b_step];
          to.c[k] = cp[t * a.c_step];
        }
      }
      // steps past the end are cut off as an episode's first is: what the last
      // state holds, finite or not, reaches no sum through them
      to.begins = lane >= live_steps ? 1 : a.resets ? a.resets[(int64_t)(seg + lane) * a.envs + env] : 0;
      const float* saved = a.saved + ((int64_t)(seg / kSegment) * a.envs + env) * a.dim * a.states;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int s = min(sg * Q + q, a.states - 1), ch = base + cg * C;
        float row[C];
        load_row<C>(saved + (int64_t)s * a.dim + first_d + ch, per_group - ch, row);
#pragma unroll
        for (int c = 0; c < C; ++c) to.before[c][q] = row[c];
      }
    };
    const int last_seg = t0 + (t1 - 1 - t0) / kSegment * kSegment;
    fetch(last_seg, next);
    for (int seg = last_seg; seg >= t0; seg -= kSegment) {
      const int live_steps = min(kSegment, a.steps - seg);
      in = next;
      const uint32_t begins = (uint32_t)__ballot(in.begins != 0);
      // prepare: steps past the end push nothing, and nothing comes from them
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int i = own_i + k * kApart;
        float delta = (float)in.dt[k] + bias, dv = (float)in.dy[k];
        if (a.softplus) delta = softplus(delta);
        if (gated) dv *= (float)in.z[k] * sigmoid((float)in.z[k]);
        m.delta[i][own] = i < live_steps ? delta : 0.0f;
        m.x[i][own] = (float)in.x[k];
        m.d[i][own] = own_live ? dv : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kRowLoads; ++k) {
        m.b[row_i + k * kRows][row_s] = (float)in.b[k];
        m.c[row_i + k * kRows][row_s] = (float)in.c[k];
      }
      lds_order();

      // (an episode's first step takes a branch of its own, the same for all
      // lanes: selecting zeros would keep a second copy of every state)
      float h[kSegment][C][Q], kept[S::kKept][C][Q];
#pragma unroll
      for (int i = 0; i < kSegment; ++i) {
        const bool first = begins >> i & 1u;
        float delta[C], plain[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          delta[c] = m.delta[i][cg * C + c];
          const float u = delta[c] * m.x[i][cg * C + c];
#pragma unroll
          for (int q = 0; q < Q; ++q) h[i][c][q] = u * m.b[i][sg * Q + q];
        }
        if (!first) {
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              const float decay = exp2_fast(delta[c] * A[c][q]);
              if (i >= kOnce) kept[i >= kOnce ? i - kOnce : 0][c][q] = decay;
              h[i][c][q] = fmaf(i == 0 ? in.before[c][q] : h[i == 0 ? 0 : i - 1][c][q], decay, h[i][c][q]);
            }
        }
        if (gated) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            plain[c] = 0.0f;
#pragma unroll
            for (int q = 0; q < Q; ++q) plain[c] = fmaf(h[i][c][q], m.c[i][sg * Q + q], plain[c]);
            m.plain[i][cg * C + c] = quad_sum(plain[c]);
          }
        }
      }
      if (seg > t0) fetch(seg - kSegment, next);
      lds_order();  // the rows are read again: kept in registers they would not fit
#pragma unroll
      for (int i = kSegment - 1; i >= 0; --i) {
        const bool first = begins >> i & 1u;
        float db[Q], dc[Q], delta[C], through[C], by[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          delta[c] = m.delta[i][cg * C + c];
          const float u = delta[c] * m.x[i][cg * C + c], dv = m.d[i][cg * C + c];
          through[c] = by[c] = 0.0f;
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            g[c][q] = fmaf(m.c[i][sg * Q + q], dv, g[c][q]);
            dc[q] = c == 0 ? dv * h[i][c][q] : fmaf(dv, h[i][c][q], dc[q]);
            db[q] = c == 0 ? g[c][q] * u : fmaf(g[c][q], u, db[q]);
            through[c] = fmaf(g[c][q], m.b[i][sg * Q + q], through[c]);
          }
        }
        if (!first) {
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < Q; ++q) {
              g[c][q] *= i >= kOnce ? kept[i >= kOnce ? i - kOnce : 0][c][q] : exp2_fast(delta[c] * A[c][q]);
              const float via = g[c][q] * (i == 0 ? in.before[c][q] : h[i == 0 ? 0 : i - 1][c][q]);
              by[c] = fmaf(via, A[c][q], by[c]);
              dA[c][q] = fmaf(via, delta[c], dA[c][q]);
            }
        } else {
          asm volatile("");  // (stays a branch)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < Q; ++q) g[c][q] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
          m.through[i][cg * C + c] = quad_sum(through[c]);
          m.by[i][cg * C + c] = quad_sum(by[c]);
        }
        // dB and dC summed over the 16 channel lanes, two sums folded into one
        // register at a time: halves of the wavefront then hold dB and dC, odd
        // rows of 16 lanes the upper half of the lane's states
#pragma unroll
        for (int q = 0; q < Q / 2; ++q) {
          const float w = fold_rows(fold_halves(db[q], dc[q]), fold_halves(db[q + Q / 2], dc[q + Q / 2]));
          // lanes rotated by 8 and by 4 in a row of 16: four lanes write the same sum
          m.cross[turn][i][(lane >> 5) * SP + sg * Q + (lane >> 4 & 1) * (Q / 2) + q] = add_dpp<0x124>(add_dpp<0x128>(w));
        }
      }
      lds_order();
      // finish: one channel a lane
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int i = own_i + k * kApart;
        if (i < live_steps && own_live) {
          const int64_t to = out + (seg + k * kApart) * out_step;
          const float xv = (float)in.x[k], dv = m.d[i][own], thr = m.through[i][own];
          float ddt = fmaf(thr, xv, m.by[i][own] * kLn2);
          if (a.softplus) ddt *= sigmoid((float)in.dt[k] + bias);
          ((T*)a.ddt)[to] = (T)ddt;
          ((T*)a.dx)[to] = (T)fmaf(thr, m.delta[i][own], skip * dv);
          dskip = fmaf(dv, xv, dskip);
          dbias += ddt;
          if (gated) {
            const float zv = (float)in.z[k], sig = sigmoid(zv);
            const float plain = fmaf(skip, xv, m.plain[i][own]);
            ((T*)a.dz)[to] = (T)((float)in.dy[k] * plain * sig * fmaf(zv, 1.0f - sig, 1.0f));
          }
        }
      }
      // dB and dC of the workgroup's channels; the wavefronts that are still
      // here write the other half of `cross` in the next segment
      __syncthreads();
      for (int e = threadIdx.x; e < kSegment * 2 * SP; e += blockDim.x) {
        const int i = e / (2 * SP), o = e % (2 * SP), s = o % SP;
        float v = 0.0f;
        for (int w = 0; w < waves; ++w) v += all[w].cross[turn][i][o];
        if (i < live_steps) {
          const int64_t row = (int64_t)(seg + i) * a.envs + env;
          if (p.blocks_per_group > 1) cross_out[(row * p.blocks + block) * (2 * SP) + o] = v;
          else if (s < a.states) ((T*)(o < SP ? a.db : a.dc))[(row * a.groups + group) * a.states + s] = (T)v;
        }
      }
      turn ^= 1;
    }
  }
  // one row of partial sums a slot: dA [dim][states], dskip [dim], dbias [dim]
  float* row = sums_out + (int64_t)slot * a.dim * (a.states + 2);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int ch = base + cg * C + c, s = sg * Q + q;
      if (ch < per_group && s < a.states) row[(int64_t)(first_d + ch) * a.states + s] = dA[c][q];
    }
#pragma unroll
  for (int k = CH; k < kWave; k <<= 1) {
    dskip += __shfl_xor(dskip, k, 64);
    dbias += __shfl_xor(dbias, k, 64);
  }
  if (lane < CH && own_live) {
    row[(int64_t)a.dim * a.states + own_d] = dskip;
    row[(int64_t)a.dim * (a.states + 1) + own_d] = dbias;
  }
}

// dB and dC of a group of several channel blocks: their sum, rounded once.
// 131,072 rows of 4 blocks x 32 sums: 24 us.
template <typename T, int SP>
__global__ __launch_bounds__(256) void cross_sum_kernel(ScanArgs a, Pieces p, const float* cross) {
  const int64_t i = block_id() * 256 + threadIdx.x;
  const int64_t row = i / (2 * SP);  // (step, env, group)
  if (row >= (int64_t)a.steps * a.envs * a.groups) return;
  const int o = (int)(i % (2 * SP)), s = o % SP;
  const float* from = cross + row * p.blocks_per_group * 2 * SP + o;
  float v = 0.0f;
  for (int k = 0; k < p.blocks_per_group; ++k) v += from[k * 2 * SP];
  if (s < a.states) ((T*)(o < SP ? a.db : a.dc))[row * a.states + s] = (T)v;
}

// One step of every env: the state is read and written once and bounds the
// kernel.  LANES lanes share a channel, 4 states (16 bytes) each; where a
// channel has no power of two of them, the last lanes have none.  16,384 envs x
// 512 channels x 16 states move 1.14 GB in 225 us (5.1 TB/s), 64 envs 4.5 MB in
// 4 us.
template <typename T, int LANES, int EACH>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x, d = i / LANES, part = i % LANES, parts = a.states / 4;
  const int64_t env0 = first_env<EACH>();
  if (env0 >= a.envs || d >= a.dim) return;
  const bool holds = part < parts;
  const int group = a.groups == 1 ? 0 : d / (a.dim / a.groups), place = d * parts + (holds ? part : 0);
  const T* b = (const T*)a.b + group * a.b_group + (holds ? part : 0) * 4;
  const T* c = (const T*)a.c + group * a.c_group + (holds ? part : 0) * 4;
  float4 h[EACH];
  float bv[EACH][4], cv[EACH][4];
  T x[EACH], dt[EACH], z[EACH];
  uint8_t begins[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t env = least(env0 + k * blockDim.y, a.envs - 1);
    h[k] = reinterpret_cast<const float4*>(a.last)[env * a.dim * parts + place];
    load_row<4>(b + env * a.b_env, 4, bv[k]);
    load_row<4>(c + env * a.c_env, 4, cv[k]);
    x[k] = ((const T*)a.x)[env * a.x_env + d];
    dt[k] = ((const T*)a.dt)[env * a.dt_env + d];
    z[k] = a.z ? ((const T*)a.z)[env * a.z_env + d] : (T)0.0f;
    begins[k] = a.resets ? a.resets[env] : 0;
  }
  const float4 decay = reinterpret_cast<const float4*>(a.a)[place];
  const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.skip ? a.skip[d] : 0.0f;
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t env = env0 + k * blockDim.y;
    float delta = (float)dt[k] + bias;
    if (a.softplus) delta = softplus(delta);
    if (begins[k]) h[k] = float4{0.0f, 0.0f, 0.0f, 0.0f};
    const float u = delta * (float)x[k], scaled = delta * kLog2e;
    h[k].x = fmaf(h[k].x, exp2_fast(scaled * decay.x), u * bv[k][0]);
    h[k].y = fmaf(h[k].y, exp2_fast(scaled * decay.y), u * bv[k][1]);
    h[k].z = fmaf(h[k].z, exp2_fast(scaled * decay.z), u * bv[k][2]);
    h[k].w = fmaf(h[k].w, exp2_fast(scaled * decay.w), u * bv[k][3]);
    float out = fmaf(h[k].x, cv[k][0], h[k].y * cv[k][1]) + fmaf(h[k].z, cv[k][2], h[k].w * cv[k][3]);
    if (!holds) out = 0.0f;
    if constexpr (LANES > 1) out = add_dpp<0xB1>(out);
    if constexpr (LANES > 2) out = add_dpp<0x4E>(out);
    if constexpr (LANES > 4) out += __shfl_xor(out, 4, 64);
    if (env >= a.envs) break;
    if (holds) reinterpret_cast<float4*>(a.last)[env * a.dim * parts + place] = h[k];
    out = fmaf(skip, (float)x[k], out);
    if (a.z) out *= (float)z[k] * sigmoid((float)z[k]);
    if (part == 0) ((T*)a.y)[env * a.dim + d] = (T)out;
  }
}
// No multiple of 4 states: a lane a channel, whose states lie apart from its
// neighbours'.  16,384 envs x 512 channels x 15 states 861 us (16 states: 220).
template <typename T>
__global__ __launch_bounds__(256) void scan_step_any_kernel(ScanArgs a) {
  const int64_t env = first_env<1>();
  const int d = blockIdx.x * blockDim.x + threadIdx.x;
  if (env >= a.envs || d >= a.dim) return;
  const int group = a.groups == 1 ? 0 : d / (a.dim / a.groups);
  const T* b = (const T*)a.b + env * a.b_env + group * a.b_group;
  const T* c = (const T*)a.c + env * a.c_env + group * a.c_group;
  const bool begins = a.resets && a.resets[env];
  const float x = (float)((const T*)a.x)[env * a.x_env + d];
  float delta = (float)((const T*)a.dt)[env * a.dt_env + d] + (a.bias ? a.bias[d] : 0.0f);
  if (a.softplus) delta = softplus(delta);
  float out = a.skip ? a.skip[d] * x : 0.0f;
  float* hp = a.last + (env * a.dim + d) * a.states;
  for (int s = 0; s < a.states; ++s) {
    const float h = fmaf(begins ? 0.0f : hp[s], exp2_fast(delta * kLog2e * a.a[(int64_t)d * a.states + s]), delta * x * (float)b[s]);
    hp[s] = h;
    out = fmaf(h, (float)c[s], out);
  }
  if (a.z) {
    const float zv = (float)((const T*)a.z)[env * a.z_env + d];
    out *= zv * sigmoid(zv);
  }
  ((T*)a.y)[env * a.dim + d] = (T)out;
}

template <typename F>
void by_states(int states, F&& f) {
  if (states <= 8) f(std::integral_constant<int, 8>{});
  else if (states <= 16) f(std::integral_constant<int, 16>{});
  else f(std::integral_constant<int, 32>{});
}
int padded(int states) { return states <= 8 ? 8 : states <= 16 ? 16 : 32; }

// Wavefronts below which the steps are cut into pieces, about how many there
// are then (4 for each of 1,024 SIMDs), and the fewest steps of a piece: two
// more launches take as long as some 40 steps (one row of 16,384 steps: 2,048
// wavefronts 220 us, 4,096 192, 8,192 208; 4,096 steps of two rows in pieces
// of at least 8 steps 92 us, 16 67; 40 steps of 16 rows in pieces of 16 30 us,
// 32 38).  A wavefront for each SIMD is not enough up to 16 states (1,024 of
// them, 128 envs x 512 channels: 128 steps x 16 states 87 us whole, 78 in pieces,
// 8 states 67 and 54, 1,024 steps x 16 states 670 and 506; 1,504 102 and 104),
// with 32 it is (122 and 132).
constexpr int64_t kFull = 1280, kFull32 = 1024, kWant = 4096, kLeastPiece = 16;
Pieces pieces_of(int steps, int envs, int dim, int groups, int states, int channels, int waves_of_block) {
  Pieces p;
  p.blocks_per_group = (dim / groups + channels * waves_of_block - 1) / (channels * waves_of_block);
  p.blocks = groups * p.blocks_per_group;
  const int64_t waves = (int64_t)envs * p.blocks * waves_of_block;
  const int64_t cuts = waves >= (states <= 16 ? kFull : kFull32) ? 1 : std::min<int64_t>((kWant + waves - 1) / waves, (steps + kLeastPiece - 1) / kLeastPiece);
  const int64_t each = (steps + cuts - 1) / cuts;
  p.chunk = (int)((each + kSegment - 1) / kSegment * kSegment);
  p.chunks = (steps + p.chunk - 1) / p.chunk;
  return p;
}
// The gradient's workgroups: up to kGradWaves wavefronts of 512 / padded
// channels each, and rows of partial sums for about 4,096 wavefronts.
int grad_waves(int dim, int groups, int states) {
  const int each = 512 / padded(states), blocks = (dim / groups + each - 1) / each;
  return blocks > 2 ? kGradWaves : blocks;
}
int grad_slots(const Pieces& p, int envs, int waves) {
  return (int)std::min<int64_t>((int64_t)p.chunks * envs, std::max<int64_t>(1, 4096 / (p.blocks * waves)));
}
Pieces grad_pieces(int steps, int envs, int dim, int groups, int states) {
  return pieces_of(steps, envs, dim, groups, states, 512 / padded(states), grad_waves(dim, groups, states));
}
// dB and dC by channel block, where a group has several
int64_t cross_floats(const Pieces& p, int steps, int envs, int states) {
  return p.blocks_per_group > 1 ? (int64_t)steps * envs * p.blocks * 2 * padded(states) : 0;
}

template <bool BACKWARD>
void launch_join(const ScanArgs& a, const Pieces& p, float* ends, const float* sums, hipStream_t st) {
  const int64_t rows = (int64_t)a.envs * a.states;
  if (!BACKWARD && p.chunks <= kFewPieces) return;
  if (p.chunks >= kManyPieces) {
    const dim3 grid = wide_grid(rows * ((a.dim + kWave - 1) / kWave));
    hipLaunchKernelGGL(join_runs_kernel<BACKWARD>, grid, dim3(kWave * kRuns), 0, st, a, p.chunks, ends, sums);
  } else {
    hipLaunchKernelGGL(join_kernel<BACKWARD>, wide_grid((rows * a.dim + 255) / 256), dim3(256), 0, st, a, p.chunks, ends, sums);
  }
}

template <typename T, int SP, int WHAT>
void launch_scan_kernel(const ScanArgs& a, const Pieces& p, float* ends, float* sums, hipStream_t st) {
  const int64_t waves = (int64_t)p.blocks * a.envs * p.chunks;
  const dim3 grid = wide_grid((waves + kWaves - 1) / kWaves);
  constexpr uint64_t e = sizeof(T);
  const uint64_t bits = (uint64_t)(uintptr_t)a.b | (uint64_t)(uintptr_t)a.c | a.b_step * e | a.b_env * e | a.b_group * e | a.c_step * e | a.c_env * e | a.c_group * e;
  if (a.states == SP && bits % 4 == 0) hipLaunchKernelGGL((scan_kernel<T, SP, WHAT, true>), grid, dim3(kWave * kWaves), 0, st, a, p, ends, sums);
  else hipLaunchKernelGGL((scan_kernel<T, SP, WHAT, false>), grid, dim3(kWave * kWaves), 0, st, a, p, ends, sums);
}

}  // namespace

int64_t scan_work(int steps, int envs, int dim, int groups, int states) {
  const Pieces p = pieces_of(steps, envs, dim, groups, states, kWave, 1);
  return p.chunks > 1 ? (int64_t)p.chunks * envs * dim * (states + 1) : 0;
}

hipError_t launch_scan(const ScanArgs& a, hipStream_t st) {
  const Pieces p = pieces_of(a.steps, a.envs, a.dim, a.groups, a.states, kWave, 1);
  float *ends = a.work, *sums = a.work + (int64_t)p.chunks * a.envs * a.dim * a.states;
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_states(a.states, [&](auto sp) {
      if (p.chunks > 1) {
        launch_scan_kernel<T, sp, ENDS>(a, p, ends, sums, st);
        launch_join<false>(a, p, ends, sums, st);
      }
      launch_scan_kernel<T, sp, FULL>(a, p, ends, sums, st);
    });
  });
  return hipGetLastError();
}

// rows of partial sums; dB and dC by channel block; what the pieces start from
int64_t scan_grad_work(int steps, int envs, int dim, int groups, int states) {
  const Pieces p = grad_pieces(steps, envs, dim, groups, states);
  int64_t n = (int64_t)grad_slots(p, envs, grad_waves(dim, groups, states)) * dim * (states + 2);
  n += cross_floats(p, steps, envs, states);
  if (p.chunks > 1) n += (int64_t)p.chunks * envs * dim * (states + 1);
  return n;
}

hipError_t launch_scan_grad(const ScanArgs& a, hipStream_t st) {
  const Pieces p = grad_pieces(a.steps, a.envs, a.dim, a.groups, a.states);
  const int waves = grad_waves(a.dim, a.groups, a.states), slots = grad_slots(p, a.envs, waves), cols = a.dim * (a.states + 2);
  float* rows = a.work;
  float* cross = rows + (int64_t)slots * cols;
  float* ends = cross + cross_floats(p, a.steps, a.envs, a.states);
  float* sums = ends + (int64_t)p.chunks * a.envs * a.dim * a.states;
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_states(a.states, [&](auto sp) {
      if (p.chunks > 1) {
        Pieces wide = p;  // the same steps, 64 channels to a wavefront
        wide.blocks_per_group = (a.dim / a.groups + kWave - 1) / kWave;
        wide.blocks = a.groups * wide.blocks_per_group;
        launch_scan_kernel<T, sp, BACK>(a, wide, ends, sums, st);
        launch_join<true>(a, p, ends, sums, st);
      }
      const size_t lds = sizeof(typename GradShape<sp>::Lds) * waves;
      hipLaunchKernelGGL((scan_grad_kernel<T, sp>), dim3((unsigned)(slots * p.blocks)), dim3(kWave * waves), lds, st, a, p, slots, (const float*)ends, cross, rows);
      if (p.blocks_per_group > 1) {
        const int64_t outs = (int64_t)a.steps * a.envs * a.groups * 2 * sp;
        hipLaunchKernelGGL((cross_sum_kernel<T, sp>), wide_grid((outs + 255) / 256), dim3(256), 0, st, a, p, (const float*)cross);
      }
    });
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_column_sum(rows, slots, SumOutputs{{a.da, a.dskip, a.dbias}, {a.dim * a.states, a.dim, a.dim}}, st);
}

hipError_t launch_scan_step(const ScanArgs& a, hipStream_t st) {
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto lanes) {
      const StepShape s = step_shape((int64_t)a.dim * lanes, a.envs);
      if (s.each == 4) hipLaunchKernelGGL((scan_step_kernel<T, lanes, 4>), s.grid(), s.block(), 0, st, a);
      else hipLaunchKernelGGL((scan_step_kernel<T, lanes, 1>), s.grid(), s.block(), 0, st, a);
    };
    if (a.states % 4) {
      StepShape s = step_shape(a.dim, 1);
      const int64_t blocks = ((int64_t)a.envs + s.rows - 1) / s.rows;
      s.grid_.y = (unsigned)std::min<int64_t>(blocks, kEnvRow);
      s.grid_.z = (unsigned)((blocks + kEnvRow - 1) / kEnvRow);
      hipLaunchKernelGGL(scan_step_any_kernel<T>, s.grid(), s.block(), 0, st, a);
    } else if (a.states == 4) go(std::integral_constant<int, 1>{});
    else if (a.states == 8) go(std::integral_constant<int, 2>{});
    else if (a.states <= 16) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
  });
  return hipGetLastError();
}

}  // namespace gbx
