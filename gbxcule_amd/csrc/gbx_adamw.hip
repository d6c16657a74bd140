// gbx_adamw.hip -- AdamW over many tensors in a launch, with its two moments
// in 32 bits or in 8 bits with a scale for each 256 elements.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = (1 - lr decay) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// An element is read and written once: 28 bytes with 32-bit states and
// parameters, 10 with 8-bit states and 16-bit parameters.
#include <algorithm>

#include "gbx_policy.h"

namespace gbx {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = kStateBlock;       // 256: a wavefront, 4 elements a lane
constexpr int kTileBlocks = 16;           // of a workgroup's tile
constexpr int kTile = kTileBlocks * kBlock;

struct Tensor {
  void* p;
  const void* g;
  int64_t n;
  uint32_t start;  // first block of its states
  uint32_t tile;   // first tile of the launch
};
constexpr int kTensors = 100;  // of a launch: they travel as kernel arguments, 4 KB at most
struct Tensors {
  int count;
  Tensor t[kTensors];
};

// 32 random bits of an element and a step: two rounds of multiplying by an odd
// constant (the fractions of the golden ratio and of the square root of 2) and
// folding the high bits in.
__device__ __forceinline__ uint32_t noise_of(uint32_t index, uint32_t key) {
  uint32_t h = (index ^ key) * 0x9E3779B9u;
  h ^= h >> 16;
  h *= 0x6A09E667u;
  return h ^ (h >> 15);
}

// v rounded to MANTISSA bits, up with the odds of its distance from the value
// below (16 random bits), so that a running mean moves even where each change
// is less than half a step of the format.  LEAST: the smallest normal value.
template <int MANTISSA>
__device__ __forceinline__ float round_8(float v, uint32_t noise16, float least) {
  constexpr int kCut = 23 - MANTISSA;
  const float mag = fabsf(v);
  const uint32_t bits = __float_as_uint(mag) + (noise16 << (kCut - 16));
  const float normal = __uint_as_float(bits & ~((1u << kCut) - 1u));
  const float quantum = least / (float)(1 << MANTISSA), steps = mag * (1.0f / quantum), whole = floorf(steps);
  const float small = (whole + floorf((steps - whole) + (float)noise16 * 0x1p-16f)) * quantum;
  return copysignf(mag < least ? small : normal, v);
}

// Largest bit pattern (absolute values order as their bits do, NaN above all)
// of the wavefront.
__device__ __forceinline__ float wave_most(uint32_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
    v = o > v ? o : v;
  }
  return __uint_as_float(v);
}
__device__ __forceinline__ uint32_t most4(const float (&v)[4]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
    m = b > m ? b : m;
  }
  return m;
}
constexpr float kScaleFloor = 1e-30f, kE4m3Max = 448.0f, kE5m2Max = 57344.0f;

template <typename P, typename G, bool SMALL>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamArgs a, Tensors ts) {
#pragma clang fp contract(off)  // each operation rounds, as in the formula
  // the workgroup's tensor: the last one whose first tile is not beyond it
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int which = -1;
#pragma unroll
  for (int k = 0; k < kTensors; k += 64) {
    const bool has = k + lane < ts.count && ts.t[min(k + lane, kTensors - 1)].tile <= blockIdx.x;
    which += __popcll(__ballot(has));
  }
  const Tensor t = ts.t[__builtin_amdgcn_readfirstlane(which)];
  const float grad_scale = a.grad_scale ? *a.grad_scale : 1.0f;
  const int64_t first = (int64_t)(blockIdx.x - t.tile) * kTile;
#pragma unroll
  for (int k = 0; k < kTileBlocks / 4; ++k) {
    const int64_t at = first + (int64_t)(k * 4 + wave) * kBlock, e = at + lane * 4;  // in the tensor
    if (at >= t.n) return;
    const int64_t block = t.start + at / kBlock, s = block * kBlock + lane * 4;  // in the states
    const int valid = (int)min<int64_t>(4, max<int64_t>(0, t.n - e));
    float p[4], g[4], m[4], v[4];
    load_row<4>((const P*)t.p + e, valid, p);
    load_row<4>((const G*)t.g + e, valid, g);
    if constexpr (SMALL) {
      const uint32_t mq = *(const uint32_t*)((const uint8_t*)a.exp_avg + s), vq = *(const uint32_t*)((const uint8_t*)a.exp_avg_sq + s);
      const float ms = a.exp_avg_scale[block], vs = a.exp_avg_sq_scale[block];
      m[0] = __builtin_amdgcn_cvt_f32_fp8((int)mq, 0) * ms;
      m[1] = __builtin_amdgcn_cvt_f32_fp8((int)mq, 1) * ms;
      m[2] = __builtin_amdgcn_cvt_f32_fp8((int)mq, 2) * ms;
      m[3] = __builtin_amdgcn_cvt_f32_fp8((int)mq, 3) * ms;
      v[0] = __builtin_amdgcn_cvt_f32_bf8((int)vq, 0) * vs;
      v[1] = __builtin_amdgcn_cvt_f32_bf8((int)vq, 1) * vs;
      v[2] = __builtin_amdgcn_cvt_f32_bf8((int)vq, 2) * vs;
      v[3] = __builtin_amdgcn_cvt_f32_bf8((int)vq, 3) * vs;
    } else {
      load_row<4>((const float*)a.exp_avg + s, 4, m);
      load_row<4>((const float*)a.exp_avg_sq + s, 4, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gi = g[i] * grad_scale;
      m[i] = m[i] * a.beta1 + gi * a.rest1;
      v[i] = v[i] * a.beta2 + gi * gi * a.rest2;
      // root and quotient to one unit in the last place: the update is added
      // to a parameter many times its size
      const float update = (m[i] * a.step_size) * rcp_fast(__builtin_amdgcn_sqrtf(v[i]) * a.inv_root2 + a.eps);
      p[i] = p[i] * a.keep - update;
    }
    store_row<4>((P*)t.p + e, valid, p);
    if constexpr (SMALL) {
      const float most_m = wave_most(most4(m)), most_v = wave_most(most4(v));
      const float top_m = most_m < kScaleFloor ? kScaleFloor : most_m, top_v = most_v < kScaleFloor ? kScaleFloor : most_v;
      const float inv_m = kE4m3Max / top_m, inv_v = kE5m2Max / top_v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t noise = noise_of((uint32_t)(s + i), a.key);
        float x = m[i] * inv_m, y = v[i] * inv_v;
        x = fabsf(x) > kE4m3Max ? copysignf(kE4m3Max, x) : x;
        y = y > kE5m2Max ? kE5m2Max : y;
        m[i] = round_8<3>(x, noise & 0xFFFFu, 0x1p-6f);
        const float q = round_8<2>(y, noise >> 16, 0x1p-14f);
        v[i] = y > 0.0f && q < 0x1p-16f ? 0x1p-16f : q;  // a second moment that is not zero stays so
      }
      int mq = __builtin_amdgcn_cvt_pk_fp8_f32(m[0], m[1], 0, false);
      mq = __builtin_amdgcn_cvt_pk_fp8_f32(m[2], m[3], mq, true);
      int vq = __builtin_amdgcn_cvt_pk_bf8_f32(v[0], v[1], 0, false);
      vq = __builtin_amdgcn_cvt_pk_bf8_f32(v[2], v[3], vq, true);
      *(uint32_t*)((uint8_t*)a.exp_avg + s) = (uint32_t)mq;
      *(uint32_t*)((uint8_t*)a.exp_avg_sq + s) = (uint32_t)vq;
      if (lane == 0) {
        a.exp_avg_scale[block] = top_m / kE4m3Max;
        a.exp_avg_sq_scale[block] = top_v / kE5m2Max;
      }
    } else {
      store_row<4>((float*)a.exp_avg + s, 4, m);
      store_row<4>((float*)a.exp_avg_sq + s, 4, v);
    }
  }
}

}  // namespace

hipError_t launch_adamw(const AdamArgs& a, hipStream_t st) {
  Tensors ts;
  for (int i = 0; i < a.count;) {
    uint32_t tiles = 0;
    ts.count = 0;
    for (; i < a.count && ts.count < kTensors; ++i) {
      if (a.sizes[i] == 0) continue;
      const int64_t more = (a.sizes[i] + kTile - 1) / kTile;
      if (ts.count > 0 && tiles + more > (1 << 23)) break;  // a grid has fewer than 2^32 threads
      ts.t[ts.count++] = Tensor{(void*)(uintptr_t)a.params[i], (const void*)(uintptr_t)a.grads[i], a.sizes[i], (uint32_t)(a.starts[i] / kBlock), tiles};
      tiles += (uint32_t)more;
    }
    if (tiles == 0) break;
    const dim3 grid(tiles), block(kThreads);
    by_element(a.elem, [&](auto p) {
      using P = decltype(p);
      auto go = [&](auto g) {
        using G = decltype(g);
        if (a.small) hipLaunchKernelGGL((adamw_kernel<P, G, true>), grid, block, 0, st, a, ts);
        else hipLaunchKernelGGL((adamw_kernel<P, G, false>), grid, block, 0, st, a, ts);
      };
      if (a.grad_elem == a.elem) go(P{});
      else go(float{});
    });
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace gbx
