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
constexpr int kBlock = kStateBlock;
constexpr int kTile = 4096;  // elements of a workgroup

struct Tensor {
  void* p;
  const void* g;
  int64_t n;
  uint32_t start;  // first block of its states
  uint32_t tile;   // first tile
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

// `mag` >= 0 rounded to MANTISSA bits, up with the odds of its distance from the
// value below (16 random bits), so that a running mean moves even where each
// change is less than half a step of the format: the random bits are added
// below the last kept bit and the rest is cut off.  Values below the smallest
// normal one, LEAST, have the spacing of [LEAST, 2 LEAST) and are rounded there.
template <int MANTISSA>
__device__ __forceinline__ float round_8(float mag, uint32_t noise16, float least) {
  constexpr int kCut = 23 - MANTISSA;
  const float lift = mag < least ? least : 0.0f;
  const uint32_t bits = __float_as_uint(mag + lift) + (noise16 << (kCut - 16));
  return __uint_as_float(bits & ~((1u << kCut) - 1u)) - lift;
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
  return o > v ? o : v;
}
// Largest bit pattern over 32 lanes of `a` in the even rows of 16 lanes and of
// `b` in the odd ones (patterns of absolute values order as the values do, NaN
// above all).
__device__ __forceinline__ uint32_t most_of_rows(uint32_t a, uint32_t b) {
  const auto folded = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  const uint32_t v = folded[0] > folded[1] ? folded[0] : folded[1];
  return max_dpp<0x121>(max_dpp<0x122>(max_dpp<0x124>(max_dpp<0x128>(v))));  // rotated by 8, 4, 2, 1
}
constexpr float kScaleFloor = 1e-30f, kE4m3Max = 448.0f, kE5m2Max = 57344.0f;

// One element's update.  The moments round at each operation, as written: in 8
// bits a unit in the last place decides which way a value turns, and the same
// formula elsewhere should turn the same way.  Root and reciprocal are right
// to one unit in the last place: what they make is added to a parameter many
// times its size.
__device__ __forceinline__ float update(const AdamArgs& a, float p, float g, float rest1, float rest2, float& m, float& v) {
#pragma clang fp contract(off)
  m = m * a.beta1 + g * rest1;
  v = v * a.beta2 + g * g * rest2;
  const float root = fmaf(__builtin_amdgcn_sqrtf(v), a.inv_root2, a.eps);
  return fmaf(-m * a.step_size, rcp_fast(root), p * a.keep);
}

// The workgroup's tensor: the last one whose first tile is not beyond it.
__device__ __forceinline__ Tensor tensor_of(const Tensors& ts) {
  const int lane = threadIdx.x & 63;
  int which = -1;
#pragma unroll
  for (int k = 0; k < kTensors; k += 64) {
    const bool has = k + lane < ts.count && ts.t[min(k + lane, kTensors - 1)].tile <= blockIdx.x;
    which += __popcll(__ballot(has));
  }
  return ts.t[__builtin_amdgcn_readfirstlane(which)];
}

// Bound by memory where the tensors are large, by the launch where they are not:
// 24 MB of two blocks' parameters and states take 7 us.
template <typename P, typename G>
__global__ __launch_bounds__(kThreads) void adamw_kernel(AdamArgs a, Tensors ts) {
  const Tensor t = tensor_of(ts);
  const float scale = a.grad_scale ? *a.grad_scale : 1.0f, rest1 = a.rest1 * scale, rest2 = a.rest2 * scale * scale;
  const int64_t first = (int64_t)(blockIdx.x - t.tile) * kTile;
  float* exp_avg = (float*)a.exp_avg + (int64_t)t.start * kBlock;
  float* exp_avg_sq = (float*)a.exp_avg_sq + (int64_t)t.start * kBlock;
#pragma unroll
  for (int k = 0; k < kTile / (4 * kThreads); ++k) {
    const int64_t e = first + (k * kThreads + threadIdx.x) * 4;
    if (e >= t.n) return;
    const int valid = (int)least(4, t.n - e);
    float p[4], g[4], m[4], v[4];
    load_row<4>((const P*)t.p + e, valid, p);
    load_row<4>((const G*)t.g + e, valid, g);
    load_row<4>(exp_avg + e, 4, m);
    load_row<4>(exp_avg_sq + e, 4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = update(a, p[i], g[i], rest1, rest2, m[i], v[i]);
    }
    store_row<4>((P*)t.p + e, valid, p);
    store_row<4>(exp_avg + e, 4, m);
    store_row<4>(exp_avg_sq + e, 4, v);
  }
}

// 8-bit states: 32 lanes hold a block of 256, 8 elements each.  160 million bf16
// parameters in three launches move 1.60 GB in 322 us (5.0 TB/s, as a copy does);
// 4 elements a lane, divisions and a square root rounded to the last bit, and
// the maxima by shuffles had the vector units bound it (466 us).
template <typename P, typename G>
__global__ __launch_bounds__(kThreads) void adamw_8_kernel(AdamArgs a, Tensors ts) {
  const Tensor t = tensor_of(ts);
  const float scale = a.grad_scale ? *a.grad_scale : 1.0f, rest1 = a.rest1 * scale, rest2 = a.rest2 * scale * scale;
  const int64_t first = (int64_t)(blockIdx.x - t.tile) * kTile;
#pragma unroll
  for (int k = 0; k < kTile / (8 * kThreads); ++k) {
    const int64_t e = first + (k * kThreads + threadIdx.x) * 8;  // in the tensor
    if (e / kBlock * kBlock >= t.n) return;                      // all 32 lanes of a block together
    const int64_t block = t.start + e / kBlock, s = (int64_t)t.start * kBlock + e;
    const int valid = t.n > e ? (int)least(8, t.n - e) : 0;
    float p[8], g[8], m[8], v[8];
    load_row<8>((const P*)t.p + e, valid, p);
    load_row<8>((const G*)t.g + e, valid, g);
    const uint2 mq = *(const uint2*)((const uint8_t*)a.exp_avg + s), vq = *(const uint2*)((const uint8_t*)a.exp_avg_sq + s);
    const float ms = a.exp_avg_scale[block], vs = a.exp_avg_sq_scale[block];
    auto widen = [](uint32_t q, float by, float* to, auto bf8) {
      if constexpr (bf8.value) {
        to[0] = __builtin_amdgcn_cvt_f32_bf8((int)q, 0) * by, to[1] = __builtin_amdgcn_cvt_f32_bf8((int)q, 1) * by;
        to[2] = __builtin_amdgcn_cvt_f32_bf8((int)q, 2) * by, to[3] = __builtin_amdgcn_cvt_f32_bf8((int)q, 3) * by;
      } else {
        to[0] = __builtin_amdgcn_cvt_f32_fp8((int)q, 0) * by, to[1] = __builtin_amdgcn_cvt_f32_fp8((int)q, 1) * by;
        to[2] = __builtin_amdgcn_cvt_f32_fp8((int)q, 2) * by, to[3] = __builtin_amdgcn_cvt_f32_fp8((int)q, 3) * by;
      }
    };
    widen(mq.x, ms, m, std::false_type{});
    widen(mq.y, ms, m + 4, std::false_type{});
    widen(vq.x, vs, v, std::true_type{});
    widen(vq.y, vs, v + 4, std::true_type{});
    uint32_t most_m = 0, most_v = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = update(a, p[i], g[i], rest1, rest2, m[i], v[i]);
      const uint32_t bm = __float_as_uint(m[i]) & 0x7FFFFFFFu, bv = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      most_m = bm > most_m ? bm : most_m;
      most_v = bv > most_v ? bv : most_v;
    }
    store_row<8>((P*)t.p + e, valid, p);
    // one reciprocal for both: the first moment's in even rows of 16 lanes
    const bool second = threadIdx.x & 16u;
    const float limit = second ? kE5m2Max : kE4m3Max, most = __uint_as_float(most_of_rows(most_m, most_v));
    const float top = most < kScaleFloor ? kScaleFloor : most, inv = (1.0f / top) * limit;
    if ((threadIdx.x & 15u) == 0u) (second ? a.exp_avg_sq_scale : a.exp_avg_scale)[block] = top * (second ? 1.0f / kE5m2Max : 1.0f / kE4m3Max);
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(inv), __float_as_uint(inv), false, false);
    // (a unit or two above the formats' largest values is cut off below)
    const float inv_m = __uint_as_float(both[0]), inv_v = __uint_as_float(both[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t noise = noise_of((uint32_t)s + i, a.key);
      m[i] *= inv_m;
      v[i] *= inv_v;
      m[i] = copysignf(round_8<3>(fabsf(m[i]), noise & 0xFFFFu, 0x1p-6f), m[i]);
      const float q = round_8<2>(v[i], noise >> 16, 0x1p-14f);
      v[i] = v[i] > 0.0f ? fmaxf(q, 0x1p-16f) : q;  // a second moment that is not zero stays so
    }
    auto narrow = [](const float* v, auto bf8) {
      if constexpr (bf8.value) return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(v[2], v[3], __builtin_amdgcn_cvt_pk_bf8_f32(v[0], v[1], 0, false), true);
      else return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), true);
    };
    *(uint2*)((uint8_t*)a.exp_avg + s) = uint2{narrow(m, std::false_type{}), narrow(m + 4, std::false_type{})};
    *(uint2*)((uint8_t*)a.exp_avg_sq + s) = uint2{narrow(v, std::true_type{}), narrow(v + 4, std::true_type{})};
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
        if (a.small) hipLaunchKernelGGL((adamw_8_kernel<P, G>), grid, block, 0, st, a, ts);
        else hipLaunchKernelGGL((adamw_kernel<P, G>), grid, block, 0, st, a, ts);
      };
      if (a.grad_elem == a.elem) go(P{});
      else go(float{});
    });
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace gbx
