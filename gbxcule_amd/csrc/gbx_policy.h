// gbx_policy.h -- operators of a policy with memory: arguments, launch
// wrappers and the device helpers that their kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gbx {

// Element types of the C ABI (GBX_F32, GBX_BF16, GBX_F16).
enum { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };

struct NormArgs {
  int64_t rows;
  int dim, elem;
  float eps;
  const void *x, *residual;  // residual may be NULL
  int64_t x_stride, residual_stride;
  const float* weight;
  void *out, *summed;  // contiguous; summed NULL without a residual
  float* scale;        // fp8 output only
  int group;           // channels that share a scale; 0: the row
};
struct NormGradArgs {
  int64_t rows;
  int dim, elem;
  float eps;
  const void *summed, *dy, *dsummed;  // dsummed may be NULL
  int64_t summed_stride, dy_stride, dsummed_stride;
  const float* weight;
  void* dx;
  float *dweight, *work;
};
struct ConvArgs {
  int steps, envs, dim, width, elem, silu;
  const void* x;
  int64_t x_step, x_env;
  const float *weight, *bias;  // [dim][width], [dim] or NULL
  const void* state;           // [envs][width - 1][dim] or NULL
  const uint8_t* resets;       // [steps][envs] or NULL
  void *y, *last;              // contiguous
  const void* dy;              // the rest: gradient only
  int64_t dy_step, dy_env;
  void* dx;
  float *dweight, *dbias, *work;
};
struct ScanArgs {
  int steps, envs, dim, groups, states, elem, softplus;
  const void *x, *dt, *z, *b, *c;  // z may be NULL
  int64_t x_step, x_env, dt_step, dt_env, z_step, z_env;
  int64_t b_step, b_env, b_group, c_step, c_env, c_group;
  const float *a, *skip, *bias;  // [dim][states], [dim] or NULL, [dim] or NULL
  const float* state;            // [envs][dim][states] or NULL
  const uint8_t* resets;         // [steps][envs] or NULL
  void* y;                       // contiguous
  float* last;                   // [envs][dim][states]
  float* saved;                  // states before every kSegment-th step, or NULL
  float* work;
  const void* dy;  // the rest: gradient only
  int64_t dy_step, dy_env;
  void *dx, *ddt, *dz, *db, *dc;  // contiguous
  float *da, *dskip, *dbias;
};
struct AdamArgs {
  int count, elem, grad_elem, small;  // small: 8-bit states
  const uint64_t *params, *grads;     // host: device addresses
  const int64_t *sizes, *starts;      // host: elements; where its states start, a multiple of kStateBlock
  void *exp_avg, *exp_avg_sq;
  float *exp_avg_scale, *exp_avg_sq_scale;  // 8 bits only
  const float* grad_scale;                  // device, may be NULL
  float beta1, rest1, beta2, rest2, step_size, inv_root2, eps, keep;
  uint32_t key;
};
constexpr int kStateBlock = 256;  // elements that share a scale
constexpr int kSegment = 8;     // steps between two saved states
constexpr int kMaxStates = 32;  // states a channel may have

// Sums over `rows` rows of partial sums that lie one after the other, in one
// order.  The columns are up to three outputs' in turn; those whose pointer is
// NULL are left out.
struct SumOutputs {
  float* out[3];
  int cols[3];
};
hipError_t launch_column_sum(const float* in, int rows, const SumOutputs& to, hipStream_t st);
hipError_t launch_rms_norm(const NormArgs& a, hipStream_t st);
int64_t norm_grad_work(int64_t rows, int dim);
hipError_t launch_rms_norm_grad(const NormGradArgs& a, hipStream_t st);
hipError_t launch_conv(const ConvArgs& a, hipStream_t st);
int64_t conv_grad_work(int steps, int envs, int dim, int width);
hipError_t launch_conv_grad(const ConvArgs& a, hipStream_t st);
hipError_t launch_conv_step(const ConvArgs& a, hipStream_t st);
int64_t scan_work(int steps, int envs, int dim, int groups, int states);
hipError_t launch_scan(const ScanArgs& a, hipStream_t st);
int64_t scan_grad_work(int steps, int envs, int dim, int groups, int states);
hipError_t launch_scan_grad(const ScanArgs& a, hipStream_t st);
hipError_t launch_scan_step(const ScanArgs& a, hipStream_t st);
hipError_t launch_adamw(const AdamArgs& a, hipStream_t st);

// A grid has fewer than 2^32 threads: more workgroups than 2^22 go to its
// second dimension, and block_id() counts them.
inline dim3 wide_grid(int64_t blocks) {
  constexpr int64_t kRow = 1 << 22;
  return blocks <= kRow ? dim3((unsigned)blocks) : dim3((unsigned)kRow, (unsigned)((blocks + kRow - 1) / kRow));
}

// Single steps: a workgroup is some lanes of a few envs.  Lanes are the grid's
// first dimension, envs the two others.  A lane takes EACH envs, with their
// loads in flight together and what envs share (weights, rates) loaded once:
// 4 from 524,288 lanes on (16,384 envs of 512 channels: the convolution's step
// 31.3 -> 26.4 us, the scan's 267 -> 234), else 1, so that few envs spread.
constexpr int kEnvRow = 1 << 15;
struct StepShape {
  int threads, rows, each;  // lanes and envs of a workgroup; envs of a lane
  dim3 grid() const { return grid_; }
  dim3 block() const { return dim3((unsigned)threads, (unsigned)rows); }
  dim3 grid_;
};
inline StepShape step_shape(int64_t lanes, int envs) {
  StepShape s;
  s.threads = 1;
  while (s.threads < 256 && s.threads < lanes) s.threads <<= 1;
  s.rows = 256 / s.threads;
  s.each = lanes * envs >= (int64_t)256 * 2048 ? 4 : 1;
  const int64_t blocks = ((int64_t)envs + s.rows * s.each - 1) / (s.rows * s.each);
  s.grid_ = dim3((unsigned)((lanes + s.threads - 1) / s.threads), (unsigned)(blocks < kEnvRow ? blocks : kEnvRow), (unsigned)((blocks + kEnvRow - 1) / kEnvRow));
  return s;
}

// f(a value of the element type)
template <typename F>
void by_element(int elem, F&& f) {
  if (elem == ELEM_F32) f(float{});
  else if (elem == ELEM_BF16) f(__bf16{});
  else f(_Float16{});
}

// `count` consecutive elements as floats, zero from `valid` on.  Rows of odd
// length start at any element, so the loads ask for no alignment: the
// compiler emits one wide load, which the hardware takes at any address.
template <int COUNT, typename T>
__device__ __forceinline__ void load_row(const T* p, int valid, float (&v)[COUNT]) {
  if (valid >= COUNT) {
    T r[COUNT];
    __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = (float)r[i];
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = i < valid ? (float)p[i] : 0.0f;
  }
}
template <int COUNT, typename T>
__device__ __forceinline__ void store_row(T* p, int valid, const float (&v)[COUNT]) {
  if (valid >= COUNT) {
    T r[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) r[i] = (T)v[i];
    __builtin_memcpy(p, r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}

// (the library's 64-bit min goes through double precision)
__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

// a lane's first env; the others follow blockDim.y apart
template <int EACH>
__device__ __forceinline__ int64_t first_env() { return ((int64_t)blockIdx.z * kEnvRow + blockIdx.y) * (blockDim.y * EACH) + threadIdx.y; }
__device__ __forceinline__ int64_t block_id() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
// 2^x, 1 / x and log2 x in one instruction each
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float sigmoid(float x) { return rcp_fast(1.0f + exp2_fast(-kLog2e * x)); }

}  // namespace gbx
