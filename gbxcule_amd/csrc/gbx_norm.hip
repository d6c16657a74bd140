// gbx_norm.hip -- root-mean-square norm with the residual's addition, its
// gradient and its output in 8 bits, and the column sums that the gradients
// of shared inputs end with.
#include "gbx_rows.h"

namespace gbx {
namespace {

// As sum_over, the maximum of bit patterns of absolute values.
template <int LANES>
__device__ __forceinline__ uint32_t max_over(uint32_t v, float* lds) {
#pragma unroll
  for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
    v = o > v ? o : v;
  }
  if constexpr (LANES > 64) {
    uint32_t* all = reinterpret_cast<uint32_t*>(lds);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) all[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) v = all[w] > v ? all[w] : v;
  }
  return v;
}

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleFloor = 1e-30f;  // keeps the scale of an all-zero group positive

// y = s * rsqrt(mean(s^2) + eps) * weight with s = x + residual rounded to the
// stream's type, so that the gradient sees the s that was normalised.
//
// LANES lanes hold one row, kVec * NV channels each, in registers: x and the
// residual are read once, y and s written once.  NV = 0 takes rows of any
// length in steps of the workgroup and reads the row a second time.
//
// Bound by memory: 131,072 rows of 512 channels in bf16 with a residual move
// 537 MB in 89 us (6.0 TB/s; a copy reaches 4.9), 20,011 rows of 1,024 to 8
// bits 144 MB in 27 us (5.4 TB/s).  64 rows take 3 us, a launch's least.
template <typename T, int LANES, int NV, int ENDS, bool FP8>
__global__ __launch_bounds__(threads_of(LANES)) void norm_kernel(NormArgs a) {
  constexpr int kRows = threads_of(LANES) / LANES, kHeld = NV ? NV : 1;
  __shared__ float lds[16];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, dim = a.dim;
  const int rounds = NV ? NV : (dim + kVec * LANES - 1) / (kVec * LANES);
  const float inv_dim = 1.0f / (float)dim;
  float w[kHeld][kVec];
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      load_row<kVec>(a.weight + e.c, e.valid, w[k]);
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* r = (const T*)a.residual + row * a.residual_stride;
    T* out = (T*)a.out + row * dim;
    T* summed = (T*)a.summed + row * dim;
    float s[kHeld][kVec], ss = 0.0f;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      float(&v)[kVec] = s[NV ? k : 0];
      load_row<kVec>(x + e.c, e.valid, v);
      if (a.residual) {
        float o[kVec];
        load_row<kVec>(r + e.c, e.valid, o);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = (float)(T)(v[i] + o[i]);
        store_row<kVec>(summed + e.c, e.valid, v);
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) ss = ENDS == LAPPED && i < e.skip ? ss : fmaf(v[i], v[i], ss);
    }
    const float rstd = rsqrtf(fmaf(sum_over<LANES>(ss, lds), inv_dim, a.eps));
    auto normed = [&](int k, float (&y)[kVec]) {
      if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] = s[k][i] * rstd * w[k][i];
      } else {
        const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
        float wk[kVec];
        load_row<kVec>((a.residual ? summed : x) + e.c, e.valid, y);
        load_row<kVec>(a.weight + e.c, e.valid, wk);
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] *= rstd * wk[i];
      }
    };
    auto most = [&](int k, const float (&y)[kVec], uint32_t m) {
      // bit patterns of absolute values order as the values do, NaN above all
      const int skip = piece_of<ENDS>(k * LANES + lane, dim).skip;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t b = __float_as_uint(y[i]) & 0x7FFFFFFFu;
        m = b > m && !(ENDS == LAPPED && i < skip) ? b : m;
      }
      return m;
    };
    if constexpr (FP8) {
      uint32_t row_most = 0;
      if (a.group == 0) {
#pragma unroll
        for (int k = 0; k < rounds; ++k) {
          float y[kVec];
          normed(k, y);
          row_most = most(k, y, row_most);
        }
        row_most = max_over<LANES>(row_most, lds);
      }
      uint8_t* q = (uint8_t*)a.out + row * dim;
      const int groups = a.group ? (dim + 127) / 128 : 1;
#pragma unroll
      for (int k = 0; k < rounds; ++k) {
        const int c = (k * LANES + lane) * kVec;  // without the shared channels, whose scale may be another one
        const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
        float y[kVec];
        normed(k, y);
        // 128 channels are 16 neighbouring lanes
        const uint32_t m = a.group ? max_over<16>(most(k, y, 0u), lds) : row_most;
        const float top = m > 0x7F800000u ? __uint_as_float(m) : fmaxf(__uint_as_float(m), kScaleFloor);
        const float inv = kE4m3Max / top;
        if (a.group ? (lane % 16 == 0 && c < dim) : (lane == 0 && k == 0)) a.scale[row * groups + (a.group ? c / 128 : 0)] = top / kE4m3Max;
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
        const uint64_t both = (uint32_t)lo | (uint64_t)(uint32_t)hi << 32;
        if (e.valid >= kVec && e.skip == 0) {
          __builtin_memcpy(q + e.c, &both, 8);
        } else {
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (i < e.valid && i >= e.skip) q[e.c + i] = (uint8_t)(both >> (8 * i));
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < rounds; ++k) {
        const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
        float y[kVec];
        normed(k, y);
        store_row<kVec>(out + e.c, e.valid, y);
      }
    }
  }
}

// With g = weight * dy and r = rsqrt(mean(s^2) + eps):
//   ds = r * g - s * r^3 * mean(g * s) + dsummed,   dweight = sum over rows of dy * s * r.
// The row stays in registers as in the forward kernel; both means come from
// one pass, so nothing but s itself has to be kept from the forward.  A
// workgroup sums dweight over its rows in registers, then over its row slots
// in LDS, and writes one row of partial sums: no atomics, one order.
//
// Bound by memory: 131,072 rows of 512 channels in bf16 with the sum's gradient
// move 537 MB in 106 us (5.1 TB/s); twice the workgroups are slower, since each
// has a row of partial sums to write and to have added.
template <typename T, int LANES, int NV, int ENDS>
__global__ __launch_bounds__(threads_of(LANES)) void norm_grad_kernel(NormGradArgs a) {
  constexpr int kThreads = threads_of(LANES), kRows = kThreads / LANES, kHeld = NV ? NV : 1;
  __shared__ float lds[16];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, dim = a.dim;
  const int rounds = NV ? NV : (dim + kVec * LANES - 1) / (kVec * LANES);
  const float inv_dim = 1.0f / (float)dim;
  float* part = a.work + (int64_t)blockIdx.x * dim;
  float w[kHeld][kVec], dw[kHeld][kVec];
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      load_row<kVec>(a.weight + e.c, e.valid, w[k]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) dw[k][i] = 0.0f;
    }
  }
  const int64_t first = (int64_t)blockIdx.x * kRows + sub;
  for (int64_t row = first; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    const T* sp = (const T*)a.summed + row * a.summed_stride;
    const T* dyp = (const T*)a.dy + row * a.dy_stride;
    const T* dsp = (const T*)a.dsummed + row * a.dsummed_stride;
    T* dxp = (T*)a.dx + row * dim;
    float s[kHeld][kVec], dy[kHeld][kVec], ss = 0.0f, gs = 0.0f;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      load_row<kVec>(sp + e.c, e.valid, s[h]);
      load_row<kVec>(dyp + e.c, e.valid, dy[h]);
      if constexpr (NV == 0) load_row<kVec>(a.weight + e.c, e.valid, w[0]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const bool mine = ENDS != LAPPED || i >= e.skip;
        ss = mine ? fmaf(s[h][i], s[h][i], ss) : ss;
        gs = mine ? fmaf(s[h][i], dy[h][i] * w[h][i], gs) : gs;
      }
    }
    const float rstd = rsqrtf(fmaf(sum_over<LANES>(ss, lds), inv_dim, a.eps));
    const float pull = sum_over<LANES>(gs, lds) * inv_dim * rstd * rstd;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      if constexpr (NV == 0) {
        load_row<kVec>(sp + e.c, e.valid, s[0]);
        load_row<kVec>(dyp + e.c, e.valid, dy[0]);
        load_row<kVec>(a.weight + e.c, e.valid, w[0]);
      }
      float dx[kVec];
      if (a.dsummed) {
        load_row<kVec>(dsp + e.c, e.valid, dx);
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) dx[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        dx[i] = fmaf(rstd, fmaf(-s[h][i], pull, dy[h][i] * w[h][i]), dx[i]);
        const float grow = dy[h][i] * (s[h][i] * rstd);
        if constexpr (NV > 0) dw[k][i] += grow;
        else if (i >= e.skip && i < e.valid) part[e.c + i] = row == first ? grow : part[e.c + i] + grow;
      }
      store_row<kVec>(dxp + e.c, e.valid, dx);
    }
  }
  if constexpr (NV > 0) {
    if constexpr (kRows > 1) {
      __shared__ float tile[kThreads * NV * kVec];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (i < e.valid) tile[sub * (LANES * NV * kVec) + e.c + i] = dw[k][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < dim; c += kThreads) {
        float v = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) v += tile[r * (LANES * NV * kVec) + c];
        part[c] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
        store_row<kVec>(part + e.c, e.valid, dw[k]);
      }
    }
  }
}

// Sums of the columns of up to three matrices that lie side by side.  16 columns
// by 64 rows of a workgroup at a time, so that a few columns still keep many
// loads in flight; one order, whatever the launch.  1,024 rows of 512 columns:
// 7 us, a quarter of it the launch.
constexpr int kSumCols = 16, kSumRows = 64;
__global__ __launch_bounds__(kSumCols* kSumRows) void column_sum_kernel(const float* in, int rows, SumOutputs to) {
  __shared__ float tile[kSumRows][kSumCols + 1];
  const int stride = to.cols[0] + to.cols[1] + to.cols[2];
  int c = blockIdx.x * kSumCols + threadIdx.x % kSumCols;
  const int r0 = threadIdx.x / kSumCols;
  float v = 0.0f;
  if (c < stride)
    for (int r = r0; r < rows; r += kSumRows) v += in[(int64_t)r * stride + c];
  tile[r0][threadIdx.x % kSumCols] = v;
  __syncthreads();
#pragma unroll
  for (int m = kSumRows / 2; m > 0; m >>= 1) {
    if (r0 < m) tile[r0][threadIdx.x % kSumCols] += tile[r0 + m][threadIdx.x % kSumCols];
    __syncthreads();
  }
  if (r0 != 0) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (c >= 0 && c < to.cols[k] && to.out[k]) to.out[k][c] = tile[0][threadIdx.x];
    c -= to.cols[k];
  }
}

}  // namespace

hipError_t launch_column_sum(const float* in, int rows, const SumOutputs& to, hipStream_t st) {
  const int cols = to.cols[0] + to.cols[1] + to.cols[2];
  hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)((cols + kSumCols - 1) / kSumCols)), dim3(kSumCols * kSumRows), 0, st, in, rows, to);
  return hipGetLastError();
}

hipError_t launch_rms_norm(const NormArgs& a, hipStream_t st) {
  const int64_t per = rows_of_block(a.dim);
  const dim3 grid((unsigned)std::min<int64_t>((a.rows + per - 1) / per, 1 << 16));
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_row_length(a.dim, [&](auto lanes, auto nv) {
      by_ends(a.dim, [&](auto ends) {
        if constexpr (ends != TINY || lanes == 16) {
          if (a.scale) hipLaunchKernelGGL((norm_kernel<T, lanes, nv, ends, true>), grid, dim3(threads_of(lanes)), 0, st, a);
          else hipLaunchKernelGGL((norm_kernel<T, lanes, nv, ends, false>), grid, dim3(threads_of(lanes)), 0, st, a);
        }
      });
    });
  });
  return hipGetLastError();
}

int64_t norm_grad_work(int64_t rows, int dim) { return (int64_t)grad_blocks(rows, dim) * dim; }

hipError_t launch_rms_norm_grad(const NormGradArgs& a, hipStream_t st) {
  const int blocks = grad_blocks(a.rows, a.dim);
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_row_length(a.dim, [&](auto lanes, auto nv) {
      by_ends(a.dim, [&](auto ends) {
        if constexpr (ends != TINY || lanes == 16) hipLaunchKernelGGL((norm_grad_kernel<T, lanes, nv, ends>), dim3((unsigned)blocks), dim3(threads_of(lanes)), 0, st, a);
      });
    });
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_column_sum(a.work, blocks, SumOutputs{{a.dweight}, {a.dim}}, st);
}

}  // namespace gbx
