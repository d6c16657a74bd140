// gbx_layer_norm.hip -- layer norm with the residual's addition and its
// gradient, with the sums of the weight's and the bias's.
#include "gbx_rows.h"

namespace gbx {
namespace {

// y = (s - mean(s)) * rsqrt(mean((s - mean(s))^2) + eps) * weight + bias with
// s = x + residual rounded to the stream's type, so that the gradient sees the
// s that was normalised.
//
// The row stays in registers (LANES lanes, kVec * NV channels each; NV = 0:
// longer rows, read again for each of the three passes), so the squares are
// those of what is left when the mean is gone: the mean of the squares minus
// the mean's square would lose as many digits as the mean is larger than the
// spread.  Bound by HBM where there are many rows and by a launch where there are
// few: 131,072 x 512 in 16 bits with a residual in 91 us (537 MB, 5.9 TB/s), with the
// gradient in 205 (1,074 MB, 5.2 TB/s); to 8,192 channels at 5.3 TB/s, over
// that, where each pass reads the row again, 3.8; 64 x 256 in 6.9 us.
template <typename T, int LANES, int NV, int ENDS>
__global__ __launch_bounds__(threads_of(LANES)) void layer_norm_kernel(LayerNormArgs a) {
  constexpr int kRows = threads_of(LANES) / LANES, kHeld = NV ? NV : 1;
  __shared__ float lds[16];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, dim = a.dim;
  const int rounds = NV ? NV : (dim + kVec * LANES - 1) / (kVec * LANES);
  const float inv_dim = 1.0f / (float)dim;
  float w[kHeld][kVec], b[kHeld][kVec];
  auto params = [&](int k, int h) {
    const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
    load_row<kVec>(a.weight + e.c, e.valid, w[h]);
    if (a.bias) {
      load_row<kVec>(a.bias + e.c, e.valid, b[h]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) b[h][i] = 0.0f;
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) params(k, k);
  }
  for (int64_t row = (int64_t)blockIdx.x * kRows + sub; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* r = (const T*)a.residual + row * a.residual_stride;
    T* out = (T*)a.out + row * dim;
    T* summed = (T*)a.summed + row * dim;
    float s[kHeld][kVec], total = 0.0f;
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
      for (int i = 0; i < kVec; ++i) total += ENDS == LAPPED && i < e.skip ? 0.0f : v[i];
    }
    const float mean = sum_over<LANES>(total, lds) * inv_dim;
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      float(&v)[kVec] = s[NV ? k : 0];
      if constexpr (NV == 0) load_row<kVec>((a.residual ? summed : x) + e.c, e.valid, v);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        v[i] -= mean;
        ss = i < e.valid && i >= e.skip ? fmaf(v[i], v[i], ss) : ss;
      }
    }
    const float rstd = rsqrtf(fmaf(sum_over<LANES>(ss, lds), inv_dim, a.eps));
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      if constexpr (NV == 0) {
        load_row<kVec>((a.residual ? summed : x) + e.c, e.valid, s[0]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) s[0][i] -= mean;
        params(k, 0);
      }
      float y[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) y[i] = fmaf(s[h][i] * rstd, w[h][i], b[h][i]);
      store_row<kVec>(out + e.c, e.valid, y);
    }
  }
}

// g - mean without a fused product: where all g are equal nothing is left, as
// their mean is of the same rounded products.
__device__ __forceinline__ float less(float g, float mean) {
#pragma clang fp contract(off)
  return g - mean;
}

// With c = s - mean(s), g = weight * dy and r = rsqrt(mean(c^2) + eps):
//   ds = r * (g - mean(g) - c * r^2 * mean(g * c)) + dsummed,
//   dweight = sum over rows of dy * c * r,  dbias = sum over rows of dy.
// The row stays in registers as in the forward kernel and its mean is summed
// again, so nothing but s itself has to be kept from the forward; the other
// three sums are made in one pass over the row, each with an exchange of its own.  A workgroup sums dweight and dbias over its rows in
// registers, then over its row slots in LDS, and writes one row of partial
// sums, dbias's columns after dweight's: no atomics, one order.  Bound by HBM; rows
// that no 16-byte load divides cost what their split lines do (20,011 x 1,023 in 32
// bits, forward and gradient: 95 us, 410 MB with x once for each, 4.3 TB/s).  Two pieces
// a lane leave registers for three wavefronts a SIMD (65,536 x 1,024 in 16 bits with a
// residual: 162 us, 3.3 TB/s); rows over 1,024 channels are a workgroup's, whose eight
// barriers a row nothing else fills (32,768 x 2,048 135 us, 4.0 TB/s; 8,192 x 8,192 182 us,
// 2.9); over 8,192 every pass reads the row again, and a workgroup's partial sums are in
// memory (4,096 x 16,384: 784 us).
template <typename T, int LANES, int NV, int ENDS>
__global__ __launch_bounds__(threads_of(LANES)) void layer_norm_grad_kernel(LayerNormGradArgs a) {
  constexpr int kThreads = threads_of(LANES), kRows = kThreads / LANES, kHeld = NV ? NV : 1;
  __shared__ float lds[16];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, dim = a.dim;
  const int rounds = NV ? NV : (dim + kVec * LANES - 1) / (kVec * LANES);
  const float inv_dim = 1.0f / (float)dim;
  float* part_w = a.work + (int64_t)blockIdx.x * 2 * dim;
  float* part_b = part_w + dim;
  float w[kHeld][kVec], dw[kHeld][kVec], db[kHeld][kVec];
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      load_row<kVec>(a.weight + e.c, e.valid, w[k]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) dw[k][i] = db[k][i] = 0.0f;
    }
  }
  const int64_t first = (int64_t)blockIdx.x * kRows + sub;
  for (int64_t row = first; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    const T* sp = (const T*)a.summed + row * a.summed_stride;
    const T* dyp = (const T*)a.dy + row * a.dy_stride;
    const T* dsp = (const T*)a.dsummed + row * a.dsummed_stride;
    T* dxp = (T*)a.dx + row * dim;
    float s[kHeld][kVec], dy[kHeld][kVec], total = 0.0f;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      load_row<kVec>(sp + e.c, e.valid, s[h]);
      if constexpr (NV > 0) load_row<kVec>(dyp + e.c, e.valid, dy[h]);
#pragma unroll
      for (int i = 0; i < kVec; ++i) total += ENDS == LAPPED && i < e.skip ? 0.0f : s[h][i];
    }
    const float mean = sum_over<LANES>(total, lds) * inv_dim;
    float ss = 0.0f, gs = 0.0f, gc = 0.0f;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      if constexpr (NV == 0) {
        load_row<kVec>(sp + e.c, e.valid, s[0]);
        load_row<kVec>(dyp + e.c, e.valid, dy[0]);
        load_row<kVec>(a.weight + e.c, e.valid, w[0]);
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const bool mine = i < e.valid && i >= e.skip;
        const float g = dy[h][i] * w[h][i];
        s[h][i] -= mean;
        ss = mine ? fmaf(s[h][i], s[h][i], ss) : ss;
        gs = mine ? gs + g : gs;
        gc = mine ? fmaf(s[h][i], g, gc) : gc;
      }
    }
    const float rstd = rsqrtf(fmaf(sum_over<LANES>(ss, lds), inv_dim, a.eps));
    const float shift = sum_over<LANES>(gs, lds) * inv_dim;
    const float pull = sum_over<LANES>(gc, lds) * inv_dim * rstd * rstd;
#pragma unroll
    for (int k = 0; k < rounds; ++k) {
      const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
      const int h = NV ? k : 0;
      if constexpr (NV == 0) {
        load_row<kVec>(sp + e.c, e.valid, s[0]);
        load_row<kVec>(dyp + e.c, e.valid, dy[0]);
        load_row<kVec>(a.weight + e.c, e.valid, w[0]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) s[0][i] -= mean;
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
        dx[i] = fmaf(rstd, fmaf(-s[h][i], pull, less(dy[h][i] * w[h][i], shift)), dx[i]);
        const float grow = dy[h][i] * (s[h][i] * rstd);
        if constexpr (NV > 0) {
          dw[k][i] += grow;
          db[k][i] += dy[h][i];
        } else if (i >= e.skip && i < e.valid) {
          part_w[e.c + i] = row == first ? grow : part_w[e.c + i] + grow;
          part_b[e.c + i] = row == first ? dy[h][i] : part_b[e.c + i] + dy[h][i];
        }
      }
      store_row<kVec>(dxp + e.c, e.valid, dx);
    }
  }
  if constexpr (NV > 0) {
    auto join = [&](const float (&mine)[kHeld][kVec], float* part) {
      if constexpr (kRows > 1) {
        __shared__ float tile[kThreads * NV * kVec];
        __syncthreads();  // the last use of tile has been read
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const Piece e = piece_of<ENDS>(k * LANES + lane, dim);
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (i < e.valid) tile[sub * (LANES * NV * kVec) + e.c + i] = mine[k][i];
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
          store_row<kVec>(part + e.c, e.valid, mine[k]);
        }
      }
    };
    join(dw, part_w);
    join(db, part_b);
  }
}

}  // namespace

hipError_t launch_layer_norm(const LayerNormArgs& a, hipStream_t st) {
  const int64_t per = rows_of_block(a.dim);
  const dim3 grid((unsigned)std::min<int64_t>((a.rows + per - 1) / per, 1 << 16));
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_row_length(a.dim, [&](auto lanes, auto nv) {
      by_ends(a.dim, [&](auto ends) {
        if constexpr (ends != TINY || lanes == 16) hipLaunchKernelGGL((layer_norm_kernel<T, lanes, nv, ends>), grid, dim3(threads_of(lanes)), 0, st, a);
      });
    });
  });
  return hipGetLastError();
}

int64_t layer_norm_grad_work(int64_t rows, int dim) { return (int64_t)grad_blocks(rows, dim) * 2 * dim; }

hipError_t launch_layer_norm_grad(const LayerNormGradArgs& a, hipStream_t st) {
  const int blocks = grad_blocks(a.rows, a.dim);
  by_element(a.elem, [&](auto t) {
    using T = decltype(t);
    by_row_length(a.dim, [&](auto lanes, auto nv) {
      by_ends(a.dim, [&](auto ends) {
        if constexpr (ends != TINY || lanes == 16) hipLaunchKernelGGL((layer_norm_grad_kernel<T, lanes, nv, ends>), dim3((unsigned)blocks), dim3(threads_of(lanes)), 0, st, a);
      });
    });
  });
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return launch_column_sum(a.work, blocks, SumOutputs{{a.dweight, a.dbias}, {a.dim, a.dim}}, st);
}

}  // namespace gbx
