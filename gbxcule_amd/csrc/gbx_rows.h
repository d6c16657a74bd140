// gbx_rows.h -- rows held in registers: how the norms' lanes share a row, where
// rows end, sums over a row's lanes.
#pragma once
#include <algorithm>

#include "gbx_policy.h"

namespace gbx {
namespace {

constexpr int kVec = 8;  // channels a lane takes at a time: 16 bytes of a 16-bit type
constexpr int threads_of(int lanes) { return lanes > 256 ? lanes : 256; }

// Where rows end.  WHOLE: with a piece of 8 channels.  LAPPED: inside one; the
// last piece then begins 8 channels before the end and shares some with the
// piece before it.  Both compute and write the same values there, and sums
// leave the shared ones out: without it the one lane with a part of a piece
// would load and store it element by element (131,072 rows of 255 channels
// forward and backward 565 us).  TINY: rows shorter than a piece.
enum Ends { WHOLE, LAPPED, TINY };
struct Piece {
  int c, valid, skip;  // first channel; channels from there on (8 or more: a whole piece); shared ones
};
template <int ENDS>
__device__ __forceinline__ Piece piece_of(int k, int dim) {
  const int c = k * kVec;
  if constexpr (ENDS == LAPPED) {
    if (c < dim) return {c < dim - kVec ? c : dim - kVec, kVec, c < dim - kVec ? 0 : c - (dim - kVec)};
  }
  return {c, ENDS == TINY ? dim - c : c < dim ? kVec : 0, 0};
}

// Sum over LANES neighbouring lanes; more than 64 are the whole workgroup.
template <int LANES>
__device__ __forceinline__ float sum_over(float v, float* lds) {
#pragma unroll
  for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) v += __shfl_xor(v, m, 64);
  if constexpr (LANES > 64) {
    __syncthreads();  // the last use of lds has been read
    if ((threadIdx.x & 63u) == 0u) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) v += lds[w];
  }
  return v;
}

// f(lanes of a row, 8-channel pieces of a lane): the fewest lanes that hold it,
// one wavefront for as long as two pieces a lane do (its sums need no LDS).
template <typename F>
void by_row_length(int dim, F&& f) {
  auto go = [&](auto lanes, auto pieces) { f(lanes, pieces); };
  using std::integral_constant;
  if (dim <= 128) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (dim <= 256) go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (dim <= 512) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (dim <= 1024) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (dim <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (dim <= 4096) go(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  else if (dim <= 8192) go(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
  else go(integral_constant<int, 256>{}, integral_constant<int, 0>{});
}
int rows_of_block(int dim) {
  int rows = 0;
  by_row_length(dim, [&](auto lanes, auto) { rows = threads_of(lanes) / lanes; });
  return rows;
}
template <typename F>
void by_ends(int dim, F&& f) {
  if (dim % kVec == 0) f(std::integral_constant<int, WHOLE>{});
  else if (dim > kVec) f(std::integral_constant<int, LAPPED>{});
  else f(std::integral_constant<int, TINY>{});
}
constexpr int kGradBlocks = 1024;  // workgroups of the gradient, each a row of partial sums
int grad_blocks(int64_t rows, int dim) {
  const int per = rows_of_block(dim);
  return (int)std::min<int64_t>((rows + per - 1) / per, kGradBlocks);
}

}  // namespace
}  // namespace gbx
