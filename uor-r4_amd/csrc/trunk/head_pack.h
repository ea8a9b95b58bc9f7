// head_pack.h - rows laid out for the tiles: those with a target next to each other, 16 bytes aligned.
#pragma once
#include "head.h"

namespace trunk {

constexpr uint32_t kPackRows = 64;  // rows of a block of the packing kernels

// The rows of a call, and where those with a target go. Rows without one (a target outside 0 .. vocab - 1)
// take no part: nothing of them is read, whatever it is, and no product is spent on them.
struct Pack {
  uint32_t rows, width, vocab, pitch;  // pitch: values of a packed row, the width up to whole 16 bytes
  int64_t stride;
  const void *x, *targets;
  bool wide;              // targets are of 64 bits
  const uint32_t *counts; // rows with a target in each block's share, or NULL: each block counts for itself
  void *to;               // [rows up to 256][pitch]
  int32_t *order, *target;  // [rows up to 256]: a packed row's own row and target (-1: none)
  uint32_t *count;          // how many rows are packed
  float *losses, *lse;      // a loss: 0 for the rows without a target
  // a gradient's:
  const float *lse_in, *dlosses, *dlse;
  float4 *factors;          // [rows up to 256], see Factors
  void *dx;                 // zeros for the rows without a target
  uint32_t dx_width;
};

__device__ __forceinline__ int32_t target_of(const void *targets, bool wide, uint32_t row, uint32_t vocab) {
  const int64_t t = wide ? ((const int64_t *)targets)[row] : ((const int32_t *)targets)[row];
  return t >= 0 && t < (int64_t)vocab ? (int32_t)t : -1;
}

// One wavefront of sums a block: how many rows of its share have a target.
static __global__ __launch_bounds__(64) void head_count(const void *targets, bool wide, uint32_t rows, uint32_t vocab, uint32_t *counts) {
  const uint32_t row = blockIdx.x * kPackRows + threadIdx.x;
  const bool there = row < rows && target_of(targets, wide, row, vocab) >= 0;
  const uint64_t which = __ballot(there);
  if (threadIdx.x == 0) counts[blockIdx.x] = __builtin_popcountll(which);
}

// The sum over a block of 256 threads, to all of them.
__device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t *scratch) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = scratch[0] + scratch[1] + scratch[2] + scratch[3];
  __syncthreads();
  return v;
}

// A gradient's factors of a packed row: G = e2 2^(z log2 e - base) for e2 = (dloss + dlse) 2^(what the
// rounding of base = lse log2 e left), less dloss at the target.
__device__ __forceinline__ float4 factors_of(float lse, float dloss, float dlse) {
  const double base = (double)lse * 1.4426950408889634;
  const float hi = (float)base, all = dloss + dlse;
  const float left = hi - hi == 0.0f ? (float)(hi - base) : 0.0f;
  return {hi, all * fmaf(left, 0.693147181f, 1.0f), dloss, 0.0f};
}

template <class T, bool GRAD>
__global__ __launch_bounds__(256) void head_pack(Pack a) {
  __shared__ uint32_t scratch[4], from[kPackRows];
  const uint32_t first = blockIdx.x * kPackRows;
  uint32_t before = 0;
  if (a.counts) {
    for (uint32_t i = threadIdx.x; i < blockIdx.x; i += 256) before += a.counts[i];
  } else {
    for (uint32_t i = threadIdx.x; i < first; i += 256) before += target_of(a.targets, a.wide, i, a.vocab) >= 0;
  }
  before = block_sum(before, scratch);
  const uint32_t row = first + threadIdx.x;
  bool none = false;
  if (threadIdx.x < kPackRows) {
    const int32_t t = row < a.rows ? target_of(a.targets, a.wide, row, a.vocab) : -1;
    const uint64_t which = __ballot(t >= 0);
    if (threadIdx.x == 0) scratch[0] = __builtin_popcountll(which);
    none = row < a.rows && t < 0;
    if (t >= 0) {
      const uint32_t place = __builtin_popcountll(which & (((uint64_t)1 << threadIdx.x) - 1));
      from[place] = row;
      a.order[before + place] = (int32_t)row;
      a.target[before + place] = t;
      if constexpr (GRAD)
        a.factors[before + place] = factors_of(a.lse_in[row], a.dlosses ? a.dlosses[row] : 0.0f, a.dlse ? a.dlse[row] : 0.0f);
    } else if (row < a.rows) {
      if (a.losses) a.losses[row] = 0.0f;
      if (a.lse) a.lse[row] = 0.0f;
    }
  }
  __syncthreads();
  const uint32_t n = scratch[0], pieces = a.pitch / kVec<T>;
  for (uint32_t i = threadIdx.x; i < n * pieces; i += 256) {
    const uint32_t r = i / pieces, col = i % pieces * kVec<T>;
    const auto v = load_some<T, kVec<T>>((const T *)a.x + (int64_t)from[r] * a.stride, true, col, a.width);
    *(Part<T> *)((T *)a.to + (uint64_t)(before + r) * a.pitch + col) = v;
  }
  if constexpr (GRAD) {  // the share's rows without a target
    for (uint32_t k = 0; k < kPackRows; k++) {
      const uint32_t other = first + k;
      if (other < a.rows && target_of(a.targets, a.wide, other, a.vocab) < 0)
        for (uint32_t c = threadIdx.x; c < a.dx_width; c += 256) ((T *)a.dx)[(uint64_t)other * a.dx_width + c] = (T)0.0f;
    }
  }
  (void)none;
  if (blockIdx.x + 1 < gridDim.x) return;
  // The last block: how many rows there are, and rows of nothing up to a tile's end.
  const uint32_t all = before + n, end = (all + kTileM - 1) / kTileM * kTileM;
  if (threadIdx.x == 0) *a.count = all;
  for (uint32_t i = all + threadIdx.x; i < end; i += 256) {
    a.order[i] = -1, a.target[i] = -1;
    if constexpr (GRAD) a.factors[i] = {0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (uint64_t i = threadIdx.x; i < (uint64_t)(end - all) * pieces; i += 256)
    *(Part<T> *)((T *)a.to + (uint64_t)(all + i / pieces) * a.pitch + i % pieces * kVec<T>) = Part<T>{};
}

// A matrix's rows as the tiles read them: `pitch` values, zeros past the width.
template <class T>
__global__ __launch_bounds__(256) void head_lay(const T *from, int64_t stride, uint32_t rows, uint32_t width, uint32_t pitch, T *to) {
  const uint32_t pieces = pitch / kVec<T>;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < (uint64_t)rows * pieces; i += gridDim.x * 256ull) {
    const uint32_t col = (uint32_t)(i % pieces) * kVec<T>;
    const uint64_t row = i / pieces;
    *(Part<T> *)(to + row * pitch + col) = load_some<T, kVec<T>>(from + (int64_t)row * stride, true, col, width);
  }
}

}  // namespace trunk
