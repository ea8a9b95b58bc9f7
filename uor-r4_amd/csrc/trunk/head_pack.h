// head_pack.h - rows laid out for the tiles: those with a target next to each other, 16 bytes aligned.
#pragma once
#include "head.h"

namespace trunk {

// Rows of a block of the packing kernels, and 16-byte pieces of each: few, as small calls wait for each of a block's turns (loss and
// gradients of 52 rows of 512: 73 us, with 32 pieces 78).
constexpr uint32_t kPackRows = 64, kPackPieces = 8;

// The rows of a call, and where those with a target go. Rows without one (a target outside 0 .. vocab - 1)
// take no part: nothing of them is read, whatever it is, and no product is spent on them.
struct Pack {
  uint32_t rows, width, vocab;
  uint32_t piece;         // packed rows of a piece, whose panels lie behind the piece's before
  int64_t stride;
  const void *x, *targets;
  bool wide;              // targets are of 64 bits
  const uint32_t *counts; // rows with a target in each block's share, or NULL: each block counts for itself
  bool summed;            // of the shares before it instead
  char *to;               // [pieces][panels][piece][64 bytes]
  int32_t *order, *target;  // [rows up to 256]: a packed row's own row and target (-1: none)
  uint32_t *count;          // how many rows are packed
  float *losses, *lse;      // a loss: 0 for the rows without a target
  // a gradient's:
  const float *lse_in, *dlosses, *dlse;
  float4 *factors;          // [rows up to 256], see Factors
  void *dx;                 // zeros for the rows without a target, or NULL
  uint8_t *present;         // [vocab up to 16] zeros, or NULL
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

// Of many blocks none adds up all those before it, which would go by their square: one block puts the sums so far in the counts'
// places, each of its threads those of a stretch of them. Of few that is a launch more for nothing. Losses over 100 words in bf16: 65,536
// rows of 64 26 us, each block adding up for itself 24; 131,072 of 64 35 and 35, of 512 83 and 88; 262,144 of 512 157 and 198; 2^20 of
// 256 320 and 540; 2^24 of 64 2,260 and 9,800.
constexpr uint32_t kManyShares = 2048;
static __global__ __launch_bounds__(1024) void head_starts(uint32_t *counts, uint32_t blocks) {
  __shared__ uint32_t sums[16];
  const uint32_t each = (blocks + 4095) / 4096 * 4, first = threadIdx.x * each, end = min(first + each, blocks);  // the array has whole fours
  uint32_t mine = 0;
#pragma unroll 8
  for (uint32_t i = first; i < end; i += 4) {
    const u32x4 v = *(const u32x4 *)(counts + i);
    mine += v[0] + v[1] + v[2] + v[3];
  }
  uint32_t before = mine;
#pragma unroll
  for (uint32_t k = 1; k < 64; k <<= 1) {
    const uint32_t v = __shfl_up(before, k);
    before += (threadIdx.x & 63) >= k ? v : 0;
  }
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = before;
  __syncthreads();
  before -= mine;
  for (uint32_t w = 0; w < threadIdx.x >> 6; w++) before += sums[w];
#pragma unroll 8
  for (uint32_t i = first; i < end; i += 4) {
    const u32x4 v = *(const u32x4 *)(counts + i);
    *(u32x4 *)(counts + i) = u32x4{before, before + v[0], before + v[0] + v[1], before + v[0] + v[1] + v[2]};
    before += v[0] + v[1] + v[2] + v[3];
  }
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

// A gradient's factors of a packed row. In bf16 G = e2 2^(z log2 e - base) for e2 = (dloss + dlse) 2^(what the
// rounding of base = lse log2 e left, with log2 e of 32 bits as the exponents have it); in 32 bits G = e2 e^(z - base) for base = lse. Less dloss at the target.
template <class T>
__device__ __forceinline__ float4 factors_of(float lse, float dloss, float dlse) {
  if constexpr (sizeof(T) == 4) return {lse, dloss + dlse, dloss, 0.0f};
  const double base = (double)lse * (double)kLog2e;
  const float hi = (float)base, all = dloss + dlse;
  const float left = hi - hi == 0.0f ? (float)(hi - base) : 0.0f;
  return {hi, all * fmaf(left, 0.693147181f, 1.0f), dloss, 0.0f};
}

// Where 16 bytes of a packed row lie: the c-th of it.
__device__ __forceinline__ uint64_t packed_at(const Pack &a, uint32_t panels, uint32_t row, uint32_t c) {
  const uint32_t piece = row / a.piece;
  return (((uint64_t)piece * panels + (c >> 2)) * a.piece + (row - piece * a.piece)) * 64 + (c & 3) * 16;
}

template <class T, bool GRAD>
__global__ __launch_bounds__(256) void head_pack(Pack a) {
  __shared__ uint32_t scratch[4], from[kPackRows], none[kPackRows];
  const uint32_t first = blockIdx.x * kPackRows;
  uint32_t before = 0;
  if (a.summed) {
    before = a.counts[blockIdx.x];
  } else {
    if (a.counts) {
      for (uint32_t i = threadIdx.x; i < blockIdx.x; i += 256) before += a.counts[i];
    } else {
      for (uint32_t i = threadIdx.x; i < first; i += 256) before += target_of(a.targets, a.wide, i, a.vocab) >= 0;
    }
    before = block_sum(before, scratch);
  }
  const uint32_t row = first + threadIdx.x;
  // The block's pieces of each row; the first block of a share writes what there is one of a row.
  const uint32_t panels = (a.width + kDeep<T> - 1) / kDeep<T>, piece0 = blockIdx.y * kPackPieces;
  const uint32_t pieces = min(kPackPieces, panels * 4 - piece0);
  const bool leads = blockIdx.y == 0;
  if (threadIdx.x < kPackRows) {
    const int32_t t = row < a.rows ? target_of(a.targets, a.wide, row, a.vocab) : -1;
    const uint64_t which = __ballot(t >= 0), below = ((uint64_t)1 << threadIdx.x) - 1;
    const uint32_t place = __builtin_popcountll(which & below);
    if (threadIdx.x == 0) scratch[0] = __builtin_popcountll(which);
    if (t >= 0) {
      from[place] = row;
      if (leads) {
        a.order[before + place] = (int32_t)row;
        a.target[before + place] = t;
        if constexpr (GRAD)
          a.factors[before + place] = factors_of<T>(a.lse_in[row], a.dlosses ? a.dlosses[row] : 0.0f, a.dlse ? a.dlse[row] : 0.0f);
      }
    } else {
      none[threadIdx.x - place] = row;
      if (leads && row < a.rows) {
        if (a.losses) a.losses[row] = 0.0f;
        if (a.lse) a.lse[row] = 0.0f;
      }
    }
  }
  __syncthreads();
  const uint32_t n = scratch[0];
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n * pieces; i += 256) {
    const uint32_t r = i / pieces, c = piece0 + i % pieces;
    const auto v = load_some<T, kVec<T>>((const T *)a.x + (int64_t)from[r] * a.stride, true, c * kVec<T>, a.width);
    *(Part<T> *)(a.to + packed_at(a, panels, before + r, c)) = v;
  }
  if constexpr (GRAD) {
    if (a.present) {
      const uint64_t blocks = (uint64_t)gridDim.x * gridDim.y, block = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
      for (uint64_t i = block * 256 + threadIdx.x; i < (a.vocab + 15) / 16; i += blocks * 256) *(u32x4 *)(a.present + i * 16) = u32x4{};
    }
    // The share's rows without a target.
    if (a.dx)
      for (uint32_t i = threadIdx.x; i < (kPackRows - n) * pieces; i += 256) {
        const uint32_t r = none[i / pieces], col = (piece0 + i % pieces) * kVec<T>;
        if (r < a.rows && col < a.width) store_some<T, kVec<T>>((T *)a.dx + (uint64_t)r * a.width, col, a.width, Part<T>{});
      }
  }
  if (blockIdx.x + 1 < gridDim.x) return;
  // The last block: how many rows there are, and rows of nothing up to a tile's end.
  const uint32_t all = before + n, end = (all + kRound - 1) / kRound * kRound;
  if (leads) {
    if (threadIdx.x == 0) *a.count = all;
    for (uint32_t i = all + threadIdx.x; i < end; i += 256) {
      a.order[i] = -1, a.target[i] = -1;
      if constexpr (GRAD) a.factors[i] = {0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  for (uint32_t i = threadIdx.x; i < (end - all) * pieces; i += 256)
    *(Part<T> *)(a.to + packed_at(a, panels, all + i / pieces, piece0 + i % pieces)) = Part<T>{};
}

// A matrix by panels, zeros past its width.
template <class T>
__global__ __launch_bounds__(256) void head_lay(const T *from, int64_t stride, uint32_t rows, uint32_t width, uint32_t panels, uint32_t all, char *to) {
  // A block takes 16 rows of four panels: 256 bytes of each are read, and 1 KB of each panel is written.
  const uint32_t quads = (panels + 3) / 4;
  for (uint64_t i = blockIdx.x; i < (uint64_t)((rows + 15) / 16) * quads; i += gridDim.x) {
    const uint32_t row = (uint32_t)(i / quads) * 16 + threadIdx.x / 16, c = (uint32_t)(i % quads) * 16 + threadIdx.x % 16;
    if (row < rows && c < panels * 4)
      *(Part<T> *)(to + ((uint64_t)(c >> 2) * all + row) * 64 + (c & 3) * 16) = load_some<T, kVec<T>>(from + (int64_t)row * stride, true, c * kVec<T>, width);
  }
}

// Packs a call's rows; `counts` is scratch memory for a number a block.
template <class T, bool GRAD>
inline void pack(Pack k, uint32_t *counts, hipStream_t stream) {
  const uint32_t blocks = (k.rows + kPackRows - 1) / kPackRows, panels = (k.width + kDeep<T> - 1) / kDeep<T>;
  if (k.rows > 4096) {  // else each block counts the rows before its own by itself
    hipLaunchKernelGGL(head_count, dim3(blocks), dim3(64), 0, stream, k.targets, k.wide, k.rows, k.vocab, counts);
    k.counts = counts;
    if (blocks >= kManyShares) {
      hipLaunchKernelGGL(head_starts, dim3(1), dim3(1024), 0, stream, counts, blocks);
      k.summed = true;
    }
  }
  hipLaunchKernelGGL((head_pack<T, GRAD>), dim3(blocks, (panels * 4 + kPackPieces - 1) / kPackPieces), dim3(256), 0, stream, k);
}
template <class T>
inline Matrix lay(const void *from, int64_t stride, uint32_t rows, uint32_t width, char *to, hipStream_t stream) {
  const uint32_t panels = (width + kDeep<T> - 1) / kDeep<T>;
  const uint64_t blocks = (uint64_t)((rows + 15) / 16) * ((panels + 3) / 4);
  hipLaunchKernelGGL((head_lay<T>), dim3((uint32_t)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream, (const T *)from, stride, rows, width,
                     panels, rows, to);
  return {to, (int64_t)rows * 64};
}

}  // namespace trunk
