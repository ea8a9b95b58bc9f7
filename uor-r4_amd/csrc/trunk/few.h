// few.h - logits of few rows, for which tiles of many are too large.
#pragma once
#include "head_pack.h"

namespace trunk {

// Few rows: bound by the matrix, which is read once, past LDS. A block takes 16 words at a time, its four wavefronts a
// quarter of their values each (every fourth 64 bytes), so that a narrow vocabulary's long rows are not one
// wavefront's chain; the rows of x lie in LDS. The quarters meet in LDS, and a thread then has the logit of one
// word for one row of each tile of 16 rows.
struct Few {
  const void *w, *x;
  int64_t w_stride, x_stride;   // values
  uint32_t rows, vocab, width, pitch;  // pitch: bytes of a row of x in LDS
  uint32_t word0, words;        // the words that are looked at
  const void *targets;
  bool wide;
  Sum *parts;                   // [blocks][rows]
};
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

constexpr uint32_t kFewPad = 17;  // floats between words of a quarter's sums

// take(j, word, z) gets each word's logit of row 16 j + threadIdx % 16, of `rows` rows; words past the last are numbers too,
// of the last word. `order`: where the rows lie, or NULL.
template <class T, int TILES, class F>
__device__ __forceinline__ void few_logits(const Few &a, uint32_t rows, const int32_t *order, F take) {
  extern __shared__ char x[];
  __shared__ float quarters[2][4][TILES][16 * kFewPad];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t pieces = (a.width + kDeep<T> - 1) / kDeep<T> * 4;
  for (uint32_t i = threadIdx.x; i < rows * pieces; i += 256) {
    const uint32_t row = order ? (uint32_t)order[i / pieces] : i / pieces;
    *(Part<T> *)(x + i / pieces * a.pitch + i % pieces * 16) =
        load_some<T, kVec<T>>((const T *)a.x + (int64_t)row * a.x_stride, true, i % pieces * kVec<T>, a.width);
  }
  __syncthreads();
  const uint32_t i16 = lane & 15, chunk = lane >> 4, full = a.width / kDeep<T>;  // stretches of 64 bytes that a row has whole
  const char *xs[TILES];
#pragma unroll
  for (int j = 0; j < TILES; j++) xs[j] = x + (16 * j + i16 < rows ? 16 * j + i16 : 0) * a.pitch + chunk * 16;
  uint32_t buffer = 0;
  for (uint32_t g = blockIdx.x; g * 16 < a.words; g += gridDim.x, buffer ^= 1) {
    const uint32_t mine = a.word0 + g * 16 + i16 < a.vocab ? a.word0 + g * 16 + i16 : a.vocab - 1;
    const T *row = (const T *)a.w + (int64_t)mine * a.w_stride;
    f32x4 sums[TILES] = {};
    auto add = [&](Part<T> w, uint32_t s) {
#pragma unroll
      for (int j = 0; j < TILES; j++) sums[j] = mma16(w, *(const Part<T> *)(xs[j] + s * 64), sums[j]);
    };
    // Eight stretches on their way while the eight before are multiplied.
    constexpr uint32_t kAhead = 8;
    Part<T> now[kAhead], next[kAhead];
    auto look = [&](Part<T> (&to)[kAhead], uint32_t s) {
#pragma unroll
      for (uint32_t k = 0; k < kAhead; k++) {
        const uint32_t at = s + 4 * k < full ? s + 4 * k : wave < full ? wave : 0;  // one too many is read again
        to[k] = loose<T, kVec<T>>(row + (full ? at * kDeep<T> + chunk * kVec<T> : 0));
      }
    };
    if (full) {
      look(now, wave);
      for (uint32_t s = wave; s < full; s += 4 * kAhead) {
        if (s + 4 * kAhead < full) look(next, s + 4 * kAhead);
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++)
          if (s + 4 * k < full) add(now[k], s + 4 * k);
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) now[k] = next[k];
      }
    }
    if (full * kDeep<T> < a.width && wave == (full & 3))
      add(load_some<T, kVec<T>>(row, true, full * kDeep<T> + chunk * kVec<T>, a.width), full);
#pragma unroll
    for (int j = 0; j < TILES; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) quarters[buffer][wave][j][(4 * chunk + r) * kFewPad + i16] = sums[j][r];
    __syncthreads();
    const uint32_t at = threadIdx.x / 16 * kFewPad + threadIdx.x % 16, word = a.word0 + g * 16 + threadIdx.x / 16;
#pragma unroll
    for (int j = 0; j < TILES; j++)
      take(j, word, (quarters[buffer][0][j][at] + quarters[buffer][1][j][at]) + (quarters[buffer][2][j][at] + quarters[buffer][3][j][at]));
  }
}

// Bytes of a row of x in LDS: 16 more than its stretches, so that 16 rows' pieces lie in different banks.
inline uint32_t few_pitch(const uor_trunk_head_args *s) { return (uint32_t)up(s->width * size_of(s->dtype), 64) + 16; }
// Whether a call's rows are few. In 32 bits they are up to 64 that fit into LDS: tiles of 64 rows spend their matrix
// instructions on rows that are none (1 row over 131,072 words of 512: 57 us, in tiles 135); the gradients' logits are
// then formed the same way, bit for bit, as small gradients are differences of their exponentials and the loss's. In bf16
// tiles read the matrix as fast (16 rows over 131,072 words of 512: 35 us, 39 here), unless they leave compute units idle (over
// 4,550 of 1,536: 18 and 15) or have to lay it out first (over 5,000 of 100: 20 and 14).
inline bool few_rows(const uor_trunk_head_args *s) {
  if (s->rows > 64 || s->rows * few_pitch(s) > 122880) return false;
  return s->dtype == UOR_TRUNK_F32 || s->vocab <= 16384 || !as_it_lies(s->weight, s->w_stride, s->vocab, s->width, s->dtype);
}

}  // namespace trunk
