// head.h - what the head's kernels share: a call's arguments and where its scratch memory lies.
#pragma once
#include "tiles.h"

namespace trunk {

// A call's matrices as the kernels read them: rows 16 bytes aligned, whole numbers of 16 bytes wide.
struct Matrix {
  const char *at;
  int64_t pitch;  // bytes from row to row, or from panel to panel
};
// What is known of a row's softmax: its largest logit, the sum of e^(logit - largest), and the target's logit,
// or the largest one's value and place. The largest one is in base 2 (times log2 e, rounded) where exponents are formed in
// one instruction, fma(z, log2 e, -most); otherwise, in 32 bits and for few rows, the logits are subtracted first, so that
// the largest one's share is 1 exactly and the loss of a sure row is right to its own size.
struct Sum {
  float most, sum, value;
  uint32_t place;
};

constexpr double kLn2 = 0.6931471805599453;

__host__ __device__ constexpr uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Which piece of `n` a block takes: those of one XCD (every eighth block) are next to each other, as they
// share what they read through its L2.
__device__ __forceinline__ uint32_t by_xcd(uint32_t block, uint32_t n) {
  const uint32_t xcd = block & 7, each = n >> 3, more = n & 7;
  return xcd * each + (xcd < more ? xcd : more) + (block >> 3);
}

// A block's row tile and share of the words. Blocks of an XCD go through eight row tiles by all shares before
// the next eight, so that what runs at once reads few rows and few words.
__device__ __forceinline__ void by_eights(uint32_t work, uint32_t row_tiles, uint32_t splits, uint32_t &row_tile, uint32_t &split) {
  const uint32_t group = work / (8 * splits), left = work - group * 8 * splits, rows = min(8u, row_tiles - group * 8);
  row_tile = group * 8 + left % rows;
  split = left / rows;
}

// Scratch memory, a stretch at a time.
struct Scratch {
  uint64_t bytes = 0;
  uint64_t take(uint64_t n) {
    const uint64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};

inline uint32_t size_of(uint32_t dtype) { return dtype == UOR_TRUNK_BF16 ? 2 : 4; }
// Whether the kernels can read a matrix as it lies.
inline bool as_it_lies(const void *p, int64_t stride, uint32_t rows, uint32_t width, uint32_t dtype) {
  const uint32_t size = size_of(dtype);
  return (uint64_t)width * size % 16 == 0 && ((uintptr_t)p & 15) == 0 &&
         (rows <= 1 || (stride * size % 16 == 0 && stride * (int64_t)size < (1 << 23)));
}
// From how many rows on a matrix is laid out by panels, whose rows could be read as they lie: it is then read
// by many row tiles. 8,192 rows at width 1,024 and 131,072 words: 2,103 us, as it lies 2,152; loss and gradients 9,489
// and 9,579.
constexpr uint32_t kLayRows = 1024;
inline bool laid_out(const uor_trunk_head_args *s) { return s->rows >= kLayRows || !as_it_lies(s->weight, s->w_stride, s->vocab, s->width, s->dtype); }
// Whether small tiles are taken: in 32 bits, where there are registers for two sets of sums of them, and where the large
// ones would leave some compute units idle (333 rows over 4,099 words of 100 in 32 bits: 18 us, 26 in large tiles; 501 over
// 5,003 of 200 and their gradients 103 and 143).
inline bool small_tiles(const uor_trunk_head_args *s) {
  return s->dtype == UOR_TRUNK_F32 || up(s->rows, Large::kN) / Large::kN * (up(s->vocab, Large::kM) / Large::kM) < 256;
}
inline int check_head(const uor_trunk_head_args *s) {
  if (!s) return fail(-1, "null argument");
  if (s->dtype > UOR_TRUNK_F32) return fail(-1, "dtype %u is neither bf16 nor f32", s->dtype);
  if (s->width < 1 || s->width > UOR_TRUNK_MAX_WIDTH) return fail(-1, "width %u outside 1..8192", s->width);
  if (s->vocab < 1 || s->vocab > UOR_TRUNK_MAX_VOCAB) return fail(-1, "a vocabulary of %u outside 1..%u", s->vocab, UOR_TRUNK_MAX_VOCAB);
  if (s->rows > UOR_TRUNK_MAX_ROWS) return fail(-1, "%u rows are more than %u", s->rows, UOR_TRUNK_MAX_ROWS);
  if (s->rows > 1 && s->x_stride < s->width) return fail(-1, "rows overlap: a stride is less than a row");
  if (s->vocab > 1 && s->w_stride < s->width) return fail(-1, "the matrix's rows overlap: a stride is less than a row");
  if (!s->weight || (s->rows && !s->x)) return fail(-1, "null x or weight");
  return 0;
}

}  // namespace trunk
