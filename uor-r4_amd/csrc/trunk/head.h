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
// the largest one's share is 1 exactly and the loss of a sure row is right to its own size. In base 2 that share is what the
// rounding of `most` left, which the loss takes back, as it divides by the same log2 e: of 32 bits, 1.3e-8 of itself off. The
// true one's inverse left 1.3e-8 of the logit: losses of sure rows were -4e-5 at a logit of 3,000.
struct Sum {
  float most, sum, value;
  uint32_t place;
};

__host__ __device__ constexpr uint64_t up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Which piece of `n` a block takes: those of one XCD (every eighth block) are next to each other, as they
// share what they read through its L2.
__device__ __forceinline__ uint32_t by_xcd(uint32_t block, uint32_t n) {
  const uint32_t xcd = block & 7, each = n >> 3, more = n & 7;
  return xcd * each + (xcd < more ? xcd : more) + (block >> 3);
}

// a / b, by 32 bits where they are, as they nearly always are: divisions of 64 are some hundred instructions.
__device__ __forceinline__ uint64_t ratio(uint64_t a, uint64_t b) { return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b; }
// Row tiles by word tiles, in even shares for groups of blocks: a group takes up to eight row tiles abreast through its share of
// the words, so that what runs at once reads few rows and few words. A unit is a word tile of a set of row tiles. Where the card takes
// all tiles at once, a block takes one, and all row tiles are abreast.
// `blocks`: how many there may be, eighths of them an XCD; `at_once`: how many the card takes.
struct RowShares {
  uint64_t units;
  uint32_t groups, tiles, sets, abreast;
  bool single, resident;  // a block has one tile; all blocks run at once
  __device__ __forceinline__ RowShares(uint32_t rows, uint32_t tile, uint32_t word_tiles, uint32_t blocks, uint32_t at_once) {
    tiles = (rows + tile - 1) / tile;
    single = (uint64_t)tiles * word_tiles <= at_once, resident = blocks <= at_once;
    sets = single ? 1 : (tiles + 7) / 8, abreast = single ? tiles : (tiles + sets - 1) / sets;
    units = (uint64_t)sets * word_tiles;
    groups = single ? word_tiles : (uint32_t)min((uint64_t)(8 * (blocks / 8 / abreast)), units);
  }
  __device__ __forceinline__ uint64_t first(uint32_t group) const { return ratio(units * group, groups); }
  __device__ __forceinline__ uint32_t of(uint64_t unit) const { return (uint32_t)ratio((unit + 1) * groups - 1, units); }
};
// Blocks for them: as many as the card takes at once (two a compute unit of large tiles, four of small ones), and up to four
// times as many of 16 tiles or more, as compute units are not equally fast: 32,768 rows of 256 over 32,768 words 600 us, in 512
// blocks 619; but 1,024 rows in 512 blocks 30, in all of the 1,024 that there is work for 37.
inline uint32_t scan_blocks(uint32_t row_tiles, uint32_t word_tiles, uint32_t at_once) {
  const uint64_t even = row_tiles * (uint64_t)word_tiles / 16 / 8 * 8;
  return (uint32_t)(even < at_once ? at_once : even < 4 * at_once ? even : 4 * at_once);
}
inline uint32_t scan_grid(uint32_t row_tiles, uint32_t word_tiles, uint32_t at_once) {
  const uint64_t all = row_tiles * (uint64_t)word_tiles;
  return all < at_once ? (uint32_t)all : scan_blocks(row_tiles, word_tiles, at_once);
}
// A block's: `tiles` word tiles of row tiles, from the word tile `word` of the row tile `row` on. With the last word tile of
// a row tile it goes on with the row tile `abreast` further.
struct Walk {
  uint32_t group, tiles, row, word, abreast, word_tiles;
  __device__ __forceinline__ Walk(const RowShares &s, uint32_t words, uint32_t block) {
    tiles = 0, abreast = s.abreast, word_tiles = words;
    if (s.single) {
      // Eight row tiles by all words, before the next eight.
      const uint32_t all = s.tiles * words;
      if (block >= all) return;
      const uint32_t work = by_xcd(block, all), set = work / (8 * words), left = work - set * 8 * words, rows = min(8u, s.tiles - 8 * set);
      group = word = left / rows, row = 8 * set + left % rows, tiles = 1;
      return;
    }
    // An XCD (every eighth block) has groups next to each other.
    const uint32_t xcd = block & 7, j = block >> 3, own = s.groups / 8 + (xcd < s.groups % 8), all = own * abreast;
    if (j >= all) return;
    // Of blocks that run at once, every 32nd of an XCD's shares a compute unit (measured). Its blocks take groups next to
    // each other, whose shares are even together where each is a tile more or less.
    const uint32_t unit = j & 31, q = unit * (all >> 5) + min(unit, all & 31) + (j >> 5);
    const uint32_t first = s.resident ? q / own : j % abreast;
    group = xcd * (s.groups / 8) + min(xcd, s.groups % 8) + (s.resident ? q % own : j / abreast);
    const uint64_t from = s.first(group);
    uint64_t to = s.first(group + 1);
    if ((s.sets - 1) * s.abreast + first >= s.tiles) to = min(to, (uint64_t)(s.sets - 1) * words);  // the last set has fewer
    if (from >= to) return;
    const uint32_t set = (uint32_t)ratio(from, words);
    tiles = (uint32_t)(to - from), row = set * s.abreast + first, word = (uint32_t)(from - (uint64_t)set * words);
  }
  // One tile on; whether it is another row tile.
  __device__ __forceinline__ bool next() {
    if (++word < word_tiles) return false;
    word = 0, row += abreast;
    return true;
  }
};

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
// by many row tiles. 8,192 rows at width 1,024 and 131,072 words: 1,920 us, as it lies 2,010; loss and gradients 8,475
// and 8,550.
constexpr uint32_t kLayRows = 1024;
inline bool laid_out(const uor_trunk_head_args *s) { return s->rows >= kLayRows || !as_it_lies(s->weight, s->w_stride, s->vocab, s->width, s->dtype); }
// A call's tiles. Small ones where large ones would leave some compute units idle (333 rows over 4,099 words of 100 in 32 bits: 18 us, 26
// in large tiles; 501 over 5,003 of 200 and their gradients 103 and 143), and in 32 bits, where there are no registers for two sets of
// sums of large ones. Tiny ones where small ones would leave half of the units idle (loss and gradients of 500 rows of 512 over 1,500
// words in 32 bits 87 us, in small tiles 95; but of 333 of 100 over 4,099 59 and 56).
struct Tiling {
  uint32_t m, n, at_once;  // at_once: that the card takes
};
template <class S>
constexpr Tiling kTiling = {S::kM, S::kN, 256 * S::kBlocks};
template <class S>
inline bool fewer_than(const uor_trunk_head_args *s, uint64_t tiles) {
  return up(s->rows, S::kN) / S::kN * (up(s->vocab, S::kM) / S::kM) < tiles;
}
// f of the call's shape of tiles, as an object of it; and what they are.
template <class T, class F>
inline void with_tiles(const uor_trunk_head_args *s, F f) {
  if (fewer_than<Small>(s, 128)) f(Tiny{});
  else if constexpr (sizeof(T) == 4) f(Small{});
  else if (fewer_than<Large>(s, 256)) f(Small{});
  else f(Large{});
}
inline Tiling tiling(const uor_trunk_head_args *s) {
  Tiling t;
  const auto set = [&](auto shape) { t = kTiling<decltype(shape)>; };
  if (s->dtype == UOR_TRUNK_F32) with_tiles<float>(s, set);
  else with_tiles<bf16>(s, set);
  return t;
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
