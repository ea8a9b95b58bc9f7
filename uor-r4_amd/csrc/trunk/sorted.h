// sorted.h - sums of rows by a number that each has, a word of the vocabulary: what the embedding's gradient and
// the targets' terms of the head's share.
//
// The rows' numbers are sorted by their words, rows of a word staying in their order: up to 4,096 by counting,
// more by digits of the word in two or three passes. Then pieces of the sorted rows are summed, each by the lanes
// that hold a row of the result; a word whose rows go over a piece's end leaves its parts to a second launch, which
// adds them up in their order. So a word that a large share of all rows has is summed by many. Other blocks of the
// first launch write zeros to the rows of words that do not occur. No sum depends on the order in which blocks run.
#pragma once
#include "trunk.h"

#include <type_traits>

namespace trunk {

// A row's word, or `vocab` for none.
__device__ __forceinline__ uint32_t token_of(const void *tokens, bool wide, uint64_t row, uint32_t vocab) {
  const int64_t t = wide ? ((const int64_t *)tokens)[row] : ((const int32_t *)tokens)[row];
  return t >= 0 && t < (int64_t)vocab ? (uint32_t)t : vocab;
}

// result[word - word0] = scale sum of weight_t rows_t over the rows t of that word, of `words` words from word0 on.
struct Sums {
  uint32_t rows, width, word0, words;
  float scale;
  int64_t stride, pitch;        // values from row to row of the rows, of the result
  const void *from;
  const float *weights;         // [rows], or NULL: 1
  void *to;
  const uint32_t *keys, *order; // [rows] sorted: words (the vocabulary's size: none), and their rows
  uint32_t length, groups;      // rows of a piece, pieces
  float *parts;                 // [groups][2][width]: a piece's first word's sum and its last one's
  uint32_t sum_blocks;          // of the first launch, the others write zeros
  uint8_t *present;             // [words] or NULL: set to 1 for words that occur, and no zeros are written for others
};

// ---------------------------------------------------------------------------------------------
// The sort.

// Up to kFew rows are sorted by counting: a row's place is how many words before its own there are. That reads
// every word for every row, but in one launch, all from LDS. 7,431 rows take 27 us; by digits, two launches each,
// one takes 16.
constexpr uint32_t kFew = 4096, kSortBlocks = 256, kMostBins = 1024, kSortThreads = 1024, kSortWaves = kSortThreads / 64;

// 64 rows a block, each of its eight wavefronts an eighth of all words; `all` is the rows up to whole 32.
static __global__ __launch_bounds__(512) void sort_few(const void *tokens, bool wide, uint32_t rows, uint32_t vocab, uint32_t all, uint32_t *keys,
                                                       uint32_t *order) {
  extern __shared__ uint32_t words[];
  __shared__ uint32_t counts[8][64];
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < all; i += 512) words[i] = i < rows ? token_of(tokens, wide, i, vocab) : ~0u;
  __syncthreads();
  const uint32_t lane = threadIdx.x & 63, part = threadIdx.x >> 6, row = blockIdx.x * 64 + lane, key = row < rows ? words[row] : 0;
  const uint32_t each = all / 8, first = part * each;
  // Rows before this one count with its own word too, rows behind it do not.
  uint32_t n = 0;
  using Four = __attribute__((ext_vector_type(4))) uint32_t;
  if (first + each <= blockIdx.x * 64) {
#pragma unroll 4
    for (uint32_t i = first; i < first + each; i += 4) {
      const Four w = *(const Four *)(words + i);
#pragma unroll
      for (int e = 0; e < 4; e++) n += w[e] <= key;
    }
  } else if (first >= blockIdx.x * 64 + 64) {
#pragma unroll 4
    for (uint32_t i = first; i < first + each; i += 4) {
      const Four w = *(const Four *)(words + i);
#pragma unroll
      for (int e = 0; e < 4; e++) n += w[e] < key;
    }
  } else {
    for (uint32_t i = first; i < first + each; i++) n += words[i] < key + (i < row);
  }
  counts[part][lane] = n;
  __syncthreads();
  if (part || row >= rows) return;
  for (int k = 1; k < 8; k++) n += counts[k][lane];
  keys[n] = key, order[n] = row;
}

// A pass over one digit of the words. A block has `share` rows next to each other, each of its
// wavefronts an even part of them.
struct Digit {
  uint32_t rows, vocab, share, shift, bins;
  bool wide;
  const void *tokens;                // the first pass's, else NULL
  const uint32_t *keys, *order;      // the pass before's
  uint32_t *counts;                  // [blocks][bins]
  uint32_t *keys_out, *order_out;
  __device__ __forceinline__ uint32_t key(uint64_t i) const { return tokens ? token_of(tokens, wide, i, vocab) : keys[i]; }
};
__device__ __forceinline__ void count_digits(const Digit &a, uint32_t *bins, uint64_t first, uint64_t end) {
#pragma unroll 4
  for (uint64_t i = first + (threadIdx.x & 63); i < end; i += 64) atomicAdd(&bins[(a.key(i) >> a.shift) & (a.bins - 1)], 1u);
}
__device__ __forceinline__ void share_of(const Digit &a, uint64_t &first, uint64_t &end) {
  const uint32_t part = a.share / kSortWaves;
  first = (uint64_t)blockIdx.x * a.share + (threadIdx.x >> 6) * part;
  end = first + part < a.rows ? first + part : a.rows;
}
static __global__ __launch_bounds__(kSortThreads) void sort_count(Digit a) {
  __shared__ uint32_t bins[kMostBins];
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) bins[b] = 0;
  __syncthreads();
  uint64_t first, end;
  share_of(a, first, end);
  count_digits(a, bins, first, end);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) a.counts[(uint64_t)blockIdx.x * a.bins + b] = bins[b];
}
// A row goes behind all rows of lower digits, those of its digit in blocks before, in wavefronts
// before and in its own wavefront before it.
static __global__ __launch_bounds__(kSortThreads) void sort_place(Digit a) {
  __shared__ uint32_t at[kSortWaves][kMostBins], before[kMostBins], all[kMostBins], sums[kSortWaves];
  for (uint32_t b = threadIdx.x; b < kSortWaves * a.bins; b += kSortThreads) at[b / a.bins][b % a.bins] = 0;
  for (uint32_t b = threadIdx.x; b < a.bins; b += kSortThreads) before[b] = all[b] = 0;
  __syncthreads();
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint64_t first, end;
  share_of(a, first, end);
  count_digits(a, at[wave], first, end);
  // A digit's rows in blocks before and in all: a thread takes a digit and an even part of the blocks. The sums of
  // whole numbers do not depend on their order.
  {
    const uint32_t parts = kSortThreads / a.bins, b = threadIdx.x % a.bins, part = threadIdx.x / a.bins;
    const uint32_t from = part * gridDim.x / parts, to = (part + 1) * gridDim.x / parts;
    uint32_t earlier = 0, sum = 0;
#pragma unroll 16
    for (uint32_t k = from; k < to; k++) {
      const uint32_t n = a.counts[(uint64_t)k * a.bins + b];
      earlier += k < blockIdx.x ? n : 0, sum += n;
    }
    atomicAdd(&before[b], earlier), atomicAdd(&all[b], sum);
  }
  __syncthreads();
  const uint32_t b = threadIdx.x, mine = b < a.bins ? all[b] : 0;
  uint32_t lower = mine;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const uint32_t v = __shfl_up(lower, k);
    lower += lane >= (uint32_t)k ? v : 0;
  }
  if (lane == 63) sums[wave] = lower;
  __syncthreads();
  if (b < a.bins) {
    uint32_t place = lower - mine + before[b];
    for (uint32_t w = 0; w < wave; w++) place += sums[w];
    for (uint32_t w = 0; w < kSortWaves; w++) {
      const uint32_t n = at[w][b];
      at[w][b] = place;
      place += n;
    }
  }
  __syncthreads();
  constexpr uint32_t kAhead = 4;
  for (uint64_t base = first; base < end; base += 64 * kAhead) {
    uint32_t keys[kAhead], rows[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      const uint64_t i = base + 64 * k + lane;
      keys[k] = i < end ? a.key(i) : 0;
      rows[k] = i < end ? (a.tokens ? (uint32_t)i : a.order[i]) : 0;
    }
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      const bool there = base + 64 * k + lane < end;
      const uint32_t digit = (keys[k] >> a.shift) & (a.bins - 1);
      uint64_t same = __ballot(there);  // the lanes of the same digit
      for (uint32_t bit = 1; bit < a.bins; bit <<= 1) {
        const uint64_t set = __ballot(there && (digit & bit));
        same &= digit & bit ? set : ~set;
      }
      if (there) {
        const uint32_t place = at[wave][digit] + __builtin_popcountll(same & (((uint64_t)1 << lane) - 1));
        a.keys_out[place] = keys[k];
        a.order_out[place] = rows[k];
      }
      __builtin_amdgcn_wave_barrier();
      if (there && !(same >> lane >> 1)) at[wave][digit] += __builtin_popcountll(same);
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// The sums.

// The first of a lane's eight columns. The last lane of a row takes its last eight, some of them also the
// lane's before it, which writes the same: rows of any width are read and written eight values at a time.
__device__ __forceinline__ uint32_t eight_of(uint32_t i, uint32_t width) { return width < 8 ? 8 * i : min(8 * i, width - 8); }

// Eight values of a row to memory, in bf16 past the caches, which hold what is read meanwhile. In f32 a lane's values are two
// stores, each of which has every other 16 bytes of its lines, so that they go through the caches, where lines become whole: lookups of
// 262,144 rows of 256 80 us, past them 99; of 32,768 13.6 and 12.0.
template <class T>
__device__ __forceinline__ void store_past(T *row, uint32_t col, uint32_t cols, V8<T> v) {
  if (sizeof(T) == 2 && col + 8 <= cols) __builtin_nontemporal_store(v, (typename Loose<T, 8>::At *)(row + col));
  else store_some<T, 8>(row, col, cols, v);
}
// Zeros of a row's 8 LANES columns, the lanes' 16 bytes next to each other; the last ones are some of those before too. In bf16 past the
// caches: of 131,072 words of 1,024, most of which do not occur, 82 us, through them 107. In f32 through them, as whole rows past
// them gain where rows are whole lines (131,072 of 1,024 for 777 rows 139 us, through them 143; for 16,384 161 and 199) and lose where they
// are not or are short (60,000 of 1,001 79 and 50; 262,144 of 256 88 and 77). With the lanes' 16 bytes 32 apart the first took 323
// past the caches and 148 through them.
template <class T, int LANES>
__device__ __forceinline__ void write_zeros(T *row, uint32_t cols, uint32_t lane) {
  constexpr uint32_t kEach = 16 / sizeof(T), kSlice = 8 * LANES;
  const uint32_t first = blockIdx.y * kSlice;
#pragma unroll
  for (uint32_t c = 0; c < kSlice; c += kEach * LANES) {
    const uint32_t col = first + c + lane * kEach;
    if (col >= cols) continue;
    if (cols < kEach) {
      store_some<T, kEach>(row, col, cols, {});
      continue;
    }
    T *at = row + min(col, cols - kEach);
    if constexpr (sizeof(T) == 2) __builtin_nontemporal_store(typename Loose<T, kEach>::Values{}, (typename Loose<T, kEach>::At *)at);
    else loose<T, kEach>(at, {});
  }
}

// The first of the sorted rows whose word is not before `key`, looked for by a whole wavefront.
__device__ __forceinline__ uint32_t first_of(const uint32_t *keys, uint32_t rows, uint32_t key) {
  if (!rows || keys[0] >= key) return 0;
  return last_before<true>(rows, [&](uint32_t i) { return keys[i] < key; }) + 1;
}

// LANES lanes take a piece of `length` sorted rows and 8 LANES of their columns.
template <class R, class T, int LANES>
__global__ __launch_bounds__(256) void sorted_sums(Sums a) {
  const uint32_t lane = threadIdx.x % LANES;
  if (blockIdx.x >= a.sum_blocks) {  // zeros: 64 words a block, those that do not occur
    const uint64_t word0 = (uint64_t)(blockIdx.x - a.sum_blocks) * 64;
    const uint32_t word = (uint32_t)word0 + (threadIdx.x & 63), key = a.word0 + word;
    // The sorted rows of the 64 words: whole wavefronts look for their ends, and each lane for its word's between.
    uint32_t lo = first_of(a.keys, a.rows, a.word0 + (uint32_t)word0), hi = first_of(a.keys, a.rows, a.word0 + (uint32_t)word0 + 64);
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (a.keys[mid] < key) lo = mid + 1;
      else hi = mid;
    }
    const uint64_t none = __ballot(word < a.words && (lo == a.rows || a.keys[lo] != key));
    for (uint32_t k = threadIdx.x / LANES; k < 64; k += 256 / LANES)
      if (none >> k & 1) write_zeros<R, LANES>((R *)a.to + (int64_t)(word0 + k) * a.pitch, a.width, lane);
    return;
  }
  const uint32_t group = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, eight = blockIdx.y * LANES + lane, col = eight_of(eight, a.width);
  const uint64_t first = (uint64_t)group * a.length;
  if (group >= a.groups || eight * 8 >= a.width) return;
  const uint64_t end = first + a.length < a.rows ? first + a.length : a.rows;
  uint32_t key = a.keys[first];
  if (key >= a.word0 + a.words || a.keys[end - 1] < a.word0) return;
  bool whole = !(first && a.keys[first - 1] == key);  // the word's rows begin in this piece
  f32x8 sum = {};
  // Where a sum goes that ends here: the result's row, or a part for the second launch.
  auto put = [&](bool ends) {
    const uint32_t word = key - a.word0;
    if (word >= a.words) return;
    if (a.present && lane == 0 && blockIdx.y == 0) a.present[word] = 1;
    if (whole && ends) {
      store_some<R, 8>((R *)a.to + (int64_t)word * a.pitch, col, a.width, __builtin_convertvector(sum * a.scale, V8<R>));
    } else {
      store_some<float, 8>(a.parts + ((uint64_t)group * 2 + (whole ? 1 : 0)) * a.width, col, a.width, sum);
    }
  };
  // Eight rows on their way at a time, and their words and numbers eight before.
  constexpr uint32_t kAhead = 8;
  uint32_t keys[kAhead], rows[kAhead];
  auto look = [&](uint64_t i) {
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      const uint64_t at = i + k < end ? i + k : end - 1;
      keys[k] = a.keys[at], rows[k] = a.order[at];
    }
  };
  look(first);
  for (uint64_t i = first; i < end; i += kAhead) {
    uint32_t now[kAhead];
    f32x8 v[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      now[k] = keys[k];
      const bool wanted = i + k < end && keys[k] - a.word0 < a.words;
      v[k] = __builtin_convertvector((load_some<T, 8>((const T *)a.from + (int64_t)rows[k] * a.stride, wanted, col, a.width)), f32x8);
      if (a.weights && wanted) v[k] *= a.weights[rows[k]];
    }
    look(i + kAhead);
#pragma unroll
    for (uint32_t k = 0; k < kAhead; k++) {
      if (i + k >= end) break;
      if (now[k] != key) {
        put(true);
        key = now[k], sum = f32x8{}, whole = true;
      }
      sum += v[k];
    }
  }
  put(end == a.rows || a.keys[end] != key);
}

// A word whose rows began in a piece and go on in the next: its parts in their order. A block a piece; its lanes'
// groups take a stretch of the parts each.
template <class R, int LANES>
__global__ __launch_bounds__(256) void sorted_join(Sums a) {
  constexpr uint32_t kGroups = 256 / LANES;
  __shared__ float joined[kGroups][LANES * 8 + 1];
  const uint32_t group = blockIdx.x, lane = threadIdx.x % LANES, part = threadIdx.x / LANES, eight = blockIdx.y * LANES + lane;
  const uint32_t col = eight_of(eight, a.width);
  const uint64_t first = (uint64_t)group * a.length, end = first + a.length;
  if (end >= a.rows) return;
  const uint32_t key = a.keys[end - 1];
  if (key - a.word0 >= a.words || a.keys[end] != key) return;  // no word goes on
  if (first && a.keys[first - 1] == key) return;               // it began before this piece
  // The last piece that has it.
  const uint32_t lo = last_before<true>(a.groups, [&](uint32_t i) { return a.keys[(uint64_t)i * a.length] <= key; });
  // This piece's second part, then the first ones of pieces group + 1 .. lo.
  const uint32_t n = lo - group + 1, each = (n + kGroups - 1) / kGroups, from = part * each, to = from + each < n ? from + each : n;
  f32x8 sum = {};
  if (eight * 8 < a.width)
#pragma unroll 8
    for (uint32_t i = from; i < to; i++)
      sum += load_some<float, 8>(a.parts + ((uint64_t)(group + i) * 2 + (i ? 0 : 1)) * a.width, true, col, a.width);
#pragma unroll
  for (int e = 0; e < 8; e++) joined[part][lane * 8 + e] = sum[e];
  __syncthreads();
  if (part || eight * 8 >= a.width) return;
  for (uint32_t p = 1; p < kGroups; p++)
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] += joined[p][lane * 8 + e];
  store_some<R, 8>((R *)a.to + (int64_t)(key - a.word0) * a.pitch, col, a.width, __builtin_convertvector(sum * a.scale, V8<R>));
}

// Lanes of a row: as many as hold it, eight values each, up to a wavefront.
inline uint32_t lanes_of_row(uint32_t width) {
  uint32_t lanes = 4;
  while (lanes * 8 < width && lanes < 64) lanes *= 2;
  return lanes;
}
// f of the number of lanes as a constant.
template <class F>
inline void with_lanes(uint32_t width, F f) {
  switch (lanes_of_row(width)) {
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 8: f(std::integral_constant<int, 8>{}); break;
    case 16: f(std::integral_constant<int, 16>{}); break;
    case 32: f(std::integral_constant<int, 32>{}); break;
    default: f(std::integral_constant<int, 64>{});
  }
}

// Host side: where a sort and its sums have what, `bytes` in all.
struct SortPlan {
  uint32_t passes, bits, blocks, share;  // passes 0: by counting, in one launch
  uint32_t length, groups;
  uint64_t keys[2], order[2], counts, parts, bytes;
};
inline SortPlan sort_plan(uint32_t rows, uint32_t vocab, uint32_t width) {
  SortPlan p{};
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  p.keys[0] = take(4ull * rows), p.order[0] = take(4ull * rows);
  if (rows > kFew) {
    uint32_t bits = 1;
    while (vocab >> bits) bits++;  // of the largest word and of none
    p.passes = (bits + 9) / 10;
    p.bits = (bits + p.passes - 1) / p.passes;  // 2^bits divides a block's threads
    p.share = 4096;
    while ((uint64_t)p.share * kSortBlocks < rows) p.share *= 2;
    p.blocks = (rows + p.share - 1) / p.share;
    p.keys[1] = take(4ull * rows), p.order[1] = take(4ull * rows);
    p.counts = take(4ull * p.blocks << p.bits);
  }
  // Eight rows are on their way together; few rows are summed in one turn where that leaves the join's launch small (gradients of 14,692
  // rows of 64 over 1,898 words 159 us, with pieces of 16 165; an embedding's of 16,384 of 1,024 89 and 83).
  p.length = (uint64_t)rows * width <= 1 << 23 ? 8 : 16;
  while (p.length < 64 && rows / p.length > 2048) p.length *= 2;
  p.groups = (rows + p.length - 1) / p.length;
  p.parts = take(8ull * p.groups * width);
  p.bytes = at;
  return p;
}
// Sorts the rows by their words; `a` takes what the sums need to know.
inline void sort_rows(const SortPlan &p, const void *tokens, bool wide, uint32_t rows, uint32_t vocab, char *work, hipStream_t stream, Sums &a) {
  uint32_t *k[2] = {(uint32_t *)(work + p.keys[0]), (uint32_t *)(work + p.keys[1])};
  uint32_t *f[2] = {(uint32_t *)(work + p.order[0]), (uint32_t *)(work + p.order[1])};
  a.rows = rows, a.length = p.length, a.groups = p.groups, a.parts = (float *)(work + p.parts);
  a.keys = k[0], a.order = f[0];
  if (!rows) return;
  if (!p.passes) {
    const uint32_t all = (rows + 31) / 32 * 32;
    hipLaunchKernelGGL(sort_few, dim3((rows + 63) / 64), dim3(512), all * sizeof(uint32_t), stream, tokens, wide, rows, vocab, all, k[0], f[0]);
    return;
  }
  for (uint32_t i = 0; i < p.passes; i++) {
    const Digit d{rows, vocab, p.share, i * p.bits, 1u << p.bits, wide, i ? nullptr : tokens, k[(i + 1) & 1], f[(i + 1) & 1],
                  (uint32_t *)(work + p.counts), k[i & 1], f[i & 1]};
    hipLaunchKernelGGL(sort_count, dim3(p.blocks), dim3(kSortThreads), 0, stream, d);
    hipLaunchKernelGGL(sort_place, dim3(p.blocks), dim3(kSortThreads), 0, stream, d);
    a.keys = d.keys_out, a.order = d.order_out;
  }
}
template <class R, class T>
inline void sum_rows(const Sums &a, hipStream_t stream) {
  with_lanes(a.width, [&](auto lanes) {
    constexpr uint32_t kGroups = 256 / lanes();
    Sums b = a;
    b.sum_blocks = (a.groups + kGroups - 1) / kGroups;
    const uint32_t slices = (a.width + lanes() * 8 - 1) / (lanes() * 8);
    hipLaunchKernelGGL((sorted_sums<R, T, lanes()>), dim3(b.sum_blocks + (a.present ? 0 : (a.words + 63) / 64), slices), dim3(256), 0, stream, b);
    if (a.groups > 1) hipLaunchKernelGGL((sorted_join<R, lanes()>), dim3(a.groups - 1, slices), dim3(256), 0, stream, b);
  });
}

}  // namespace trunk
