// head_grad.hip - the gradients of the head's softmax cross entropy, without keeping its logits:
//
//   G_tv = (dloss_t + dlse_t) e^(z_tv - lse_t) - dloss_t [v = target_t],  dx = G W,  dW = G^T x.
//
// A piece of the rows by a piece of the vocabulary at a time: one launch computes the piece's logits again
// and writes its G, in the type of x, to scratch memory; one takes G W and one G^T x from it. dx is summed over the pieces of the
// vocabulary and dW over those of the rows, in 32 bits. Where a product's tiles leave compute units idle in the card's last turn, the
// summed axis is shared out evenly instead, and the shares of a tile are joined by a launch behind. How many rows are packed is known
// on the card alone, so that what a block does is worked out there, of the rows that there are.
//
// G is rounded to bf16 where x is, half a step (2^-8) of each value, independent of the others. Of the largest,
// the target's, that would be an error of the whole row: it is left out of G, and its terms G_t,target W_target
// and G_t,target x_t are added to dx and dW in 32 bits at their ends, dW's by sorted targets.
#include "few.h"
#include "sorted.h"

namespace trunk {

struct Logits {
  Matrix w, x;      // x: the piece's panels
  uint32_t rows, vocab, width;
  uint32_t row0, piece_rows, word0, word_tiles;  // the piece, in the shape's tiles
  uint32_t blocks, at_once;  // see RowShares
  const uint32_t *count;
  const int32_t *target;
  const float4 *factors;
  const int32_t *order;
  float *terms;     // [rows of the call]: the targets' G, where x is bf16
  char *g;          // [words / a panel's][g_rows][64 bytes]
  uint32_t g_rows;
};

template <class T, class S, Lies W>
struct LogitTiles {
  static constexpr int kStores = S::M * S::N * (sizeof(T) == 2 ? 2 : 4);
  const Logits &a;
  uint32_t tiles;
  Walk ahead, at;   // in the piece
  int lane, wave;
  float base[S::N], all[S::N], one[S::N];
  int32_t target[S::N], place[S::N];

  // A row tile's beginning.
  __device__ __forceinline__ void open() {
#pragma unroll
    for (int j = 0; j < S::N; j++) {
      const uint32_t row = a.row0 + at.row * S::kN + 32 * S::N * (wave & 1) + 32 * j + (lane & 31);
      const float4 f = a.factors[row];
      base[j] = f.x, all[j] = f.y, one[j] = f.z, target[j] = a.target[row], place[j] = a.order[row];
    }
  }
  __device__ __forceinline__ uint32_t stages(uint32_t) const { return (a.width + kDeep<T> - 1) / kDeep<T>; }

  // A logit's share of its row; in 32 bits with what the rounding of its exponent leaves.
  static __device__ __forceinline__ float share(float z, float base) {
    if constexpr (sizeof(T) == 2) return exp2_(fmaf(z, kLog2e, -base));
    const float v = z - base < -120.0f ? -120.0f : z - base, t = v * kLog2e;
    const float left = fmaf(v, 1.92596299e-8f, fmaf(v, kLog2e, -t)), e = exp2_(t);
    return fmaf(e, left * 0.693147181f, e);
  }
  template <class FA, class FB>
  __device__ __forceinline__ void feed(uint32_t, FA &fa, FB &fb) {
    const uint32_t word = a.word0 + ahead.word * S::kM, row0 = ahead.row * S::kN;
    ahead.next();
    fa.start(a.w.at + (int64_t)word * (W == ROWS ? a.w.pitch : 64), a.w.pitch, a.vocab - word, a.width);
    fb.start(a.x.at + row0 * 64, a.x.pitch, S::kN, a.width);
  }
  __device__ __forceinline__ void take(uint32_t n, f32x16 (&z)[S::M][S::N]) {
    const int half = lane >> 5;
    const uint32_t word = a.word0 + at.word * S::kM + 32 * S::M * (wave >> 1), row0 = at.row * S::kN;
    if (word + 32 * S::M > a.vocab) cut_rows(z, a.vocab > word ? a.vocab - word : 0, half);  // their G is 0
#pragma unroll
    for (int j = 0; j < S::N; j++) {
#pragma unroll
      for (int i = 0; i < S::M; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) z[i][j][r] = all[j] * share(z[i][j][r], base[j]);
      const uint32_t own_word = (uint32_t)target[j] - word;
      if (__any(own_word < 32 * S::M)) {
        float term = 0.0f;
        const int own = (int)own_word - 4 * half;
#pragma unroll
        for (int i = 0; i < S::M; i++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const bool here = own == 32 * i + row_of(r, 0);
            if constexpr (sizeof(T) == 2) term = here ? z[i][j][r] : term, z[i][j][r] = here ? 0.0f : z[i][j][r];
            else z[i][j][r] -= here ? one[j] : 0.0f;
          }
        if (sizeof(T) == 2 && own_word < 32 * S::M && (int)(own_word >> 2 & 1) == half) a.terms[place[j]] = term - one[j];
      }
      const uint64_t panel = (uint64_t)a.g_rows * 64;
      char *to = a.g + (word - a.word0) / kDeep<T> * panel + (row0 + 32 * S::N * (wave & 1) + 32 * j + (lane & 31)) * 64;
#pragma unroll
      for (int i = 0; i < S::M; i++) {
        if constexpr (sizeof(T) == 2) {
          // A lane has four words of every eight, the lane 32 on the other four: they change places, so that
          // each writes eight next to each other.
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            uint32_t p[2][2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const bf16x2 lo = {(bf16)z[i][j][4 * q + 2 * e], (bf16)z[i][j][4 * q + 2 * e + 1]};
              const bf16x2 hi = {(bf16)z[i][j][4 * q + 4 + 2 * e], (bf16)z[i][j][4 * q + 5 + 2 * e]};
              const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi), false, false);
              p[0][e] = both[0], p[1][e] = both[1];
            }
            *(u32x4 *)(to + i * panel + 16 * (q + half)) = u32x4{p[0][0], p[0][1], p[1][0], p[1][1]};
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; q++)
            *(f32x4 *)(to + (2 * i + q / 2) * panel + 32 * (q & 1) + 16 * half) = f32x4{z[i][j][4 * q], z[i][j][4 * q + 1], z[i][j][4 * q + 2], z[i][j][4 * q + 3]};
        }
      }
    }
    if (at.next() && n + 1 < tiles) open();
  }
};

template <class T, class S, Lies W>
__global__ __launch_bounds__(256, S::kBlocks) void head_logits(Logits a) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  const uint32_t count = *a.count, rows = count > a.row0 ? min(count - a.row0, a.piece_rows) : 0;
  const Walk walk(RowShares(rows, S::kN, a.word_tiles, a.blocks, a.at_once), a.word_tiles, blockIdx.x);
  if (!walk.tiles) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  LogitTiles<T, S, W> tiles{a, walk.tiles, walk, walk, lane, wave};
  tiles.open();
  run_tiles<T, S, true, W, true, PANELS>(lds, tiles);
}

// The same for few rows of 32 bits. A block's 16 words are a panel of G.
struct FewLogits {
  Few f;
  const uint32_t *count;
  const int32_t *order, *target;
  const float4 *factors;
  char *g;          // [words / 16][g_rows][64 bytes]
  uint32_t g_rows;
};
template <int TILES>
__global__ __launch_bounds__(256) void head_few_logits(FewLogits a) {
  using Tiles = LogitTiles<float, Small, ROWS>;
  const uint32_t rows = *a.count;
  float4 factor[TILES];
  int32_t target[TILES];
#pragma unroll
  for (int j = 0; j < TILES; j++) {
    const uint32_t row = 16 * j + threadIdx.x % 16;
    factor[j] = a.factors[row], target[j] = a.target[row];
  }
  few_logits<float, TILES>(a.f, rows, a.order, [&](int j, uint32_t word, float z) {
    const uint32_t row = 16 * j + threadIdx.x % 16, at = word - a.f.word0;
    if (row >= rows) return;
    const float g = word < a.f.vocab ? factor[j].y * Tiles::share(z, factor[j].x) - ((int32_t)word == target[j] ? factor[j].z : 0.0f) : 0.0f;
    *(float *)(a.g + ((uint64_t)(at / 16) * a.g_rows + row) * 64 + at % 16 * 4) = g;
  });
}

// How a product's blocks share it. A group of blocks takes all columns' tiles abreast through its share of the row tiles'
// stages, so that it reads its rows of G once. A tile that is whole in a group's share ends there; of others every group leaves its
// sums in a slot, two of which a block has: of a tile that begins in its share, and of one that does not.
struct Split {
  uint32_t m, k;           // the piece's rows of the result and its summed axis; of dx or dW fewer, where fewer rows are packed
  uint32_t row0;           // the piece's first packed row
  const uint32_t *count;   // how many packed rows there are
  uint32_t tile_m, tile_n, n_tiles;
  uint32_t groups;         // or 0: a group has one row tile
  bool dw;
};
// Values between slots, so that blocks that write theirs in step do not meet in a memory channel.
constexpr uint32_t kSlotPad = 64;
struct SplitShares {
  uint32_t there, k, stages;  // rows of the piece; the summed axis; its stages
  uint32_t units, groups;     // row tiles by stages: under 2^18, so that their product with the groups is of 32 bits
  uint32_t m_tiles, of_tile;  // groups of a row tile, where all have as many: then no group has two, and those of all tiles go abreast
  __device__ __forceinline__ SplitShares(const Split &a, uint32_t deep) {
    there = *a.count > a.row0 ? *a.count - a.row0 : 0;
    k = a.dw && there < a.k ? there : a.k;
    m_tiles = ((!a.dw && there < a.m ? there : a.m) + a.tile_m - 1) / a.tile_m;
    stages = (k + deep - 1) / deep;
    units = m_tiles * stages;
    groups = m_tiles;
    of_tile = 1;
    if (!a.groups) return;
    of_tile = 0;
    if (!units) {
      groups = 0;
      return;
    }
    groups = min(a.groups, units < 8 ? 1u : units / 8);  // eight stages at least, or four
    const uint32_t more = (groups + m_tiles - 1) / m_tiles, fewer = more * m_tiles == groups ? more : more - 1;
    if (more * m_tiles <= a.groups && more * m_tiles * 4 <= units) of_tile = more;
    else if (fewer && (groups - fewer * m_tiles) * 16 <= groups) of_tile = fewer;
    if (of_tile) groups = of_tile * m_tiles;
  }
  __device__ __forceinline__ uint32_t first(uint32_t group) const { return units * group / groups; }
  __device__ __forceinline__ uint32_t of(uint32_t unit) const { return ((unit + 1) * groups - 1) / units; }
};

// A product of a piece: out[m][n] (+)= sum_k a[m][k] b[k][n].
struct Product {
  Split split;
  Matrix a, b;             // a: panels of G
  uint32_t n;              // columns, whole 16 bytes of values
  float *slots;            // [blocks][2][a tile's rows][a tile's columns], kSlotPad apart
  float *sums;             // [rows of the result][n_pitch]: the pieces' so far
  uint32_t n_pitch;
  bool first;              // nothing has been summed before
  // A result that is whole with a tile is rounded and written, with the targets' terms.
  void *to;                // [words][n_to], the piece's first (dx: [rows of the call][n_to]), or NULL
  uint32_t words, n_to;    // words: of the piece (dx: not looked at)
  bool f32;                // its type
  const uint8_t *present;  // dW: which words have terms
  const float *terms;      // dW: [words][n_pitch], or NULL; dx: [rows of the call], or NULL
  const int32_t *order, *target;  // dx: packed rows' places and targets
  const void *w;           // dx: the matrix as the caller has it
  int64_t w_stride;
};

// v of the lane next to an even one, or before an odd one.
__device__ __forceinline__ float neighbour(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, false));
}


// DW: the summed axis are the rows of x, else the words. B: how x or the matrix lies.
template <class T, class S, bool DW, Lies B>
struct ProductTiles {
  static constexpr bool kPuts = DW || S::M * S::N <= 4;  // large tiles of dx have sums of pieces to join anyway
  static constexpr int kStores = 0;
  const Product &p;
  const SplitShares &share;
  uint32_t tiles, slot, m_tile, n0, from, to, there;  // from, to: the block's units; m_tile: its first
  int lane, wave;
  // The n-th tile's part of the summed axis, in stages.
  __device__ __forceinline__ uint32_t begin(uint32_t n) const { return n ? 0 : from - m_tile * share.stages; }
  __device__ __forceinline__ uint32_t end(uint32_t n) const { return n + 1 < tiles ? share.stages : to - (m_tile + n) * share.stages; }
  __device__ __forceinline__ uint32_t stages(uint32_t n) const { return end(n) - begin(n); }
  template <class FA, class FB>
  __device__ __forceinline__ void feed(uint32_t n, FA &fa, FB &fb) {
    const uint32_t m0 = (m_tile + n) * S::kM, k0 = begin(n) * kDeep<T>, k1 = end(n) * kDeep<T>, depth = min(k1, share.k) - k0;
    // k0, m0 and n0 are whole panels.
    if constexpr (DW) {
      fa.start(p.a.at + m0 / kDeep<T> * p.a.pitch + (uint64_t)k0 * 64, p.a.pitch, S::kM, depth);
    } else {
      fa.start(p.a.at + k0 / kDeep<T> * p.a.pitch + (uint64_t)m0 * 64, p.a.pitch, S::kM, depth);
    }
    if constexpr (B == PANELS) fb.start(p.b.at + n0 / kDeep<T> * p.b.pitch + (uint64_t)k0 * 64, p.b.pitch, p.n - n0, depth);
    else fb.start(p.b.at + (int64_t)k0 * p.b.pitch + n0 * sizeof(T), p.b.pitch, p.n - n0, depth);
  }
  // bf16 results go out two columns a lane: two rows of a pair of lanes change places. What is to be known of 32 rows is
  // read by a lane each, and the terms of eight of a lane's rows are on their way together: one at a time, behind each other's loads,
  // loss and gradients of 200 rows of 512 over 100 words took 59 us, so 47.
  __device__ __forceinline__ void put(uint32_t m0, f32x16 (&sums)[S::M][S::N]) {
    const int half = lane >> 5;
    const uint32_t word0 = m0 + 32 * S::M * (wave >> 1), col0 = n0 + 32 * S::N * (wave & 1) + (lane & 31), most = DW ? p.words : there;
    const bool pairs = !p.f32 && p.n_to % 2 == 0 && ((uintptr_t)p.to & 3) == 0;
#pragma unroll
    for (int i = 0; i < S::M; i++) {
      const uint32_t word = word0 + 32 * i + (lane & 31);
      const bool mine = word < most;
      uint32_t place = word, has = 0;
      int32_t target = 0;
      float factor = 0.0f;
      if constexpr (!DW) place = mine ? (uint32_t)p.order[p.split.row0 + word] : 0;
      if constexpr (sizeof(T) == 2) {
        has = (uint32_t)__ballot(mine && p.terms && (!DW || p.present[word]));
        if constexpr (!DW)
          if (has) target = mine ? p.target[p.split.row0 + word] : 0, factor = p.terms[place];
      }
#pragma unroll
      for (int j = 0; j < S::N; j++) {
        const uint32_t col = col0 + 32 * j;
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += 8) {
          float terms[8] = {};
          if (sizeof(T) == 2 && has) {
#pragma unroll
            for (int r = 0; r < 8; r++) {
              const uint32_t row = row_of(r0 + r, half);
              const bool on = has >> row & 1 && col < p.n_to;
              float v;
              if constexpr (DW) {
                v = p.terms[on ? (uint64_t)(word0 + 32 * i + row) * p.n_pitch + col : 0];
              } else {
                const int32_t word = __shfl(target, row);
                v = __shfl(factor, row) * (float)((const bf16 *)p.w)[on ? word * p.w_stride + col : 0];
              }
              terms[r] = on ? v : 0.0f;
            }
          }
#pragma unroll
          for (int r = 0; r < 8; r += 2) {
            const uint32_t row = row_of(r0 + r, half);
            uint64_t places[2] = {word0 + 32 * i + row, word0 + 32 * i + row + 1};
            if constexpr (!DW) places[0] = (uint32_t)__shfl((int)place, row), places[1] = (uint32_t)__shfl((int)place, row + 1);
            put(word0 + 32 * i + row, most, places, col, pairs, sums[i][j][r0 + r] + terms[r], sums[i][j][r0 + r + 1] + terms[r + 1]);
          }
          asm volatile("" ::: "memory");  // else all the words' terms are read, and kept, before any is used
        }
      }
    }
  }
  __device__ __forceinline__ void put(uint32_t word, uint32_t most, const uint64_t (&places)[2], uint32_t col, bool pairs, float a, float b) {
    if (pairs) {
      const float other = neighbour(lane & 1 ? a : b);
      const bf16x2 v = {(bf16)(lane & 1 ? other : a), (bf16)(lane & 1 ? b : other)};
      const uint32_t at = col & ~1u;
      if (word + (lane & 1) < most && at < p.n_to) *(bf16x2 *)((bf16 *)p.to + places[lane & 1] * p.n_to + at) = v;
    } else if (col < p.n_to) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        if (word + e >= most) continue;
        const uint64_t at = places[e] * p.n_to + col;
        if (p.f32) ((float *)p.to)[at] = e ? b : a;
        else ((bf16 *)p.to)[at] = (bf16)(e ? b : a);
      }
    }
  }
  __device__ __forceinline__ void take(uint32_t n, f32x16 (&sums)[S::M][S::N]) {
    const int half = lane >> 5;
    const uint32_t m0 = (m_tile + n) * S::kM;
    const bool whole = begin(n) == 0 && end(n) == share.stages;
    if constexpr (kPuts)
      if (whole && p.to) return put(m0, sums);
    const uint32_t row = 32 * S::M * (wave >> 1) + 4 * half, col = 32 * S::N * (wave & 1) + (lane & 31);
    if (!whole) {
      float *to = p.slots + (uint64_t)(2 * slot + (begin(n) == 0)) * (S::kM * S::kN + kSlotPad) + row * S::kN + col;
#pragma unroll
      for (int i = 0; i < S::M; i++)
#pragma unroll
        for (int r = 0; r < 16; r++)
#pragma unroll
          for (int j = 0; j < S::N; j++) to[(32 * i + row_of(r, 0)) * S::kN + 32 * j] = sums[i][j][r];
      return;
    }
    float *to = p.sums + (uint64_t)(m0 + row) * p.n_pitch + n0 + col;
#pragma unroll
    for (int i = 0; i < S::M; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        float *at = to + (uint64_t)((32 * i + row_of(r, 0)) * p.n_pitch);
#pragma unroll
        for (int j = 0; j < S::N; j++) at[32 * j] = p.first ? sums[i][j][r] : at[32 * j] + sums[i][j][r];
      }
  }
};

template <class T, class S, bool DW, Lies B>
__global__ __launch_bounds__(256, S::kBlocks) void head_product(Product p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  const SplitShares share(p.split, kDeep<T>);
  const uint32_t blocks = share.groups * p.split.n_tiles;
  if (blockIdx.x >= blocks) return;
  const uint32_t work = by_xcd(blockIdx.x, blocks), n_tile = work % p.split.n_tiles, n0 = n_tile * S::kN;
  uint32_t group = work / p.split.n_tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (!share.stages) {  // sums over nothing, a tile a group
    ProductTiles<T, S, DW, B> tiles{p, share, 1, 0, group, n0, 0, 0, share.there, lane, wave};
    f32x16 sums[S::M][S::N] = {};
    return tiles.take(0, sums);
  }
  uint32_t from, to, m_tile, n = 1;
  if (share.of_tile) {
    const uint32_t part = group / share.m_tiles;
    m_tile = group - part * share.m_tiles, group = m_tile * share.of_tile + part;
    const uint32_t each = share.stages / share.of_tile, one = share.stages - each * share.of_tile;  // so many have one more
    from = m_tile * share.stages + part * each + min(part, one), to = from + each + (part < one);
  } else {
    from = share.first(group), to = share.first(group + 1), m_tile = from / share.stages, n = (to - 1) / share.stages - m_tile + 1;
  }
  ProductTiles<T, S, DW, B> tiles{p, share, n, group * p.split.n_tiles + n_tile, m_tile, n0, from, to, share.there, lane, wave};
  run_tiles<T, S, !DW, PANELS, false, B>(lds, tiles);
}

// A product's tiles that no group has whole (or, where the product has not written them to their places, all tiles): the groups'
// sums in their order, added to those of the pieces before; with the last piece rounded to the result's type. dx: packed
// rows go to their own places, with their targets' terms.
struct Ends {
  Split split;
  uint32_t deep;           // values of a stage
  const float *slots;
  float *sums;             // the piece's
  uint32_t n, n_pitch;
  bool first, last;        // piece
  bool put;                // the product has written whole tiles to their places
  uint32_t rows;           // of the result's that are wanted; of dx as many as are packed
  const int32_t *order, *target;
  const float *terms;      // dx: [rows of the call], or NULL
  const float *word_terms; // dW: [words][n_pitch], or NULL
  const uint8_t *present;  // dW's words with terms
  const void *w;           // the matrix as the caller has it
  int64_t w_stride;
  void *to;
};
// SHARES threads take eight values of a row, a stretch of the slots each.
template <class R, int SHARES>
__global__ __launch_bounds__(256) void head_sums(Ends a) {
  constexpr uint32_t kEach = 256 / SHARES;
  __shared__ float joined[SHARES > 1 ? 256 : 1][9];
  const SplitShares share(a.split, a.deep);
  // A block has some rows of a tile.
  const uint32_t m_tile = blockIdx.x / a.split.n_tiles, n_tile = blockIdx.x % a.split.n_tiles;
  const uint32_t mine = threadIdx.x / kEach, i = blockIdx.y * kEach + threadIdx.x % kEach, pieces = a.split.tile_n / 8;
  const uint32_t row_in = i / pieces, col_in = i % pieces * 8, row = m_tile * a.split.tile_m + row_in, col = n_tile * a.split.tile_n + col_in;
  const uint32_t limit = !a.split.dw && share.there < a.rows ? share.there : a.rows;
  // The groups that have some of the tile.
  uint32_t first = 0, n = 0;
  if (m_tile * a.split.tile_m >= limit) return;
  const uint32_t unit = m_tile * share.stages;
  if (share.of_tile) first = m_tile * share.of_tile, n = share.of_tile;
  else if (share.stages) first = share.of(unit), n = share.of(unit + share.stages - 1) - first + 1;
  const bool whole = n == 1;
  if (whole && (a.put || !a.last)) return;
  const bool wanted = row < limit && col < a.n;
  f32x8 v = {};
  if (wanted && !whole) {
    const uint32_t from = n * mine / SHARES, to = n * (mine + 1) / SHARES, tile = a.split.tile_m * a.split.tile_n + kSlotPad;
#pragma unroll 8
    for (uint32_t g = from; g < to; g++)
      v += loose<float, 8>(a.slots + (uint64_t)(2 * ((first + g) * a.split.n_tiles + n_tile) + (g == 0)) * tile + row_in * a.split.tile_n + col_in);
  }
  if constexpr (SHARES > 1) {
#pragma unroll
    for (int e = 0; e < 8; e++) joined[threadIdx.x][e] = v[e];
    __syncthreads();
    if (mine == 0)
      for (int k = 1; k < SHARES; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += joined[k * kEach + threadIdx.x][e];
  }
  if (!wanted || mine) return;
  float *sums = a.sums + (uint64_t)row * a.n_pitch + col;
  if (whole || !a.first) v += loose<float, 8>(sums);
  if (!a.last) {
    loose<float, 8>(sums, v);
    return;
  }
  const uint64_t place = a.order ? (uint64_t)(uint32_t)a.order[a.split.row0 + row] : row;
  if (a.present && a.present[row]) v += loose<float, 8>(a.word_terms + (uint64_t)row * a.n_pitch + col);
  if (a.terms)
    v += __builtin_convertvector((load_some<bf16, 8>((const bf16 *)a.w + a.target[a.split.row0 + row] * a.w_stride, true, col, a.n)), f32x8) *
         a.terms[place];
  store_some<R, 8>((R *)a.to + place * a.n, col, a.n, __builtin_convertvector(v, V8<R>));
}

// The targets' terms of dW for few rows, without a sort: a wavefront a row and 512 columns. The first row of
// a word sums all of them, in their order.
constexpr uint32_t kFewTerms = 256;
template <class T>
__global__ __launch_bounds__(64) void head_terms(Sums a, const void *targets, bool wide, uint32_t vocab) {
  const uint32_t row = blockIdx.x, eight = blockIdx.y * 64 + threadIdx.x, col = eight_of(eight, a.width);
  const int32_t mine = target_of(targets, wide, row, vocab);
  if (mine < 0 || (uint32_t)mine - a.word0 >= a.words) return;
  uint64_t same[kFewTerms / 64];
  bool later = false;
#pragma unroll
  for (uint32_t k = 0; k < kFewTerms / 64; k++) {
    const uint32_t other = 64 * k + threadIdx.x;
    same[k] = __ballot(other < a.rows && target_of(targets, wide, other < a.rows ? other : 0, vocab) == mine);
    later |= row >= 64 * k && (same[k] & (row - 64 * k < 64 ? ((uint64_t)1 << (row - 64 * k)) - 1 : ~(uint64_t)0));
  }
  if (later) return;
  f32x8 sum = {};
#pragma unroll
  for (uint32_t k = 0; k < kFewTerms / 64; k++)
    for (uint64_t left = eight * 8 < a.width ? same[k] : 0; left; left &= left - 1) {
      const uint32_t other = 64 * k + __builtin_ctzll(left);
      sum += __builtin_convertvector((load_some<T, 8>((const T *)a.from + (int64_t)other * a.stride, true, col, a.width)), f32x8) * a.weights[other];
    }
  const uint32_t word = (uint32_t)mine - a.word0;
  if (threadIdx.x == 0 && blockIdx.y == 0) a.present[word] = 1;
  if (eight * 8 < a.width) store_some<float, 8>((float *)a.to + (int64_t)word * a.pitch, col, a.width, sum);
}

// The gradient of no rows.
template <class R>
__global__ __launch_bounds__(256) void head_nothing(R *to, uint64_t n) {
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) to[i] = (R)0.0f;
}

namespace {

// Bytes of a piece's G. Larger pieces read and write the sums so far less often; this much is a small part of
// the memory of the card. Loss and gradients of 32,768 rows (a quarter without a target) at width 256 and 32,768
// words: 256 MB 2,615 us, 512 MB 2,350, 1 GB 2,150 to 2,205, 2 GB 2,205 to 2,260; 8,192 rows at width 1,024 and 131,072
// words: 8,490, 8,555, 8,475 and 8,450.
constexpr uint64_t kPiece = 1ull << 30;

struct GradPlan {
  bool lay;
  uint32_t width, rows, words;  // a row's values; rows and words of a piece, whole tiles
  uint32_t all_rows, all_words;          // of the call, whole tiles
  uint32_t tile_m, tile_n, at_once, n_tiles, n_pitch;
  uint32_t x_rows, w_rows;               // how many rows' and words' sums are kept at once
  bool puts_x, puts_w;                   // products write whole tiles to their places: there are no pieces to be summed
  SortPlan sort;                         // of the targets, where x is bf16
  uint64_t g, dx, dw, slots, word_terms, w, x, order, target, factors, terms, sorted, present, counts, count, bytes;
};
// Groups that share a product's stages, or 0 where each takes a row tile. Tiles that do not fill the card's last turn leave it idle
// for so many stages (of 0.9 us in large bf16 tiles and of 2.1 us in 32 bits); the tiles' sums in slots cost up to 40 us and 20.
// 7,260 rows of 609 over 2,562 words in 32 bits 848 us, without shares 1,017; 24,576 of 32,768 rows of 256 over 32,768 words 2,199 and
// 2,511; 1,322 rows of 1,838 over 11,168 words, whose dW would gain 30 stages, 425 with them and 366 without.
uint32_t groups_for(const GradPlan &p, uint32_t m, uint32_t k, uint32_t deep) {
  const uint64_t tiles = (uint64_t)((m + p.tile_m - 1) / p.tile_m) * p.n_tiles, stages = (k + deep - 1) / deep;
  const uint64_t idle = (tiles + p.at_once - 1) / p.at_once * stages - tiles * stages / p.at_once;
  return stages < 16 || (2 * tiles > p.at_once && idle < (deep == 32 ? 48 : 12)) ? 0 : p.at_once / p.n_tiles;
}
// The size of even pieces of `all` that are `most` at most, in whole large tiles.
uint32_t even_pieces(uint64_t all, uint64_t most) {
  const uint64_t n = (all + most - 1) / most;
  return (uint32_t)up((all + n - 1) / n, kRound);
}
GradPlan grad_plan(const uor_trunk_head_args *s) {
  GradPlan p{};
  const uint32_t size = size_of(s->dtype), deep = 64 / size;
  p.width = (uint32_t)up(s->width, 16 / size);
  p.lay = laid_out(s);
  const Tiling t = tiling(s);
  p.tile_m = t.m, p.tile_n = t.n, p.at_once = t.at_once;
  p.all_rows = (uint32_t)up(s->rows, kRound), p.all_words = (uint32_t)up(s->vocab, kRound);
  // A piece of about as many rows as words, whose sums are read and written the least for the G between.
  const uint64_t values = kPiece / size;
  uint64_t side = kRound;
  while ((side + kRound) * (side + kRound) <= values) side += kRound;
  p.rows = even_pieces(p.all_rows, side);
  p.words = even_pieces(p.all_words, values / p.rows / kRound * kRound);
  p.rows = even_pieces(p.all_rows, values / p.words / kRound * kRound);
  p.n_tiles = (p.width + p.tile_n - 1) / p.tile_n;
  p.n_pitch = p.n_tiles * p.tile_n;
  // With the rows' pieces outside, the sums of dx are kept of one of them and those of dW of all words; or the
  // other way round.
  const bool rows_outside = p.all_rows - p.rows > p.all_words - p.words;
  p.x_rows = rows_outside ? p.rows : p.all_rows, p.w_rows = rows_outside ? p.all_words : p.words;
  p.puts_x = p.tile_m < Large::kM && p.words >= p.all_words, p.puts_w = p.rows >= p.all_rows;
  const uint64_t x_units = s->dx ? (uint64_t)p.rows / p.tile_m * (p.words / deep) : 0;
  const uint64_t w_units = s->dweight ? (uint64_t)p.words / p.tile_m * (p.rows / deep) : 0;
  const uint64_t units = x_units > w_units ? x_units : w_units, groups = p.at_once / p.n_tiles, most = units < 8 ? 1 : units / 4;  // see SplitShares
  Scratch at;
  p.g = at.take((uint64_t)p.rows * p.words * size);
  p.dx = at.take(!s->dx || p.puts_x ? 0 : 4ull * p.x_rows * p.n_pitch);
  p.dw = at.take(!s->dweight || p.puts_w ? 0 : 4ull * p.w_rows * p.n_pitch);
  p.slots = at.take(8ull * (groups < most ? groups : most) * p.n_tiles * (p.tile_m * p.tile_n + kSlotPad));
  p.word_terms = at.take(size == 2 && s->dweight ? 4ull * p.words * p.n_pitch : 0);
  p.w = at.take(p.lay ? s->vocab * up(s->width * size, 64) : 0);
  p.x = at.take(up(p.all_rows, p.rows) * up(s->width * size, 64));
  p.order = at.take(4ull * p.all_rows);
  p.target = at.take(4ull * p.all_rows);
  p.factors = at.take(16ull * p.all_rows);
  if (size == 2) {
    p.sort = sort_plan(s->rows, s->vocab, s->width);
    p.sorted = at.take(s->dweight ? p.sort.bytes : 0);
    p.terms = at.take(4ull * s->rows);
    p.present = at.take(s->dweight ? s->vocab : 0);
  }
  p.counts = at.take((s->rows + kPackRows - 1) / kPackRows * 4);
  p.count = at.take(4);
  p.bytes = at.bytes;
  return p;
}

template <class R>
void sums(const Ends &a, hipStream_t stream) {
  const uint32_t m_tiles = (a.rows + a.split.tile_m - 1) / a.split.tile_m;
  const auto run = [&](auto kernel, uint32_t each) {
    hipLaunchKernelGGL(kernel, dim3(m_tiles * a.split.n_tiles, a.split.tile_m * a.split.tile_n / 8 / each), dim3(256), 0, stream, a);
  };
  if (a.split.groups >= 16 * m_tiles) run(head_sums<R, 8>, 32);
  else run(head_sums<R, 1>, 256);
}

template <class T>
int grad(const uor_trunk_head_args *s, char *work, hipStream_t stream) {
  const GradPlan p = grad_plan(s);
  const int64_t panel = (int64_t)p.rows * 64;  // of G and of a piece of x
  Matrix w{(const char *)s->weight, s->w_stride * (int64_t)sizeof(T)};
  if (p.lay) w = lay<T>(s->weight, s->w_stride, s->vocab, s->width, work + p.w, stream);
  uint32_t *count = (uint32_t *)(work + p.count);
  Pack k{};
  k.rows = s->rows, k.width = s->width, k.vocab = s->vocab, k.piece = p.rows, k.stride = s->x_stride;
  k.x = s->x, k.targets = s->targets, k.wide = s->wide != 0;
  k.to = work + p.x, k.order = (int32_t *)(work + p.order), k.target = (int32_t *)(work + p.target), k.count = count;
  k.lse_in = s->lse, k.dlosses = s->dlosses, k.dlse = s->dlse, k.factors = (float4 *)(work + p.factors);
  k.dx = s->dx, k.present = sizeof(T) == 2 && s->dweight ? (uint8_t *)(work + p.present) : nullptr;
  pack<T, true>(k, (uint32_t *)(work + p.counts), stream);
  constexpr bool kTerms = sizeof(T) == 2;
  float *terms = kTerms ? (float *)(work + p.terms) : nullptr;
  Sums t{};
  if (kTerms && s->dweight) {
    t.width = s->width, t.scale = 1.0f, t.stride = s->x_stride, t.pitch = p.n_pitch, t.from = s->x, t.weights = terms, t.present = k.present;
    t.rows = s->rows;
    if (s->rows > kFewTerms) sort_rows(p.sort, s->targets, s->wide != 0, s->rows, s->vocab, work + p.sorted, stream, t);
  }
  // Of the two axes' pieces, one's are outside: see grad_plan.
  const uint32_t row_pieces = (s->rows + p.rows - 1) / p.rows, word_pieces = (s->vocab + p.words - 1) / p.words;
  const bool rows_outside = p.x_rows < p.all_rows;
  for (uint32_t i = 0; i < row_pieces * word_pieces; i++) {
    const uint32_t row_piece = rows_outside ? i / word_pieces : i % row_pieces, word_piece = rows_outside ? i % word_pieces : i / row_pieces;
    const uint32_t row0 = row_piece * p.rows, word0 = word_piece * p.words;
    const uint32_t rows = s->rows - row0 < p.rows ? s->rows - row0 : p.rows, words = s->vocab - word0 < p.words ? s->vocab - word0 : p.words;
    const uint32_t word_tiles = (words + p.tile_m - 1) / p.tile_m;
    Logits l{};
    const Matrix x{work + p.x + (uint64_t)row0 * up(s->width * sizeof(T), 64), panel};
    l.w = w, l.x = x, l.rows = s->rows, l.vocab = s->vocab, l.width = p.width;
    l.row0 = row0, l.piece_rows = rows, l.word0 = word0, l.word_tiles = word_tiles;
    l.count = count, l.target = k.target, l.factors = k.factors, l.order = k.order, l.terms = terms, l.g = work + p.g, l.g_rows = p.rows;
    const uint32_t row_tiles = (rows + p.tile_n - 1) / p.tile_n;
    l.blocks = scan_blocks(row_tiles, word_tiles, p.at_once), l.at_once = p.at_once;
    const auto logits = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(scan_grid(row_tiles, word_tiles, p.at_once)), dim3(256), 0, stream, l); };
    bool few = false;
    if constexpr (sizeof(T) == 4) few = few_rows(s);
    if (few) {
      const Few f{s->weight, s->x, s->w_stride, s->x_stride, s->rows, s->vocab, s->width, few_pitch(s), word0, words, nullptr, false, nullptr};
      const FewLogits v{f, count, k.order, k.target, k.factors, work + p.g, p.rows};
      const uint32_t groups = (words + 15) / 16;
      const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(groups < 1024 ? groups : 1024), dim3(256), s->rows * f.pitch, stream, v); };
      if constexpr (sizeof(T) == 4) s->rows <= 16 ? run(head_few_logits<1>) : s->rows <= 32 ? run(head_few_logits<2>) : run(head_few_logits<4>);
    } else {
      with_tiles<T>(s, [&](auto shape) {
        using S = decltype(shape);
        p.lay ? logits(head_logits<T, S, PANELS>) : logits(head_logits<T, S, ROWS>);
      });
    }
    constexpr uint32_t deep = kDeep<T>;
    Product a{};
    const auto product = [&](auto kernel) {
      const uint32_t groups = a.split.groups ? a.split.groups : (a.split.m + p.tile_m - 1) / p.tile_m;
      hipLaunchKernelGGL(kernel, dim3(groups * p.n_tiles), dim3(256), 0, stream, a);
    };
    a.split = {0, 0, row0, count, p.tile_m, p.tile_n, p.n_tiles, 0, false};
    a.a = {work + p.g, panel}, a.n = p.width, a.n_pitch = p.n_pitch, a.slots = (float *)(work + p.slots);
    Ends e{};
    e.deep = deep, e.slots = a.slots, e.n = s->width, e.n_pitch = p.n_pitch;
    if (s->dx) {
      a.split.m = rows, a.split.k = words, a.split.groups = groups_for(p, rows, words, deep);
      a.b = {w.at + (int64_t)word0 * (p.lay ? 64 : w.pitch), w.pitch};
      a.sums = (float *)(work + p.dx) + (uint64_t)(rows_outside ? 0 : row0) * p.n_pitch, a.first = word0 == 0;
      if (p.puts_x) {
        a.to = s->dx, a.n_to = s->width, a.f32 = sizeof(T) == 4;
        a.terms = terms, a.order = k.order, a.target = k.target, a.w = s->weight, a.w_stride = s->w_stride;
      }
      with_tiles<T>(s, [&](auto shape) {
        using S = decltype(shape);
        p.lay ? product(head_product<T, S, false, PANELS>) : product(head_product<T, S, false, ROWS>);
      });
      e.split = a.split, e.sums = a.sums, e.first = a.first, e.last = word_piece + 1 == word_pieces, e.put = p.puts_x, e.rows = rows;
      e.order = k.order, e.target = k.target, e.terms = terms, e.w = s->weight, e.w_stride = s->w_stride, e.to = s->dx;
      if (a.split.groups || (e.last && !e.put)) sums<T>(e, stream);
    }
    if (s->dweight) {
      a.split.m = words, a.split.k = rows, a.split.groups = groups_for(p, words, rows, deep), a.split.dw = true;
      a.b = x;
      a.sums = (float *)(work + p.dw) + (uint64_t)(rows_outside ? word0 : 0) * p.n_pitch, a.first = row0 == 0;
      a.to = nullptr, a.terms = nullptr;
      const bool last = row_piece + 1 == row_pieces, f32 = s->dweight_dtype == UOR_TRUNK_F32;
      void *to = (char *)s->dweight + (uint64_t)word0 * s->width * size_of(s->dweight_dtype);
      if (kTerms && last) {
        t.word0 = word0, t.words = words, t.to = work + p.word_terms, t.present = k.present + word0;
        if (s->rows <= kFewTerms)
          hipLaunchKernelGGL((head_terms<T>), dim3(s->rows, (s->width + 511) / 512), dim3(64), 0, stream, t, s->targets, s->wide != 0, s->vocab);
        else sum_rows<float, T>(t, stream);
      }
      if (p.puts_w) {
        a.to = to, a.words = words, a.n_to = s->width, a.f32 = f32;
        if (kTerms) a.present = t.present, a.terms = (const float *)t.to;
      }
      with_tiles<T>(s, [&](auto shape) { product(head_product<T, decltype(shape), true, PANELS>); });
      e.split = a.split, e.sums = a.sums, e.first = a.first, e.last = last, e.put = p.puts_w, e.rows = words;
      e.order = nullptr, e.terms = nullptr, e.to = to;
      if (kTerms && last) e.present = t.present, e.word_terms = (const float *)t.to;
      if (a.split.groups || (last && !e.put)) f32 ? sums<float>(e, stream) : sums<bf16>(e, stream);
    }
  }
  return launched();
}

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" uint64_t uor_trunk_loss_backward_workspace_bytes(const uor_trunk_head_args *s) { return check_head(s) || !s->rows ? 0 : grad_plan(s).bytes; }

extern "C" int uor_trunk_loss_backward_async(const uor_trunk_head_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_head(s)) return e;
  if (s->dweight_dtype > UOR_TRUNK_F32) return fail(-1, "dweight_dtype %u is neither bf16 nor f32", s->dweight_dtype);
  if (s->rows && (!s->targets || !s->lse)) return fail(-1, "null targets or lse");
  if (!s->dx && !s->dweight) return 0;
  if (!s->rows) {
    if (!s->dweight) return 0;
    const OnDevice on(s->device);
    if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
    const uint64_t n = (uint64_t)s->vocab * s->width;
    if (s->dweight_dtype == UOR_TRUNK_BF16)
      hipLaunchKernelGGL((head_nothing<bf16>), dim3(2048), dim3(256), 0, (hipStream_t)stream, (bf16 *)s->dweight, n);
    else
      hipLaunchKernelGGL((head_nothing<float>), dim3(2048), dim3(256), 0, (hipStream_t)stream, (float *)s->dweight, n);
    return launched();
  }
  const uint64_t want = uor_trunk_loss_backward_workspace_bytes(s);
  if (!workspace || bytes < want || (uintptr_t)workspace % 256)
    return fail(-1, "a workspace of %llu bytes, aligned to 256, is wanted", (unsigned long long)want);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? grad<bf16>(s, (char *)workspace, (hipStream_t)stream) : grad<float>(s, (char *)workspace, (hipStream_t)stream);
}
