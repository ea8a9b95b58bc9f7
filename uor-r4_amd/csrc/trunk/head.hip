// head.hip - the head over a vocabulary without keeping its logits: the rows' softmax cross entropy, and
// the largest logit's token with its log probability.
//
//   z_tv = x_t . W_v,  lse_t = log sum_v e^z_tv,  loss_t = lse_t - z_t,target
//   token_t = argmax_v z_tv (the lowest of equals),  logprob_t = z_t,token - lse_t
//
// A block takes 128 rows through some of the vocabulary, 256 words a tile. The words are the result's rows, so
// that a lane has 64 logits of one row of x in registers: their largest, and the sum of 2^(z log2 e - most), are
// kept from tile to tile as a lane's own. Pieces of the vocabulary are joined by a second launch, in their order.
#include "head_pack.h"

namespace trunk {

struct Scan {
  Matrix w, x;
  uint32_t rows, vocab, width;  // width: values of a row, whole 16 bytes
  uint32_t row_tiles, word_tiles, splits;  // in the shape's tiles
  const uint32_t *count;        // how many rows there are, or NULL: `rows`
  const int32_t *target;        // [rows up to 256]
  Sum *parts;                   // [2 splits][rows of row_tiles]
};

// Logits' running softmax; BASE2: `most` is in base 2, see Sum.
template <bool BASE2>
struct Running {
  float most = -3e38f, sum = 0.0f;
  static __device__ __forceinline__ float power(float v) { return exp2_(BASE2 ? v : v * kLog2e); }
  static __device__ __forceinline__ float term(float z, float most) { return BASE2 ? exp2_(fmaf(z, kLog2e, -most)) : power(z - most); }
  static __device__ __forceinline__ float scaled(float z) { return BASE2 ? z * kLog2e : z; }
  __device__ __forceinline__ void join(float most2, float sum2) {
    const float m = fmaxf(most, most2);
    sum = sum * power(most - m) + sum2 * power(most2 - m);
    most = m;
  }
};

template <class T, class S, bool PICK, Lies W>
struct ScanTiles {
  static constexpr Lies kX = PICK ? W : PANELS;
  using Run = Running<sizeof(T) == 2>;
  static constexpr int kStores = 0;
  const Scan &a;
  uint32_t tiles, stages, row0, word0;
  int lane, wave;
  Run run[S::N];
  float value[S::N];
  uint32_t place[S::N];
  int32_t target[S::N];

  template <class FA, class FB>
  __device__ __forceinline__ void feed(uint32_t n, FA &fa, FB &fb) {
    const uint32_t word = word0 + n * S::kM;
    fa.start(a.w.at + (int64_t)word * (W == ROWS ? a.w.pitch : 64), a.w.pitch, a.vocab - word, a.width);
    fb.start(a.x.at + (int64_t)row0 * (kX == ROWS ? a.x.pitch : 64), a.x.pitch, a.rows - row0, a.width);
  }
  __device__ __forceinline__ void take(uint32_t n, f32x16 (&z)[S::M][S::N]) {
    const int half = lane >> 5;
    const uint32_t word = word0 + n * S::kM + 32 * S::M * (wave >> 1);
    if (word + 32 * S::M > a.vocab) cut_rows(z, a.vocab > word ? a.vocab - word : 0, half);  // words that are none
#pragma unroll
    for (int j = 0; j < S::N; j++) {
      float most = z[0][j][0];
#pragma unroll
      for (int i = 0; i < S::M; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) most = fmaxf(most, z[i][j][r]);
      if constexpr (PICK) {
        if (__any(most > value[j])) {  // seldom after the first tiles
          uint32_t at = 0;
#pragma unroll
          for (int i = S::M - 1; i >= 0; i--)
#pragma unroll
            for (int r = 15; r >= 0; r--) at = z[i][j][r] == most ? 32 * i + row_of(r, 0) : at;
          if (most > value[j]) value[j] = most, place[j] = word + at + 4 * half;
        }
      } else {
        const uint32_t at = (uint32_t)target[j] - word;
        if (__any(at < 32 * S::M)) {
          const int own = (int)at - 4 * half;
#pragma unroll
          for (int i = 0; i < S::M; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) value[j] = own == 32 * i + row_of(r, 0) ? z[i][j][r] : value[j];
        }
      }
      const float base = fmaxf(run[j].most, Run::scaled(most));
      float sum[S::M] = {};
#pragma unroll
      for (int i = 0; i < S::M; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) sum[i] += Run::term(z[i][j][r], base);
      run[j].sum = fmaf(run[j].sum, Run::power(run[j].most - base), S::M > 2 ? (sum[0] + sum[1]) + (sum[2] + sum[S::M - 1]) : sum[0] + sum[1]);
      run[j].most = base;
    }
  }
};

// `value` and `place` of two parts of a row: the target's logit, which one of them has at most, or the largest.
template <bool PICK>
__device__ __forceinline__ void join_value(float &value, uint32_t &place, float value2, uint32_t place2) {
  if constexpr (PICK) {
    const bool other = value2 > value || (value2 == value && place2 < place);
    value = other ? value2 : value;
    place = other ? place2 : place;
  } else {
    value += value2;
  }
}

template <class T, class S, bool PICK, Lies W>
__global__ __launch_bounds__(256, S::kBlocks) void head_scan(Scan a) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  uint32_t row_tile, split;
  by_eights(by_xcd(blockIdx.x, gridDim.x), a.row_tiles, a.splits, row_tile, split);
  const uint32_t row0 = row_tile * S::kN;
  if (a.count && row0 >= *a.count) return;
  const uint32_t first = (uint32_t)((uint64_t)a.word_tiles * split / a.splits), end = (uint32_t)((uint64_t)a.word_tiles * (split + 1) / a.splits);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  ScanTiles<T, S, PICK, W> tiles{a, end - first, (a.width + kDeep<T> - 1) / kDeep<T>, row0, first * S::kM, lane, wave};
#pragma unroll
  for (int j = 0; j < S::N; j++) {
    tiles.value[j] = PICK ? -__builtin_inff() : 0.0f, tiles.place[j] = 0;
    tiles.target[j] = PICK ? -1 : a.target[row0 + 32 * S::N * (wave & 1) + 32 * j + (lane & 31)];
  }
  run_tiles<T, S, true, W, true, tiles.kX>(lds, tiles);
#pragma unroll
  for (int j = 0; j < S::N; j++) {
    auto run = tiles.run[j];
    run.join(__shfl_xor(run.most, 32), __shfl_xor(run.sum, 32));
    float value = tiles.value[j];
    uint32_t place = tiles.place[j];
    join_value<PICK>(value, place, __shfl_xor(value, 32), __shfl_xor(place, 32));
    if (lane < 32)
      a.parts[(uint64_t)(2 * split + (wave >> 1)) * (a.row_tiles * S::kN) + row0 + 32 * S::N * (wave & 1) + 32 * j + lane] =
          Sum{run.most, run.sum, value, place};
  }
}

// Few rows: bound by the matrix, which is read once, past LDS. A block takes 16 words at a time, its four wavefronts a
// quarter of their values each (every fourth 64 bytes), so that a narrow vocabulary's long rows are not one
// wavefront's chain; the rows of x lie in LDS. The quarters meet in LDS, and a thread then has the logit of one
// word for one row of each tile of 16 rows.
struct Few {
  const void *w, *x;
  int64_t w_stride, x_stride;   // values
  uint32_t rows, vocab, width, pitch;  // pitch: bytes of a row of x in LDS
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

template <class T, bool PICK, int TILES>
__global__ __launch_bounds__(256) void head_few(Few a) {
  extern __shared__ char x[];
  __shared__ float quarters[2][4][TILES][16 * kFewPad];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t pieces = (a.width + kDeep<T> - 1) / kDeep<T> * 4;
  for (uint32_t i = threadIdx.x; i < a.rows * pieces; i += 256)
    *(Part<T> *)(x + i / pieces * a.pitch + i % pieces * 16) =
        load_some<T, kVec<T>>((const T *)a.x + (int64_t)(i / pieces) * a.x_stride, true, i % pieces * kVec<T>, a.width);
  __syncthreads();
  const uint32_t i16 = lane & 15, chunk = lane >> 4, full = a.width / kDeep<T>;  // stretches of 64 bytes that a row has whole
  const char *xs[TILES];
#pragma unroll
  for (int j = 0; j < TILES; j++) xs[j] = x + (16 * j + i16 < a.rows ? 16 * j + i16 : 0) * a.pitch + chunk * 16;
  using Run = Running<false>;
  Run run[TILES];
  float value[TILES];
  uint32_t place[TILES];
  int64_t target[TILES];
#pragma unroll
  for (int j = 0; j < TILES; j++) {
    const uint32_t row = 16 * j + threadIdx.x % 16;
    value[j] = PICK ? -__builtin_inff() : 0.0f, place[j] = ~0u;
    target[j] = !PICK && row < a.rows ? target_of(a.targets, a.wide, row, a.vocab) : -1;
  }
  uint32_t buffer = 0;
  for (uint32_t g = blockIdx.x; g * 16 < a.vocab; g += gridDim.x, buffer ^= 1) {
    const uint32_t mine = g * 16 + i16 < a.vocab ? g * 16 + i16 : a.vocab - 1;
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
    const uint32_t at = threadIdx.x / 16 * kFewPad + threadIdx.x % 16, word = g * 16 + threadIdx.x / 16;
#pragma unroll
    for (int j = 0; j < TILES; j++) {
      float z = (quarters[buffer][0][j][at] + quarters[buffer][1][j][at]) + (quarters[buffer][2][j][at] + quarters[buffer][3][j][at]);
      if (word >= a.vocab) z = -__builtin_inff();
      if constexpr (PICK) {
        if (z > value[j]) value[j] = z, place[j] = word;
      } else {
        if ((int64_t)word == target[j]) value[j] = z;
      }
      const float base = fmaxf(run[j].most, z);
      run[j].sum = fmaf(run[j].sum, Run::power(run[j].most - base), Run::term(z, base));
      run[j].most = base;
    }
  }
  __shared__ Sum joined[4][16];
#pragma unroll
  for (int j = 0; j < TILES; j++) {
#pragma unroll
    for (int k = 16; k < 64; k <<= 1) {
      run[j].join(__shfl_xor(run[j].most, k), __shfl_xor(run[j].sum, k));
      join_value<PICK>(value[j], place[j], __shfl_xor(value[j], k), __shfl_xor(place[j], k));
    }
    __syncthreads();
    if (lane < 16) joined[wave][lane] = Sum{run[j].most, run[j].sum, value[j], place[j]};
    __syncthreads();
    if (threadIdx.x < 16 && 16 * j + threadIdx.x < a.rows) {
      for (int w = 1; w < 4; w++) {
        const Sum p = joined[w][threadIdx.x];
        run[j].join(p.most, p.sum);
        join_value<PICK>(value[j], place[j], p.value, p.place);
      }
      a.parts[(uint64_t)blockIdx.x * a.rows + 16 * j + threadIdx.x] = Sum{run[j].most, run[j].sum, value[j], place[j]};
    }
  }
}

// WAVES wavefronts join a row's parts, which are `across` apart.
template <bool PICK, int WAVES, bool BASE2>
__global__ __launch_bounds__(256) void head_join(const Sum *parts, uint32_t n, uint32_t across, uint32_t rows, const uint32_t *count,
                                                 const int32_t *order, const void *targets, bool wide, uint32_t vocab, float *losses, float *lse,
                                                 int64_t *tokens, float *logprobs) {
  __shared__ Sum joined[4];
  const uint32_t row = blockIdx.x * (4 / WAVES) + threadIdx.x / (64 * WAVES), lane = threadIdx.x % (64 * WAVES);
  if (row >= (count ? *count : rows)) return;  // with WAVES of 4: all of the block
  Running<BASE2> run;
  float value = PICK ? -__builtin_inff() : 0.0f;
  uint32_t place = PICK ? ~0u : 0;
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += 64 * WAVES) {
    const Sum p = parts[(uint64_t)i * across + row];
    run.join(p.most, p.sum);
    join_value<PICK>(value, place, p.value, p.place);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    run.join(__shfl_xor(run.most, k), __shfl_xor(run.sum, k));
    join_value<PICK>(value, place, __shfl_xor(value, k), __shfl_xor(place, k));
  }
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) joined[threadIdx.x >> 6] = Sum{run.most, run.sum, value, place};
    __syncthreads();
    for (int w = 1; w < WAVES; w++) {
      run.join(joined[w].most, joined[w].sum);
      join_value<PICK>(value, place, joined[w].value, joined[w].place);
    }
  }
  if (lane) return;
  const double most = BASE2 ? (double)run.most * kLn2 : (double)run.most, rest = log((double)run.sum);
  if constexpr (PICK) {
    tokens[row] = place == ~0u ? 0 : place;
    logprobs[row] = (float)((double)value - most - rest);
  } else {
    // Packed rows have a target; others may have none.
    const uint32_t at = order ? (uint32_t)order[row] : row;
    const bool there = order || target_of(targets, wide, row, vocab) >= 0;
    lse[at] = there ? (float)(most + rest) : 0.0f;
    losses[at] = there ? (float)(most - (double)value + rest) : 0.0f;
  }
}

namespace {


// Parts of the vocabulary that blocks take by themselves. The card takes 512 blocks of large tiles at once (1,024 of
// small ones). Four times as many even out; but a block of few tiles spends its time on its first loads, so a part
// has four tiles at least where that leaves no compute unit idle.
uint32_t splits_of(uint32_t row_tiles, uint32_t word_tiles, uint32_t at_once) {
  const uint32_t even = (4 * at_once + row_tiles - 1) / row_tiles, fill = (at_once + row_tiles - 1) / row_tiles;
  const uint32_t most = fill > word_tiles / 4 ? fill : word_tiles / 4, n = even < most ? even : most;
  return n < 1 ? 1 : n < word_tiles ? n : word_tiles;
}

// Bytes of a row of x in LDS: 16 more than its stretches, so that 16 rows' pieces lie in different banks.
uint32_t few_pitch(const uor_trunk_head_args *s) { return (uint32_t)up(s->width * size_of(s->dtype), 64) + 16; }
// Whether a call's rows are few. In 32 bits they are up to 64 that fit into LDS: tiles of 64 rows spend their matrix
// instructions on rows that are none (1 row over 131,072 words of 512: 57 us, in tiles 135). In bf16 tiles read the matrix
// as fast (16 rows over 131,072 words of 512: 35 us, 39 here), unless they leave compute units idle (over 4,550 of
// 1,536: 18 and 15) or have to lay it out first (over 5,000 of 100: 20 and 14).
bool few_rows(const uor_trunk_head_args *s) {
  if (s->rows > 64 || s->rows * few_pitch(s) > 122880) return false;
  return s->dtype == UOR_TRUNK_F32 || s->vocab <= 16384 || !as_it_lies(s->weight, s->w_stride, s->vocab, s->width, s->dtype);
}

// Where a call's scratch memory has what.
struct Plan {
  bool lay, small;  // the matrix is laid out anew; small tiles
  uint32_t few;  // blocks of the few rows' kernel, or 0
  uint32_t width, row_tiles, word_tiles, splits;
  uint64_t parts, w, x, order, target, counts, count, bytes;
};
Plan plan_of(const uor_trunk_head_args *s, bool pick) {
  Plan p{};
  const uint32_t size = size_of(s->dtype);
  if (few_rows(s)) {
    const uint32_t groups = (s->vocab + 15) / 16;
    p.few = groups < 1024 ? groups : 1024;
    p.bytes = up((uint64_t)p.few * s->rows * sizeof(Sum), 256);
    return p;
  }
  p.width = (uint32_t)up(s->width, 16 / size);
  p.lay = pick ? !as_it_lies(s->weight, s->w_stride, s->vocab, s->width, s->dtype) ||
                     !as_it_lies(s->x, s->x_stride, s->rows, s->width, s->dtype)
               : laid_out(s);
  p.small = small_tiles(s);
  const uint32_t n = p.small ? Small::kN : Large::kN, m = p.small ? Small::kM : Large::kM;
  p.row_tiles = (s->rows + n - 1) / n;
  p.word_tiles = (s->vocab + m - 1) / m;
  p.splits = splits_of(p.row_tiles, p.word_tiles, p.small ? 1024 : 512);
  Scratch at;
  const uint64_t rows = up(s->rows, kRound);
  p.parts = at.take(2ull * p.splits * p.row_tiles * n * sizeof(Sum));
  p.w = at.take(p.lay ? s->vocab * up(s->width * size, 64) : 0);
  p.x = at.take(pick && !p.lay ? 0 : rows * up(s->width * size, 64));
  p.order = at.take(pick ? 0 : rows * 4);
  p.target = at.take(pick ? 0 : rows * 4);
  p.counts = at.take(pick ? 0 : (s->rows + kPackRows - 1) / kPackRows * 4);
  p.count = at.take(pick ? 0 : 4);
  p.bytes = at.bytes;
  return p;
}

template <class T, bool PICK>
int scan(const uor_trunk_head_args *s, char *work, hipStream_t stream) {
  const Plan p = plan_of(s, PICK);
  const auto join = [&](auto kernel, uint32_t each, const Sum *parts, uint32_t n, uint32_t across, const uint32_t *count) {
    hipLaunchKernelGGL(kernel, dim3((s->rows + each - 1) / each), dim3(256), 0, stream, parts, n, across, s->rows, count,
                       PICK || p.few ? nullptr : (const int32_t *)(work + p.order), s->targets, s->wide != 0, s->vocab, s->losses, s->lse, s->tokens,
                       s->logprobs);
  };
  if (p.few) {
    const Few f{s->weight, s->x, s->w_stride, s->x_stride, s->rows, s->vocab, s->width, few_pitch(s), s->targets, s->wide != 0, (Sum *)work};
    const uint32_t lds = s->rows * f.pitch;
    if (s->rows <= 16) hipLaunchKernelGGL((head_few<T, PICK, 1>), dim3(p.few), dim3(256), lds, stream, f);
    else if (s->rows <= 32) hipLaunchKernelGGL((head_few<T, PICK, 2>), dim3(p.few), dim3(256), lds, stream, f);
    else hipLaunchKernelGGL((head_few<T, PICK, 4>), dim3(p.few), dim3(256), lds, stream, f);
    join(head_join<PICK, 4, false>, 1, f.parts, p.few, s->rows, nullptr);
    return launched();
  }
  Scan a{};
  a.rows = s->rows, a.vocab = s->vocab, a.width = p.width;
  a.row_tiles = p.row_tiles, a.word_tiles = p.word_tiles, a.splits = p.splits;
  a.parts = (Sum *)(work + p.parts);
  a.w = {(const char *)s->weight, s->w_stride * (int64_t)sizeof(T)};
  if (p.lay) a.w = lay<T>(s->weight, s->w_stride, s->vocab, s->width, work + p.w, stream);
  if constexpr (PICK) {
    if (p.lay) a.x = lay<T>(s->x, s->x_stride, s->rows, s->width, work + p.x, stream);
    else a.x = {(const char *)s->x, s->x_stride * (int64_t)sizeof(T)};
  } else {
    Pack k{};
    k.rows = s->rows, k.width = s->width, k.vocab = s->vocab, k.piece = (uint32_t)up(s->rows, kRound), k.stride = s->x_stride;
    a.x = {work + p.x, (int64_t)k.piece * 64};
    k.x = s->x, k.targets = s->targets, k.wide = s->wide != 0;
    k.to = work + p.x, k.order = (int32_t *)(work + p.order), k.target = (int32_t *)(work + p.target);
    k.count = (uint32_t *)(work + p.count), k.losses = s->losses, k.lse = s->lse;
    pack<T, false>(k, (uint32_t *)(work + p.counts), stream);
    a.count = k.count, a.target = k.target;
  }
  const dim3 grid(p.row_tiles * p.splits);
  const uint32_t across = p.row_tiles * (p.small ? Small::kN : Large::kN);
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a); };
  if (p.small) p.lay ? run(head_scan<T, Small, PICK, PANELS>) : run(head_scan<T, Small, PICK, ROWS>);
  else if constexpr (sizeof(T) == 2) p.lay ? run(head_scan<T, Large, PICK, PANELS>) : run(head_scan<T, Large, PICK, ROWS>);
  constexpr bool kBase2 = sizeof(T) == 2;
  if (p.splits > 64) join(head_join<PICK, 4, kBase2>, 1, a.parts, 2 * p.splits, across, a.count);
  else join(head_join<PICK, 1, kBase2>, 4, a.parts, 2 * p.splits, across, a.count);
  return launched();
}

template <bool PICK>
int scan(const uor_trunk_head_args *s, void *workspace, uint64_t bytes, void *stream) {
  const uint64_t want = plan_of(s, PICK).bytes;
  if (!workspace || bytes < want || (uintptr_t)workspace % 256)
    return fail(-1, "a workspace of %llu bytes, aligned to 256, is wanted", (unsigned long long)want);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? scan<bf16, PICK>(s, (char *)workspace, (hipStream_t)stream)
                                    : scan<float, PICK>(s, (char *)workspace, (hipStream_t)stream);
}

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" uint64_t uor_trunk_sizeof_head(void) { return sizeof(uor_trunk_head_args); }

extern "C" uint64_t uor_trunk_loss_workspace_bytes(const uor_trunk_head_args *s) { return check_head(s) || !s->rows ? 0 : plan_of(s, false).bytes; }

extern "C" int uor_trunk_loss_async(const uor_trunk_head_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_head(s)) return e;
  if (!s->rows) return 0;
  if (!s->targets || !s->losses || !s->lse) return fail(-1, "null targets, losses or lse");
  return scan<false>(s, workspace, bytes, stream);
}

extern "C" uint64_t uor_trunk_choose_workspace_bytes(const uor_trunk_head_args *s) { return check_head(s) || !s->rows ? 0 : plan_of(s, true).bytes; }

extern "C" int uor_trunk_choose_async(const uor_trunk_head_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_head(s)) return e;
  if (!s->rows) return 0;
  if (!s->tokens || !s->logprobs) return fail(-1, "null tokens or logprobs");
  return scan<true>(s, workspace, bytes, stream);
}
