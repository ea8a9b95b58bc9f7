// head.hip - the head over a vocabulary without keeping its logits: the rows' softmax cross entropy, and
// the largest logit's token with its log probability.
//
//   z_tv = x_t . W_v,  lse_t = log sum_v e^z_tv,  loss_t = lse_t - z_t,target
//   token_t = argmax_v z_tv (the lowest of equals),  logprob_t = z_t,token - lse_t
//
// A block takes 128 rows through some of the vocabulary, 256 words a tile, and then the next rows. The words are the result's rows, so
// that a lane has 64 logits of one row of x in registers: their largest, and the sum of 2^(z log2 e - most), are
// kept from tile to tile as a lane's own. Parts of a row are joined by a second launch, in their order.
// Shares of blocks are even to a tile: 11,917 of 17,024 rows of 1,609 over 2,479 words 130 us, with shares of rows by shares of
// words, which left the card's last turn two thirds empty, 204.
#include "few.h"

namespace trunk {

struct Scan {
  Matrix w, x;
  uint32_t rows, vocab, width;  // width: values of a row, whole 16 bytes
  uint32_t word_tiles;          // in the shape's tiles
  uint32_t blocks, at_once;     // see RowShares
  const uint32_t *count;        // how many rows there are, or NULL: `rows`
  const int32_t *target;        // [rows up to 256] of packed rows
  const void *targets;          // the caller's, of rows that are not
  bool wide;
  Sum *parts;                   // [group + set][abreast][2][a tile's rows], see RowShares: groups and sets go on together
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

template <class T, class S, bool PICK, Lies W, Lies X>
struct ScanTiles {
  using Run = Running<sizeof(T) == 2>;
  static constexpr int kStores = 0;
  const Scan &a;
  uint32_t tiles;
  Walk ahead, at;
  int lane, wave;
  Run run[S::N];
  float value[S::N];
  uint32_t place[S::N];
  int32_t target[S::N];

  // A row tile's beginning and end.
  __device__ __forceinline__ void open() {
#pragma unroll
    for (int j = 0; j < S::N; j++) {
      run[j] = Run{}, value[j] = PICK ? -__builtin_inff() : 0.0f, place[j] = 0;
      const uint32_t row = at.row * S::kN + 32 * S::N * (wave & 1) + 32 * j + (lane & 31);
      if constexpr (PICK) target[j] = -1;
      else if constexpr (X == PANELS) target[j] = a.target[row];
      else target[j] = row < a.rows ? target_of(a.targets, a.wide, row, a.vocab) : -1;
    }
  }
  __device__ __forceinline__ void close() {
    Sum *to = a.parts + ((uint64_t)(2 * (at.group * at.abreast + at.row) + (wave >> 1))) * S::kN + 32 * S::N * (wave & 1);
#pragma unroll
    for (int j = 0; j < S::N; j++) {
      run[j].join(__shfl_xor(run[j].most, 32), __shfl_xor(run[j].sum, 32));
      join_value<PICK>(value[j], place[j], __shfl_xor(value[j], 32), __shfl_xor(place[j], 32));
      if (lane < 32) to[32 * j + lane] = Sum{run[j].most, run[j].sum, value[j], place[j]};
    }
  }
  __device__ __forceinline__ uint32_t stages(uint32_t) const { return (a.width + kDeep<T> - 1) / kDeep<T>; }
  template <class FA, class FB>
  __device__ __forceinline__ void feed(uint32_t, FA &fa, FB &fb) {
    const uint32_t word = ahead.word * S::kM, row0 = ahead.row * S::kN;
    ahead.next();
    fa.start(a.w.at + (int64_t)word * (W == ROWS ? a.w.pitch : 64), a.w.pitch, a.vocab - word, a.width);
    fb.start(a.x.at + (int64_t)row0 * (X == ROWS ? a.x.pitch : 64), a.x.pitch, a.rows - row0, a.width);
  }
  __device__ __forceinline__ void take(uint32_t n, f32x16 (&z)[S::M][S::N]) {
    const int half = lane >> 5;
    const uint32_t word = at.word * S::kM + 32 * S::M * (wave >> 1);
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
      float total = sum[0];
      if constexpr (S::M >= 2) total += sum[1];
      if constexpr (S::M == 4) total += sum[2] + sum[3];
      run[j].sum = fmaf(run[j].sum, Run::power(run[j].most - base), total);
      run[j].most = base;
    }
    if (at.word + 1 == at.word_tiles || n + 1 == tiles) close();
    if (at.next() && n + 1 < tiles) open();
  }
};

template <class T, class S, bool PICK, Lies W, Lies X>
__global__ __launch_bounds__(256, S::kBlocks) void head_scan(Scan a) {
  __shared__ __attribute__((aligned(1024))) char lds[S::kLdsBytes];
  const uint32_t rows = a.count ? *a.count : a.rows;
  const Walk walk(RowShares(rows, S::kN, a.word_tiles, a.blocks, a.at_once), a.word_tiles, blockIdx.x);
  if (!walk.tiles) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  ScanTiles<T, S, PICK, W, X> tiles{a, walk.tiles, walk, walk, lane, wave};
  tiles.open();
  run_tiles<T, S, true, W, true, X>(lds, tiles);
}

template <class T, bool PICK, int TILES>
__global__ __launch_bounds__(256) void head_few(Few a) {
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
  few_logits<T, TILES>(a, a.rows, nullptr, [&](int j, uint32_t word, float z) {
    if (word >= a.vocab) z = -__builtin_inff();
    if constexpr (PICK) {
      if (z > value[j]) value[j] = z, place[j] = word;
    } else {
      if ((int64_t)word == target[j]) value[j] = z;
    }
    const float base = fmaxf(run[j].most, z);
    run[j].sum = fmaf(run[j].sum, Run::power(run[j].most - base), Run::term(z, base));
    run[j].most = base;
  });
  __shared__ Sum joined[4][16];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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

// LANES threads join a row's parts: of tiles of `tile` rows, see Scan, or (0) of few rows, one a block.
template <bool PICK, int LANES, bool BASE2>
__global__ __launch_bounds__(256) void head_join(const Sum *parts, uint32_t tile, uint32_t word_tiles, uint32_t blocks, uint32_t at_once,
                                                 uint32_t rows, const uint32_t *count, const int32_t *order, const void *targets, bool wide,
                                                 uint32_t vocab, float *losses, float *lse, int64_t *tokens, float *logprobs) {
  __shared__ Sum joined[4];
  const uint32_t row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const uint32_t all = count ? *count : rows;
  if (row >= all) return;  // with 256 lanes: all of the block
  uint32_t n = blocks, across = rows, two = 2 * rows;  // parts, and from one to the next and to the one after
  const Sum *from = parts + row;
  if (tile) {
    const RowShares s(all, tile, word_tiles, blocks, at_once);
    const uint32_t at = row / tile, set = at / s.abreast;
    const uint32_t first = s.of((uint64_t)set * word_tiles), last = s.of((uint64_t)(set + 1) * word_tiles - 1);
    n = 2 * (last - first + 1), across = tile, two = 2 * s.abreast * tile;
    from = parts + (uint64_t)2 * (first * s.abreast + at) * tile + row % tile;
  }
  Running<BASE2> run;
  float value = PICK ? -__builtin_inff() : 0.0f;
  uint32_t place = PICK ? ~0u : 0;
#pragma unroll 4
  for (uint32_t i = lane; i < n; i += LANES) {
    const Sum p = from[(uint64_t)(i >> 1) * two + (i & 1) * across];
    run.join(p.most, p.sum);
    join_value<PICK>(value, place, p.value, p.place);
  }
#pragma unroll
  for (int k = 1; k < (LANES < 64 ? LANES : 64); k <<= 1) {
    run.join(__shfl_xor(run.most, k), __shfl_xor(run.sum, k));
    join_value<PICK>(value, place, __shfl_xor(value, k), __shfl_xor(place, k));
  }
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) joined[threadIdx.x >> 6] = Sum{run.most, run.sum, value, place};
    __syncthreads();
    for (int w = 1; w < LANES / 64; w++) {
      run.join(joined[w].most, joined[w].sum);
      join_value<PICK>(value, place, joined[w].value, joined[w].place);
    }
  }
  if (lane) return;
  const double most = BASE2 ? (double)run.most / (double)kLog2e : (double)run.most, rest = log((double)run.sum);
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

// Whether a loss takes its rows as they lie, those without a target too, whose results are then dropped: where one tile a block is
// all there is, and its products are too little to be worth the rows' packing. 333 rows of 200 over 4,100 words in 32 bits 16 us,
// packed 19; of 512 over 8,000 43 and, seven in ten without a target, 32; 800 rows of 512 over 8,000 in bf16 20 and 27, or 21 and 17.
bool as_they_are(const uor_trunk_head_args *s, uint64_t tiles, uint32_t at_once) {
  return tiles <= at_once && 2.0 * s->rows * s->vocab * s->width <= (s->dtype == UOR_TRUNK_F32 ? 1.2e9 : 7e9) &&
         as_it_lies(s->x, s->x_stride, s->rows, s->width, s->dtype);
}
// Where a call's scratch memory has what.
struct Plan {
  bool lay;     // the matrix is laid out anew
  bool packed;  // a loss: the rows with a target next to each other
  uint32_t few;  // blocks of the few rows' kernel, or 0
  uint32_t width, tile, word_tiles, at_once, blocks, grid;
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
  const Tiling t = tiling(s);
  p.tile = t.n, p.at_once = t.at_once, p.word_tiles = (s->vocab + t.m - 1) / t.m;
  const uint32_t row_tiles = (s->rows + t.n - 1) / t.n;
  p.blocks = scan_blocks(row_tiles, p.word_tiles, p.at_once), p.grid = scan_grid(row_tiles, p.word_tiles, p.at_once);
  Scratch at;
  const uint64_t rows = up(s->rows, kRound);
  p.packed = !pick && (p.lay || !as_they_are(s, (uint64_t)row_tiles * p.word_tiles, p.at_once));
  p.parts = at.take(2ull * (p.grid + row_tiles) * p.tile * sizeof(Sum));
  p.w = at.take(p.lay ? s->vocab * up(s->width * size, 64) : 0);
  p.x = at.take(p.lay || p.packed ? rows * up(s->width * size, 64) : 0);
  p.order = at.take(p.packed ? rows * 4 : 0);
  p.target = at.take(p.packed ? rows * 4 : 0);
  p.counts = at.take(p.packed ? (s->rows + kPackRows - 1) / kPackRows * 4 : 0);
  p.count = at.take(p.packed ? 4 : 0);
  p.bytes = at.bytes;
  return p;
}

template <class T, bool PICK>
int scan(const uor_trunk_head_args *s, char *work, hipStream_t stream) {
  const Plan p = plan_of(s, PICK);
  const auto join = [&](auto kernel, uint32_t lanes, const Sum *parts, uint32_t blocks, const uint32_t *count) {
    const uint32_t each = 256 / lanes;
    hipLaunchKernelGGL(kernel, dim3((s->rows + each - 1) / each), dim3(256), 0, stream, parts, p.tile, p.word_tiles, blocks, p.at_once, s->rows, count,
                       p.packed ? (const int32_t *)(work + p.order) : nullptr, s->targets, s->wide != 0, s->vocab, s->losses, s->lse, s->tokens,
                       s->logprobs);
  };
  if (p.few) {
    const Few f{s->weight, s->x, s->w_stride, s->x_stride, s->rows, s->vocab, s->width, few_pitch(s), 0, s->vocab, s->targets, s->wide != 0, (Sum *)work};
    const uint32_t lds = s->rows * f.pitch;
    if (s->rows <= 16) hipLaunchKernelGGL((head_few<T, PICK, 1>), dim3(p.few), dim3(256), lds, stream, f);
    else if (s->rows <= 32) hipLaunchKernelGGL((head_few<T, PICK, 2>), dim3(p.few), dim3(256), lds, stream, f);
    else hipLaunchKernelGGL((head_few<T, PICK, 4>), dim3(p.few), dim3(256), lds, stream, f);
    join(head_join<PICK, 256, false>, 256, f.parts, p.few, nullptr);
    return launched();
  }
  Scan a{};
  a.rows = s->rows, a.vocab = s->vocab, a.width = p.width;
  a.word_tiles = p.word_tiles, a.blocks = p.blocks, a.at_once = p.at_once;
  a.parts = (Sum *)(work + p.parts);
  a.w = {(const char *)s->weight, s->w_stride * (int64_t)sizeof(T)};
  if (p.lay) a.w = lay<T>(s->weight, s->w_stride, s->vocab, s->width, work + p.w, stream);
  a.targets = s->targets, a.wide = s->wide != 0;
  if (!p.packed) {
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
  const dim3 grid(p.grid);
  const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a); };
  with_tiles<T>(s, [&](auto shape) {
    using S = decltype(shape);
    constexpr Lies kOther = PICK ? ROWS : PANELS;
    if (p.lay) run(head_scan<T, S, PICK, PANELS, PANELS>);
    else if (PICK || !p.packed) run(head_scan<T, S, PICK, ROWS, ROWS>);
    else run(head_scan<T, S, PICK, ROWS, kOther>);
  });
  constexpr bool kBase2 = sizeof(T) == 2;
  // More than 128 parts a row: by a block. Many rows of few parts: by four threads, which read those of many rows side by side
  // (32,768 rows of 16 to 18 parts: 5 us, by a wavefront 20 to 24).
  const uint32_t row_tiles = (s->rows + p.tile - 1) / p.tile;
  const uint64_t groups = min((uint64_t)p.word_tiles, (uint64_t)p.blocks / row_tiles);
  if (groups > 64) join(head_join<PICK, 256, kBase2>, 256, a.parts, p.blocks, a.count);
  else if (groups > 16 || s->rows < 4096) join(head_join<PICK, 64, kBase2>, 64, a.parts, p.blocks, a.count);
  else join(head_join<PICK, 4, kBase2>, 4, a.parts, p.blocks, a.count);
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
