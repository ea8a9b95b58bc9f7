// conv.hip - the short causal convolution of each channel over its sequence's last rows: over
// packed sequences, its gradient, and for single tokens over device slots.
//
// Bound by its rows, read once and written once. A thread walks down a run of rows with eight
// channels (16 bytes of bf16) and the rows before it in registers; a batch of rows is read before the
// first is used. 300 bf16 prompts of up to 509 by 640 channels: 52 us, 3.7 TB/s; a row at a time 103.
// The gradient holds sums, gradients and rows of four channels, three wavefronts a SIMD; it reads a
// batch ahead, and rows in a run's middle ask nothing row by row, so that no store is waited for:
// 2,048 sequences of 128 take 258 us, 3.9 TB/s; with eight channels, in blocks of 512 threads, 390
// where four took 307, without the middle 354.
#include "trunk.h"

#include <type_traits>

namespace trunk {

// Rows of a thread's run: the rows before it are read twice, and a gradient computes those after it
// twice. Shorter runs fill the card sooner.
constexpr uint32_t kRun = 16, kGradRun = 32;
constexpr int kBatch = 4, kRowBatch = 8;  // rows that are read together, in a gradient and without
// A gradient's registers leave a SIMD three wavefronts, twelve a compute unit: one block of 768 threads,
// and no more blocks than compute units, so that all begin at once: 258 us; 768 blocks 279, 512 threads
// (one block still) 299, 384 (two, a sixth of the lanes idle) 379, 1,024 (128 registers a thread) 387: 2,048
// bf16 sequences of 128 by 640 channels, the only number of channels that was timed. Others may leave more
// lanes idle: a third of them at 2,048 channels, 42 of a hundred at 1,792.
constexpr uint32_t kGradThreads = 768, kMostGradBlocks = 256;

struct Conv {
  Rows rows;
  uint32_t channels, pieces, slots;
  int64_t x_stride, y_stride;
  const void *x;
  const float *weight, *bias;
  const void *initial;
  void *y, *final;
  const int32_t *index;
  void *states;
  const void *dy, *dfinal;
  void *dx, *dinitial;
  float *parts;      // [blocks][TAPS + 1][channels]: sums of a block's runs
  uint32_t workers;  // lines of the grid
  bool silu;
};

// A thread's E channels of a row: eight, or in a gradient, which holds more of them, four. WIDE: all
// rows are whole pieces of eight channels, aligned to 16 bytes.
template <class T, int E>
using Raw = __attribute__((ext_vector_type(E))) T;
template <int E>
using Some = __attribute__((ext_vector_type(E))) float;

template <class T, bool WIDE, int E>
__device__ __forceinline__ void put_some(T *row, uint32_t col, uint32_t cols, Some<E> v) {
  const Raw<T, E> o = __builtin_convertvector(v, Raw<T, E>);
  if constexpr (WIDE) {
    *(Raw<T, E> *)(row + col) = o;
  } else {
    store_some<T, E>(row, col, cols, o);
  }
}
template <class T, bool WIDE, int E>
__device__ __forceinline__ Raw<T, E> raw_some(const void *base, int64_t at, uint32_t col, uint32_t cols) {
  const T *row = (const T *)base + at;
  if constexpr (WIDE) return *(const Raw<T, E> *)(row + col);
  else return load_some<T, E>(row, true, col, cols);
}
template <class T, bool WIDE, int E>
__device__ __forceinline__ Some<E> row_some(const void *base, int64_t at, uint32_t col, uint32_t cols) {
  return __builtin_convertvector(raw_some<T, WIDE, E>(base, at, col, cols), Some<E>);
}
// A block's threads: `lines` runs by the channels' pieces of E, or one run by THREADS of them.
struct Lane {
  uint32_t line, run, c;
};
template <int E, uint32_t THREADS>
__host__ __device__ __forceinline__ uint32_t lines_of(uint32_t channels) {
  const uint32_t groups = (channels + E - 1) / E;
  return groups > THREADS ? 1 : THREADS / groups;
}
template <int E, uint32_t THREADS>
__host__ __device__ __forceinline__ uint32_t parts_of(uint32_t channels) {
  return ((channels + E - 1) / E + THREADS - 1) / THREADS;
}
template <int E, uint32_t THREADS>
__device__ __forceinline__ bool lane_of(const Conv &a, Lane &l) {
  const uint32_t groups = (a.channels + E - 1) / E, parts = parts_of<E, THREADS>(a.channels), lines = lines_of<E, THREADS>(a.channels);
  const uint32_t thread = blockIdx.x % parts * THREADS + threadIdx.x;
  l.line = parts > 1 ? 0 : thread / groups, l.run = blockIdx.x / parts * lines + l.line;
  l.c = (parts > 1 ? thread : thread % groups) * E;
  return l.line < lines && l.c < a.channels;
}
template <int TAPS, bool WIDE, int E>
__device__ __forceinline__ void taps_of(const Conv &a, uint32_t c, Some<E> (&w)[TAPS], Some<E> &bias) {
  // A channel's taps are next to each other; whole pieces ask for no channel that is not there.
#pragma unroll
  for (int e = 0; e < E; e++) {
    Some<TAPS> taps = 0.0f;
    if (WIDE || c + e < a.channels) taps = loose<float, TAPS>(a.weight + (uint64_t)(c + e) * TAPS);
#pragma unroll
    for (int k = 0; k < TAPS; k++) w[k][e] = taps[k];
  }
  bias = a.bias ? load_some<float, E>(a.bias, true, c, a.channels) : Some<E>(0.0f);
}
// Row `first - TAPS + 1 + k` of the sequence for each k < TAPS - 1: its own, or one before it.
template <class T, int TAPS, bool WIDE, int E>
__device__ __forceinline__ void rows_before(const Conv &a, const Piece &at, uint32_t c, Some<E> *window) {
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) {
    const int64_t row = (int64_t)at.first - (TAPS - 1) + k, back = row - at.start;
    window[k] = Some<E>(0.0f);
    if (back >= 0) window[k] = row_some<T, WIDE, E>(a.x, row * a.x_stride, c, a.channels);
    else if (a.initial)
      window[k] = row_some<T, WIDE, E>(a.initial, ((int64_t)at.seq * (TAPS - 1) + (TAPS - 1) + back) * a.channels, c, a.channels);
  }
}
// bias + sum of w[k] rows[k]: the rows before the one that is last.
template <int TAPS, int E>
__device__ __forceinline__ Some<E> weighted(const Some<E> *rows, const Some<E> (&w)[TAPS], const Some<E> &bias) {
  Some<E> v = bias;
#pragma unroll
  for (int k = 0; k < TAPS; k++) v = __builtin_elementwise_fma(rows[k], w[k], v);  // one rounding in every form
  return v;
}
template <class T, int E>
__device__ __forceinline__ Some<E> silu(Some<E> v) {
#pragma unroll
  for (int e = 0; e < E; e++) v[e] *= sigmoid_of<T>(v[e]);
  return v;
}

template <class T, int TAPS, bool WIDE>
__global__ __launch_bounds__(256, 3) void conv_rows(Conv a) {
  constexpr int E = 8, kPast = TAPS - 1;
  clear_unowned(a.rows, (T *)a.y, a.y_stride, a.channels);
  Lane l;
  Piece at;
  if (!lane_of<E, 256>(a, l) || l.run >= a.pieces || !piece(a.rows, l.run, kRun, at)) return;
  const uint32_t c = l.c;
  Some<E> w[TAPS], bias, rows[kPast + kRowBatch];
  taps_of<TAPS, WIDE, E>(a, c, w, bias);
  rows_before<T, TAPS, WIDE, E>(a, at, c, rows);
  uint32_t left = 0;  // rows of the last batch
  for (uint32_t first = at.first; first < at.end; first += kRowBatch) {
    left = min(at.end - first, (uint32_t)kRowBatch);
    const T *x = (const T *)a.x + (int64_t)first * a.x_stride;
#pragma unroll
    for (int k = 0; k < kRowBatch; k++) {
      rows[kPast + k] = row_some<T, WIDE, E>(x, 0, c, a.channels);
      x += first + k + 1 < at.end ? a.x_stride : 0;  // rows past the last are read as the last
    }
#pragma unroll
    for (int k = 0; k < kRowBatch; k++) {
      Some<E> v = weighted<TAPS, E>(rows + k, w, bias);
      if (a.silu) v = silu<T, E>(v);
      if (k < (int)left) put_some<T, WIDE, E>((T *)a.y + (first + k) * a.y_stride, c, a.channels, v);
    }
    if (first + kRowBatch < at.end) {
#pragma unroll
      for (int k = 0; k < kPast; k++) rows[k] = rows[kRowBatch + k];
    }
  }
  if (a.final && at.end == at.stop) {
#pragma unroll
    for (int k = 0; k < kPast; k++) {
      Some<E> v = rows[k];
#pragma unroll
      for (int n = 1; n <= kRowBatch; n++) v = left == (uint32_t)n ? rows[k + n] : v;
      put_some<T, WIDE, E>((T *)a.final + ((int64_t)at.seq * kPast + k) * a.channels, c, a.channels, v);
    }
  }
}

// dx of a row needs the gradients before the activation of the TAPS - 1 rows after it: a run goes
// that far past its end, and dx follows TAPS - 1 rows behind. The parameters' sums take a run's own
// rows; a line's runs are fixed, and a block's lines are joined in their order, so that all sums
// have one order.
template <class T, int TAPS, bool WIDE>
__global__ __launch_bounds__(kGradThreads, 3) void conv_grad_rows(Conv a) {
  constexpr int E = 4, kPast = TAPS - 1;
  __shared__ float joined[kGradThreads * E];
  clear_unowned(a.rows, (T *)a.dx, a.channels, a.channels);
  Lane l;
  const bool there = lane_of<E, kGradThreads>(a, l);
  const uint32_t c = l.c;
  Some<E> sums[TAPS + 1];
#pragma unroll
  for (int k = 0; k <= TAPS; k++) sums[k] = Some<E>(0.0f);
  if (there) {
    Some<E> w[TAPS], bias;
    taps_of<TAPS, WIDE, E>(a, c, w, bias);
    for (uint32_t number = l.run; number < a.pieces; number += a.workers) {
      Piece at;
      if (!piece(a.rows, number, kGradRun, at)) continue;
      // rows[kPast + k] and d[kPast + k]: of row first + k, and before them those of the rows before.
      Some<E> rows[kPast + kBatch], d[kPast + kBatch];
      rows_before<T, TAPS, WIDE, E>(a, at, c, rows);
#pragma unroll
      for (int k = 0; k < kPast; k++) d[k] = Some<E>(0.0f);
      // A sequence's first run emits the rows before the sequence too.
      const int64_t emit = at.number ? at.first : (int64_t)at.start - kPast;
      const uint32_t last = at.end + kPast;  // a run of no rows still has the rows before
      Raw<T, E> xs[kBatch], gs[kBatch], next_x[kBatch], next_g[kBatch];
      const auto fetch = [&](uint32_t first) {  // a batch ahead; rows past the last are read as the last, and not used
        const uint32_t most = at.stop - 1, from = min(first, most);
        const T *x = (const T *)a.x + (int64_t)from * a.x_stride, *g = (const T *)a.dy + (int64_t)from * a.y_stride;
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
          next_x[k] = raw_some<T, WIDE, E>(x, 0, c, a.channels);
          next_g[k] = raw_some<T, WIDE, E>(g, 0, c, a.channels);
          const bool more = first + k < most;
          x += more ? a.x_stride : 0;
          g += more ? a.y_stride : 0;
        }
      };
#pragma unroll
      for (int k = 0; k < kBatch; k++) next_x[k] = next_g[k] = Raw<T, E>((T)0.0f);
      if (at.start != at.stop) fetch(at.first);
      // A batch of rows. EDGE: some may be past the run's last, or before the first that it emits;
      // where none is, nothing is asked row by row, and stores are not waited for.
      const auto batch = [&](uint32_t first, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
        for (int k = 0; k < kBatch; k++) xs[k] = next_x[k], gs[k] = next_g[k];
        if (at.start != at.stop) fetch(first + kBatch);
#pragma unroll
        for (int b = 0; b < kBatch; b++) {
          const uint32_t t = first + b;
          rows[kPast + b] = __builtin_convertvector(xs[b], Some<E>);
          Some<E> g = __builtin_convertvector(gs[b], Some<E>);
          if (a.silu) {
            const Some<E> v = weighted<TAPS, E>(rows + b, w, bias);
#pragma unroll
            for (int e = 0; e < E; e++) {
              const float s = sigmoid_of<T>(v[e]);
              g[e] *= s * fmaf(v[e], 1.0f - s, 1.0f);
            }
          }
          if (EDGE && t >= at.stop) g = Some<E>(0.0f);  // whatever the rows before are
          d[kPast + b] = g;
          if (!EDGE || t < at.end) {
#pragma unroll
            for (int k = 0; k < TAPS; k++) sums[k] = __builtin_elementwise_fma(g, rows[b + k], sums[k]);
            sums[TAPS] += g;
          }
          const int64_t row = (int64_t)t - kPast;
          if (EDGE && (row < emit || t >= last)) continue;
          Some<E> v = d[b] * w[kPast];
#pragma unroll
          for (int k = 1; k < TAPS; k++) v = __builtin_elementwise_fma(d[b + k], w[kPast - k], v);
          if (EDGE) {
            const int64_t back = row - ((int64_t)at.stop - kPast);  // its place among the sequence's last rows
            if (a.dfinal && back >= 0) v += row_some<T, WIDE, E>(a.dfinal, ((int64_t)at.seq * kPast + back) * a.channels, c, a.channels);
            if (row < (int64_t)at.start) {
              const int64_t k = row - at.start + kPast;
              if (a.dinitial) put_some<T, WIDE, E>((T *)a.dinitial + ((int64_t)at.seq * kPast + k) * a.channels, c, a.channels, v);
              continue;
            }
          }
          put_some<T, WIDE, E>((T *)a.dx + row * a.channels, c, a.channels, v);
        }
#pragma unroll
        for (int k = 0; k < kPast; k++) rows[k] = rows[kBatch + k], d[k] = d[kBatch + k];
      };
      // The rows that no batch of the middle may reach past: the run's end, and before the sequence's
      // last rows, which have gradients of their own.
      const int64_t middle = min((int64_t)at.end, (int64_t)at.stop - 1);
      uint32_t first = at.first;
      if (first < last) batch(first, std::true_type{}), first += kBatch;
      for (; first + kBatch <= middle; first += kBatch) batch(first, std::false_type{});
      for (; first < last; first += kBatch) batch(first, std::true_type{});
    }
  }
  // The block's lines side by side.
  const uint32_t parts = parts_of<E, kGradThreads>(a.channels), lines = lines_of<E, kGradThreads>(a.channels);
  const uint32_t groups = (a.channels + E - 1) / E, block = blockIdx.x / parts, c0 = blockIdx.x % parts * kGradThreads * E;
  const uint32_t width = parts > 1 ? kGradThreads * E : groups * E;
#pragma unroll
  for (int k = 0; k <= TAPS; k++) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; e++) joined[threadIdx.x * E + e] = sums[k][e];
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < width && c0 + at < a.channels; at += kGradThreads) {
      float v = 0.0f;
      for (uint32_t line = 0; line < lines; line++) v += joined[line * groups * E + at];
      a.parts[((uint64_t)block * (TAPS + 1) + k) * a.channels + c0 + at] = v;
    }
  }
}

__global__ __launch_bounds__(1024) void conv_grad_sums(const float *parts, uint32_t blocks, uint32_t channels, uint32_t taps,
                                                       float *dweight, float *dbias) {
  sum_columns(parts, blocks, (taps + 1) * channels, [&](uint32_t at, float v) {
    const uint32_t k = at / channels, c = at % channels;
    if (k < taps) dweight[c * taps + k] = v;
    else if (dbias) dbias[c] = v;
  });
}

template <class T, int TAPS, bool WIDE>
__global__ __launch_bounds__(256) void conv_step(Conv a) {
  constexpr int E = 8;
  const uint32_t groups = (a.channels + 7) / 8;
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = (uint32_t)(id / groups), c = (uint32_t)(id % groups) * 8;
  if (row >= a.rows.tokens) return;
  const int64_t slot = a.index ? a.index[row] : (int64_t)row;
  T *y = (T *)a.y + row * a.y_stride;
  if (slot < 0 || slot >= a.slots) {
    put_some<T, WIDE, E>(y, c, a.channels, Some<E>(0.0f));
    return;
  }
  Some<E> w[TAPS], bias, rows[TAPS];
  T *state = (T *)a.states + slot * (TAPS - 1) * a.channels;
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) rows[k] = row_some<T, WIDE, E>(state, (int64_t)k * a.channels, c, a.channels);
  rows[TAPS - 1] = row_some<T, WIDE, E>(a.x, row * a.x_stride, c, a.channels);
  taps_of<TAPS, WIDE, E>(a, c, w, bias);
  Some<E> v = weighted<TAPS, E>(rows, w, bias);
  if (a.silu) v = silu<T, E>(v);
  put_some<T, WIDE, E>(y, c, a.channels, v);
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) put_some<T, WIDE, E>(state + k * a.channels, c, a.channels, rows[k + 1]);
}

namespace {

int check_conv(const uor_trunk_conv_args *s, bool step) {
  if (!s) return fail(-1, "null argument");
  if (s->dtype > UOR_TRUNK_F32) return fail(-1, "dtype %u is neither bf16 nor f32", s->dtype);
  if (s->channels < 1 || s->channels > (1u << 24)) return fail(-1, "%u channels", s->channels);
  if (s->taps < 1 || s->taps > UOR_TRUNK_MAX_TAPS) return fail(-1, "%u taps outside 1..4", s->taps);
  if (s->tokens > 0x7fffffffu - 64) return fail(-1, "%u rows: too many", s->tokens);
  if (!step && (s->seqs < 1 || s->seqs > 0x7fffffffu)) return fail(-1, "%u sequences", s->seqs);
  if (!step && !s->offsets && s->seqs != 1) return fail(-1, "%u sequences without offsets", s->seqs);
  if ((s->tokens && !s->x) || !s->weight) return fail(-1, "null rows or weight");
  if (s->tokens > 1 && (s->x_stride < s->channels || s->y_stride < s->channels)) return fail(-1, "rows overlap: a stride is less than a row");
  if (((uint64_t)s->tokens + s->seqs) * ((s->channels + 7) / 8) / 32 > 0x3fffffffu) return fail(-1, "too many rows and channels for one call");
  return 0;
}
Conv conv_of(const uor_trunk_conv_args *s, uint32_t run) {
  Conv a{};
  a.rows = Rows{s->offsets, s->tokens, s->seqs};
  a.channels = s->channels, a.pieces = pieces(s->tokens, s->seqs, run), a.slots = s->slots;
  a.x_stride = s->x_stride, a.y_stride = s->y_stride;
  a.x = s->x, a.weight = s->weight, a.bias = s->bias, a.initial = s->initial, a.y = s->y, a.final = s->final;
  a.index = s->index, a.states = s->states, a.dy = s->dy, a.dfinal = s->dfinal, a.dx = s->dx, a.dinitial = s->dinitial;
  a.silu = s->silu != 0;
  return a;
}
bool wide_of(const uor_trunk_conv_args *s) {
  const uint32_t bytes = s->dtype == UOR_TRUNK_BF16 ? 2 : 4;
  if (s->channels % 8) return false;
  const auto wide = [&](const void *p, int64_t stride) { return aligned16(p, stride, bytes); };
  return wide(s->x, s->x_stride) && wide(s->y, s->y_stride) && wide(s->dy, s->y_stride) && wide(s->initial, 0) && wide(s->final, 0) &&
         wide(s->states, 0) && wide(s->dfinal, 0) && wide(s->dinitial, 0) && wide(s->dx, 0);
}
// The blocks of `runs` runs, and of a gradient: one for each compute unit at most.
uint32_t blocks_of(uint32_t runs, uint32_t channels) {
  const uint32_t lines = lines_of<8, 256>(channels);
  return (runs + lines - 1) / lines * parts_of<8, 256>(channels);
}
uint32_t grad_blocks_of(uint32_t runs, uint32_t channels) {
  const uint32_t lines = lines_of<4, kGradThreads>(channels), parts = parts_of<4, kGradThreads>(channels);
  const uint32_t few = (runs + lines - 1) / lines, most = (kMostGradBlocks + parts - 1) / parts;
  return few < 1 ? 1 : few < most ? few : most;
}
template <template <class, int, bool> class F, class T, bool WIDE, class... V>
int by_taps(uint32_t taps, V... v) {
  switch (taps) {
    case 1: return F<T, 1, WIDE>::run(v...);
    case 2: return F<T, 2, WIDE>::run(v...);
    case 3: return F<T, 3, WIDE>::run(v...);
    default: return F<T, 4, WIDE>::run(v...);
  }
}
template <template <class, int, bool> class F, class... V>
int by_form(const uor_trunk_conv_args *s, V... v) {
  const bool wide = wide_of(s);
  if (s->dtype == UOR_TRUNK_BF16) return wide ? by_taps<F, bf16, true>(s->taps, v...) : by_taps<F, bf16, false>(s->taps, v...);
  return wide ? by_taps<F, float, true>(s->taps, v...) : by_taps<F, float, false>(s->taps, v...);
}
template <class T, int TAPS, bool WIDE>
struct RowsCall {
  static int run(Conv a, hipStream_t stream) {
    hipLaunchKernelGGL((conv_rows<T, TAPS, WIDE>), dim3(blocks_of(a.pieces, a.channels)), dim3(256), 0, stream, a);
    return launched();
  }
};
template <class T, int TAPS, bool WIDE>
struct StepCall {
  static int run(Conv a, hipStream_t stream) {
    const uint64_t threads = (uint64_t)a.rows.tokens * ((a.channels + 7) / 8);
    hipLaunchKernelGGL((conv_step<T, TAPS, WIDE>), dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, stream, a);
    return launched();
  }
};
template <class T, int TAPS, bool WIDE>
struct GradCall {
  static int run(Conv a, uint32_t blocks, float *dweight, float *dbias, hipStream_t stream) {
    const uint32_t parts = parts_of<4, kGradThreads>(a.channels);
    hipLaunchKernelGGL((conv_grad_rows<T, TAPS, WIDE>), dim3(blocks * parts), dim3(kGradThreads), 0, stream, a);
    hipLaunchKernelGGL(conv_grad_sums, dim3((a.channels * (TAPS + 1) + 63) / 64), dim3(1024), 0, stream, a.parts, blocks,
                       a.channels, (uint32_t)TAPS, dweight, dbias);
    return launched();
  }
};

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" int uor_trunk_conv_async(const uor_trunk_conv_args *s, void *stream) {
  if (const int e = check_conv(s, false)) return e;
  if (s->tokens && !s->y) return fail(-1, "null y");
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return by_form<RowsCall>(s, conv_of(s, kRun), (hipStream_t)stream);
}

extern "C" int uor_trunk_conv_step_async(const uor_trunk_conv_args *s, void *stream) {
  if (const int e = check_conv(s, true)) return e;
  if (!s->tokens) return 0;
  if (!s->y || (!s->states && s->taps > 1)) return fail(-1, "null y or states");
  if (!s->index && s->slots < s->tokens) return fail(-1, "%u rows for %u states", s->tokens, s->slots);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return by_form<StepCall>(s, conv_of(s, kRun), (hipStream_t)stream);
}

extern "C" uint64_t uor_trunk_conv_backward_workspace_bytes(const uor_trunk_conv_args *s) {
  if (check_conv(s, false)) return 0;
  return (uint64_t)grad_blocks_of(pieces(s->tokens, s->seqs, kGradRun), s->channels) * (s->taps + 1) * s->channels * sizeof(float);
}

extern "C" int uor_trunk_conv_backward_async(const uor_trunk_conv_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_conv(s, false)) return e;
  if ((s->tokens && (!s->dy || !s->dx)) || !s->dweight) return fail(-1, "null dy, dx or dweight");
  const uint64_t want = uor_trunk_conv_backward_workspace_bytes(s);
  if (!workspace || bytes < want || (uintptr_t)workspace % 16)
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)want);
  Conv a = conv_of(s, kGradRun);
  const uint32_t blocks = grad_blocks_of(a.pieces, s->channels);
  a.workers = blocks * lines_of<4, kGradThreads>(s->channels);
  a.parts = (float *)workspace;
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return by_form<GradCall>(s, a, blocks, s->dweight, s->dbias, (hipStream_t)stream);
}
