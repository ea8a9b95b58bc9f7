// conv.hip - the short causal convolution of each channel over its sequence's last rows: over
// packed sequences, its gradient, and for single tokens over device slots.
//
// Bound by its rows, read once and written once. A thread walks down a run of rows with eight
// channels (16 bytes of bf16) and the rows before it in registers.
#include "trunk.h"

namespace trunk {

constexpr uint32_t kRun = 32;  // rows of a thread's run: the rows before it are read twice

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
  float *parts;      // [workers][TAPS + 1][channels]: sums of a worker's runs
  uint32_t workers;
  bool x_wide, y_wide, state_wide, silu;
};

template <class T>
__device__ __forceinline__ void store8(T *row, uint32_t col, uint32_t cols, bool wide, f32x8 v) {
  const V8<T> o = __builtin_convertvector(v, V8<T>);
  if (wide && col + 8 <= cols) {
    *(V8<T> *)(row + col) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (col + e < cols) row[col + e] = o[e];
}
template <class T>
__device__ __forceinline__ f32x8 row8(const void *base, int64_t at, uint32_t col, uint32_t cols, bool wide) {
  return __builtin_convertvector(load8((const T *)base + at, true, col, cols, wide), f32x8);
}
template <int TAPS>
__device__ __forceinline__ void taps_of(const Conv &a, uint32_t c, f32x8 (&w)[TAPS], f32x8 &bias) {
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const bool there = c + e < a.channels;
#pragma unroll
    for (int k = 0; k < TAPS; k++) w[k][e] = there ? a.weight[(c + e) * TAPS + k] : 0.0f;
    bias[e] = there && a.bias ? a.bias[c + e] : 0.0f;
  }
}
// Row `first - TAPS + 1 + k` of the sequence for each k < TAPS - 1: its own, or one before it.
template <class T, int TAPS>
__device__ __forceinline__ void rows_before(const Conv &a, const Piece &at, uint32_t c, f32x8 *window) {
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) {
    const int64_t row = (int64_t)at.first - (TAPS - 1) + k, back = row - at.start;
    window[k] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (back >= 0) window[k] = row8<T>(a.x, row * a.x_stride, c, a.channels, a.x_wide);
    else if (a.initial)
      window[k] = row8<T>(a.initial, ((int64_t)at.seq * (TAPS - 1) + (TAPS - 1) + back) * a.channels, c, a.channels, a.state_wide);
  }
}
template <int TAPS>
__device__ __forceinline__ f32x8 weighted(const f32x8 *window, const f32x8 &x, const f32x8 (&w)[TAPS], const f32x8 &bias) {
  f32x8 v = bias;
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) v += window[k] * w[k];
  return v + x * w[TAPS - 1];
}
template <int TAPS>
__device__ __forceinline__ void shift(f32x8 *window, const f32x8 &x) {
#pragma unroll
  for (int k = 0; k + 2 < TAPS; k++) window[k] = window[k + 1];
  if (TAPS > 1) window[TAPS - 2] = x;
}

template <class T, int TAPS>
__global__ __launch_bounds__(256) void conv_rows(Conv a) {
  const uint32_t groups = (a.channels + 7) / 8;
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t number = (uint32_t)(id / groups), c = (uint32_t)(id % groups) * 8;
  Piece at;
  if (number >= a.pieces || !piece(a.rows, number, kRun, at)) return;
  f32x8 w[TAPS], bias, window[TAPS];
  taps_of<TAPS>(a, c, w, bias);
  rows_before<T, TAPS>(a, at, c, window);
#pragma unroll 4
  for (uint32_t t = at.first; t < at.end; t++) {
    const f32x8 x = row8<T>(a.x, t * a.x_stride, c, a.channels, a.x_wide);
    f32x8 v = weighted<TAPS>(window, x, w, bias);
    shift<TAPS>(window, x);
    if (a.silu) {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= sigmoid(v[e]);
    }
    store8((T *)a.y + t * a.y_stride, c, a.channels, a.y_wide, v);
  }
  if (a.final && at.end == at.stop) {
#pragma unroll
    for (int k = 0; k < TAPS - 1; k++)
      store8((T *)a.final + ((int64_t)at.seq * (TAPS - 1) + k) * a.channels, c, a.channels, a.state_wide, window[k]);
  }
}

// dx of a row needs the gradients before the activation of the TAPS - 1 rows after it: a run goes
// that far past its end, and dx follows TAPS - 1 rows behind. The parameters' sums take a run's own
// rows; a worker's runs are fixed, so that its sums have one order.
template <class T, int TAPS>
__global__ __launch_bounds__(256) void conv_grad_rows(Conv a) {
  const uint32_t groups = (a.channels + 7) / 8;
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t worker = (uint32_t)(id / groups), c = (uint32_t)(id % groups) * 8;
  if (worker >= a.workers) return;
  f32x8 w[TAPS], bias, sums[TAPS + 1];
  taps_of<TAPS>(a, c, w, bias);
#pragma unroll
  for (int k = 0; k <= TAPS; k++) sums[k] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
  for (uint32_t number = worker; number < a.pieces; number += a.workers) {
    Piece at;
    if (!piece(a.rows, number, kRun, at)) continue;
    f32x8 window[TAPS], d[TAPS];  // the rows before t; the gradients at rows t - TAPS + 1 .. t
    rows_before<T, TAPS>(a, at, c, window);
#pragma unroll
    for (int k = 0; k < TAPS; k++) d[k] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
    // A sequence's first run emits the rows before the sequence too.
    const int64_t emit = at.number ? at.first : (int64_t)at.start - (TAPS - 1);
#pragma unroll 2
    for (int64_t t = at.first; t < (int64_t)at.end + TAPS - 1; t++) {
#pragma unroll
      for (int k = 0; k + 1 < TAPS; k++) d[k] = d[k + 1];
      d[TAPS - 1] = f32x8{0, 0, 0, 0, 0, 0, 0, 0};
      if (t < at.stop) {
        const f32x8 x = row8<T>(a.x, t * a.x_stride, c, a.channels, a.x_wide);
        f32x8 g = row8<T>(a.dy, t * a.y_stride, c, a.channels, a.y_wide);
        if (a.silu) {
          const f32x8 v = weighted<TAPS>(window, x, w, bias);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float s = sigmoid(v[e]);
            g[e] *= s * (1.0f + v[e] * (1.0f - s));
          }
        }
        d[TAPS - 1] = g;
        if (t < at.end) {
#pragma unroll
          for (int k = 0; k < TAPS - 1; k++) sums[k] += g * window[k];
          sums[TAPS - 1] += g * x;
          sums[TAPS] += g;
        }
        shift<TAPS>(window, x);
      }
      const int64_t row = t - (TAPS - 1);
      if (row < emit) continue;
      f32x8 v = d[0] * w[TAPS - 1];
#pragma unroll
      for (int k = 1; k < TAPS; k++) v += d[k] * w[TAPS - 1 - k];
      const int64_t last = row - ((int64_t)at.stop - (TAPS - 1));  // its place among the sequence's last rows
      if (a.dfinal && last >= 0)
        v += row8<T>(a.dfinal, ((int64_t)at.seq * (TAPS - 1) + last) * a.channels, c, a.channels, a.state_wide);
      if (row >= (int64_t)at.start) {
        store8((T *)a.dx + row * a.channels, c, a.channels, a.state_wide, v);
      } else if (a.dinitial) {
        const int64_t k = row - at.start + TAPS - 1;
        store8((T *)a.dinitial + ((int64_t)at.seq * (TAPS - 1) + k) * a.channels, c, a.channels, a.state_wide, v);
      }
    }
  }
#pragma unroll
  for (int k = 0; k <= TAPS; k++)
    store8(a.parts + ((uint64_t)worker * (TAPS + 1) + k) * a.channels, c, a.channels, a.channels % 4 == 0, sums[k]);
}

// The workers' sums, one block 64 sums: four threads a sum, each a quarter of the workers.
__global__ __launch_bounds__(256) void conv_grad_sums(const float *parts, uint32_t workers, uint32_t channels, uint32_t taps,
                                                      float *dweight, float *dbias) {
  __shared__ float part[4][64];
  const uint32_t at = blockIdx.x * 64 + threadIdx.x % 64, n = (taps + 1) * channels, quarter = threadIdx.x / 64;
  float v = 0.0f;
  if (at < n)
    for (uint32_t w = quarter; w < workers; w += 4) v += parts[(uint64_t)w * n + at];
  part[quarter][threadIdx.x % 64] = v;
  __syncthreads();
  if (quarter || at >= n) return;
  v = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
  const uint32_t k = at / channels, c = at % channels;
  if (k < taps) dweight[c * taps + k] = v;
  else if (dbias) dbias[c] = v;
}

template <class T, int TAPS>
__global__ __launch_bounds__(256) void conv_step(Conv a) {
  const uint32_t groups = (a.channels + 7) / 8;
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t row = (uint32_t)(id / groups), c = (uint32_t)(id % groups) * 8;
  if (row >= a.rows.tokens) return;
  const int64_t slot = a.index ? a.index[row] : (int64_t)row;
  T *y = (T *)a.y + row * a.y_stride;
  if (slot < 0 || slot >= a.slots) {
    store8(y, c, a.channels, a.y_wide, f32x8{0, 0, 0, 0, 0, 0, 0, 0});
    return;
  }
  f32x8 w[TAPS], bias, window[TAPS];
  T *state = (T *)a.states + slot * (TAPS - 1) * a.channels;
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) window[k] = row8<T>(state, (int64_t)k * a.channels, c, a.channels, a.state_wide);
  const f32x8 x = row8<T>(a.x, row * a.x_stride, c, a.channels, a.x_wide);
  taps_of<TAPS>(a, c, w, bias);
  f32x8 v = weighted<TAPS>(window, x, w, bias);
  shift<TAPS>(window, x);
  if (a.silu) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] *= sigmoid(v[e]);
  }
  store8(y, c, a.channels, a.y_wide, v);
#pragma unroll
  for (int k = 0; k < TAPS - 1; k++) store8(state, k * a.channels + c, (k + 1) * a.channels, a.state_wide, window[k]);
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
Conv conv_of(const uor_trunk_conv_args *s) {
  const uint32_t bytes = s->dtype == UOR_TRUNK_BF16 ? 2 : 4;
  const auto wide = [&](const void *p, int64_t stride) { return aligned16(p, stride, bytes); };
  Conv a{};
  a.rows = Rows{s->offsets, s->tokens, s->seqs};
  a.channels = s->channels, a.pieces = pieces(s->tokens, s->seqs, kRun), a.slots = s->slots;
  a.x_stride = s->x_stride, a.y_stride = s->y_stride;
  a.x = s->x, a.weight = s->weight, a.bias = s->bias, a.initial = s->initial, a.y = s->y, a.final = s->final;
  a.index = s->index, a.states = s->states, a.dy = s->dy, a.dfinal = s->dfinal, a.dx = s->dx, a.dinitial = s->dinitial;
  a.silu = s->silu != 0;
  a.x_wide = wide(s->x, s->x_stride), a.y_wide = wide(s->y ? s->y : s->dy, s->y_stride);
  a.state_wide = wide(s->initial, s->channels) && wide(s->final, s->channels) && wide(s->states, s->channels) &&
                 wide(s->dfinal, s->channels) && wide(s->dinitial, s->channels) && wide(s->dx, s->channels);
  return a;
}
// Workers of a gradient: enough threads for the card, and at least four runs each where there are so many.
uint32_t workers_of(uint32_t count, uint32_t channels) {
  const uint32_t groups = (channels + 7) / 8, most = (1u << 18) / groups + 1, few = (count + 3) / 4;
  return few < most ? few : most;
}
template <template <class, int> class F, class... V>
int by_taps(const uor_trunk_conv_args *s, V... v) {
  if (s->dtype == UOR_TRUNK_BF16)
    switch (s->taps) {
      case 1: return F<bf16, 1>::run(v...);
      case 2: return F<bf16, 2>::run(v...);
      case 3: return F<bf16, 3>::run(v...);
      default: return F<bf16, 4>::run(v...);
    }
  switch (s->taps) {
    case 1: return F<float, 1>::run(v...);
    case 2: return F<float, 2>::run(v...);
    case 3: return F<float, 3>::run(v...);
    default: return F<float, 4>::run(v...);
  }
}
uint32_t blocks_of(uint64_t rows, uint32_t channels) { return (uint32_t)((rows * ((channels + 7) / 8) + 255) / 256); }
template <class T, int TAPS>
struct RowsCall {
  static int run(Conv a, hipStream_t stream) {
    hipLaunchKernelGGL((conv_rows<T, TAPS>), dim3(blocks_of(a.pieces, a.channels)), dim3(256), 0, stream, a);
    return launched();
  }
};
template <class T, int TAPS>
struct StepCall {
  static int run(Conv a, hipStream_t stream) {
    hipLaunchKernelGGL((conv_step<T, TAPS>), dim3(blocks_of(a.rows.tokens, a.channels)), dim3(256), 0, stream, a);
    return launched();
  }
};
template <class T, int TAPS>
struct GradCall {
  static int run(Conv a, float *dweight, float *dbias, hipStream_t stream) {
    hipLaunchKernelGGL((conv_grad_rows<T, TAPS>), dim3(blocks_of(a.workers, a.channels)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(conv_grad_sums, dim3((a.channels * (TAPS + 1) + 63) / 64), dim3(256), 0, stream, a.parts, a.workers,
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
  return by_taps<RowsCall>(s, conv_of(s), (hipStream_t)stream);
}

extern "C" int uor_trunk_conv_step_async(const uor_trunk_conv_args *s, void *stream) {
  if (const int e = check_conv(s, true)) return e;
  if (!s->tokens) return 0;
  if (!s->y || (!s->states && s->taps > 1)) return fail(-1, "null y or states");
  if (!s->index && s->slots < s->tokens) return fail(-1, "%u rows for %u states", s->tokens, s->slots);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return by_taps<StepCall>(s, conv_of(s), (hipStream_t)stream);
}

extern "C" uint64_t uor_trunk_conv_backward_workspace_bytes(const uor_trunk_conv_args *s) {
  if (check_conv(s, false)) return 0;
  return (uint64_t)workers_of(pieces(s->tokens, s->seqs, kRun), s->channels) * (s->taps + 1) * s->channels * sizeof(float);
}

extern "C" int uor_trunk_conv_backward_async(const uor_trunk_conv_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_conv(s, false)) return e;
  if ((s->tokens && (!s->dy || !s->dx)) || !s->dweight) return fail(-1, "null dy, dx or dweight");
  const uint64_t want = uor_trunk_conv_backward_workspace_bytes(s);
  if (!workspace || bytes < want || (uintptr_t)workspace % 16)
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)want);
  Conv a = conv_of(s);
  a.workers = workers_of(a.pieces, s->channels);
  a.parts = (float *)workspace;
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return by_taps<GradCall>(s, a, s->dweight, s->dbias, (hipStream_t)stream);
}
