// scan_step.hip - the scan for single tokens: sessions' states in device slots, updated in place.
//
// One block takes one head of one session. Bound by the state, read and written once: LN lanes hold
// a row of it, four values each, with their four of B and C in registers, and y is their sum. 1,024
// sessions of 8 heads of 64 by 64, 268 MB of states read and written: 57 us, 4.7 TB/s; with B and C
// read a value at a time 67.
#include "scan.h"

namespace trunk {

struct Step {
  uint32_t heads, groups, dim, state, slots;
  int64_t x_stride, dt_stride, b_stride, c_stride, y_stride;
  const void *x, *dt, *B, *C;
  const float *A, *D, *bias;
  const int32_t *index;
  float *states;
  void *y;
  bool wide;
};

template <class T, int LN>
__global__ __launch_bounds__(256) void scan_step(Step a) {
  constexpr int kRows = 256 / LN;
  const uint32_t row = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const uint32_t group = head / (a.heads / a.groups);
  const int64_t slot = a.index ? a.index[row] : (int64_t)row;
  const T *x = (const T *)a.x + row * a.x_stride + head * a.dim;
  T *y = (T *)a.y + row * a.y_stride + head * a.dim;
  if (slot < 0 || slot >= a.slots) {
    for (uint32_t p = threadIdx.x; p < a.dim; p += 256) y[p] = (T)0.0f;
    return;
  }
  const int ln = threadIdx.x % LN, pr = threadIdx.x / LN;
  const uint32_t n = 4 * ln;
  const T *B = (const T *)a.B + row * a.b_stride + group * a.state, *C = (const T *)a.C + row * a.c_stride + group * a.state;
  const float step = softplus((float)((const T *)a.dt)[row * a.dt_stride + head] + (a.bias ? a.bias[head] : 0.0f));
  const float decay = exp2_(step * a.A[head] * kLog2e), skip = a.D ? a.D[head] : 0.0f;
  const f32x4 b = __builtin_convertvector((load_some<T, 4>(B, true, n, a.state)), f32x4);
  const f32x4 c = __builtin_convertvector((load_some<T, 4>(C, true, n, a.state)), f32x4);
  float *states = a.states + ((uint64_t)slot * a.heads + head) * a.dim * a.state;
  for (uint32_t p = pr; p < a.dim; p += kRows) {
    float *at = states + (uint64_t)p * a.state + n;
    f32x4 h = {0, 0, 0, 0};
    if (a.wide) {
      if (n < a.state) h = *(const f32x4 *)at;
    } else {
      h = load_some<float, 4>(at - n, true, n, a.state);
    }
    const float v = (float)x[p], in = step * v;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      h[e] = h[e] * decay + in * b[e];
      if (n + e < a.state) sum += h[e] * c[e];
    }
    if (a.wide) {
      if (n < a.state) *(f32x4 *)at = h;
    } else {
      store_some<float, 4>(at - n, n, a.state, h);
    }
#pragma unroll
    for (int k = 1; k < LN; k <<= 1) sum += __shfl_xor(sum, k);
    if (ln == 0) y[p] = (T)(sum + skip * v);
  }
}

namespace {
template <class T>
int launch(const Step &a, uint32_t rows, hipStream_t stream) {
  const dim3 grid(rows * a.heads), block(256);
  if (a.state <= 32) hipLaunchKernelGGL((scan_step<T, 8>), grid, block, 0, stream, a);
  else if (a.state <= 64) hipLaunchKernelGGL((scan_step<T, 16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((scan_step<T, 32>), grid, block, 0, stream, a);
  return launched();
}
}  // namespace

}  // namespace trunk

using namespace trunk;

extern "C" int uor_trunk_scan_step_async(const uor_trunk_scan_args *s, void *stream) {
  if (const int e = check_scan(s, true)) return e;
  if (!s->tokens) return 0;
  if (!s->y || !s->states) return fail(-1, "null y or states");
  if (!s->index && s->slots < s->tokens) return fail(-1, "%u rows for %u states", s->tokens, s->slots);
  if ((uint64_t)s->tokens * s->heads > 0x7fffffffu) return fail(-1, "too many rows and heads for one call");
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  const Step a{s->heads, s->groups, s->dim, s->state, s->slots, s->x_stride, s->dt_stride, s->b_stride, s->c_stride,
               s->y_stride, s->x, s->dt, s->B, s->C, s->A, s->D, s->dt_bias, s->index, s->states, s->y,
               s->state % 4 == 0 && ((uintptr_t)s->states & 15) == 0};
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(a, s->tokens, (hipStream_t)stream) : launch<float>(a, s->tokens, (hipStream_t)stream);
}
