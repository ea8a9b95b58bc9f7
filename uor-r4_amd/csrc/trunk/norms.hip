// norms.hip - the norms before and after a block, fused with its gate and residual scale:
//
//   v = out silu(gate),  r' = residual + scale v rsqrt(mean v^2 + eps) post,
//   n = r' rsqrt(mean r'^2 + eps) pre,
//
// and their gradients. Bound by the rows, each read once and written once: LANES lanes hold a row,
// V pieces of eight values each, from its first read to its last write; means are sums of 32 bits.
// A block goes through many rows with the parameters, and in a gradient their sums, in registers.
// 152,700 bf16 rows of 256: 76 us, 5.2 TB/s; gradients of 131,072 of 512: 209 us, 5.1 TB/s, 9 of
// them the sums over blocks.
#include "trunk.h"

namespace trunk {

struct Norms {
  uint32_t rows, width, workers;  // workers: blocks of the grid
  float eps, share;               // share = 1 / width
  int64_t residual_stride, out_stride, gate_stride;
  const void *residual, *out, *gate;
  const float *post, *scale, *pre;
  void *residual_out, *normed;
  const void *dresidual_out, *dnormed;
  void *dresidual, *dout, *dgate;
  float *parts;  // [workers][3][width]: a block's sums of dpost, dscale, dpre
};

// The sum over a row's lanes, to all of them; `scratch` where a row has more than a wavefront.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float *scratch) {
#pragma unroll
  for (int k = 1; k < (LANES < 64 ? LANES : 64); k <<= 1) v += __shfl_xor(v, k);
  if constexpr (LANES > 64) {
    __syncthreads();  // the sum before has been read
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < LANES / 64; k++) v += scratch[k];
  }
  return v;
}
__device__ __forceinline__ f32x8 eight(float v) { return f32x8{v, v, v, v, v, v, v, v}; }
__device__ __forceinline__ float total(f32x8 v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }
// A parameter's eight values, `other` without one; what is past the last column meets only zeros.
__device__ __forceinline__ f32x8 param8(const float *p, uint32_t col, uint32_t cols, float other) {
  return p ? load_some<float, 8>(p, true, col, cols) : eight(other);
}
template <class T>
__device__ __forceinline__ f32x8 values(const void *base, int64_t at, bool there, uint32_t col, uint32_t cols) {
  return __builtin_convertvector((load_some<T, 8>((const T *)base + at, there && base, col, cols)), f32x8);
}
template <class T>
__device__ __forceinline__ void put(void *base, int64_t at, uint32_t col, uint32_t cols, f32x8 v) {
  store_some<T, 8>((T *)base + at, col, cols, __builtin_convertvector(v, V8<T>));
}

// Threads of a block: rows of up to a wavefront share 256, longer ones have a block.
template <int LANES>
constexpr int kBlock = LANES <= 64 ? 256 : LANES;

template <class T, int LANES, int V>
__global__ __launch_bounds__(kBlock<LANES>) void norms_rows(Norms a) {
  __shared__ float scratch[LANES / 64 + 1];
  constexpr uint32_t kRows = kBlock<LANES> / LANES;
  const uint32_t lane = threadIdx.x % LANES;
  f32x8 post[V], scale[V], pre[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const uint32_t c = (i * LANES + lane) * 8;
    post[i] = param8(a.post, c, a.width, 1.0f), scale[i] = param8(a.scale, c, a.width, 1.0f), pre[i] = param8(a.pre, c, a.width, 1.0f);
  }
  for (uint64_t base = (uint64_t)blockIdx.x * kRows; base < a.rows; base += (uint64_t)gridDim.x * kRows) {
    const uint64_t row = base + threadIdx.x / LANES;
    const bool there = row < a.rows;
    f32x8 r[V], v[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      const uint32_t c = (i * LANES + lane) * 8;
      r[i] = values<T>(a.residual, row * a.residual_stride, there, c, a.width);
      v[i] = values<T>(a.out, row * a.out_stride, there, c, a.width);
      if (a.gate) {
        const f32x8 z = values<T>(a.gate, row * a.gate_stride, there, c, a.width);
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= z[e] * sigmoid_of<T>(z[e]);
      }
    }
    if (a.out) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) sum += total(v[i] * v[i]);
      const float inverse = rsqrtf(row_sum<LANES>(sum, scratch) * a.share + a.eps);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const uint32_t c = (i * LANES + lane) * 8;
        r[i] += scale[i] * (v[i] * inverse * post[i]);
        if (there) put<T>(a.residual_out, row * a.width, c, a.width, r[i]);
      }
    }
    if (a.pre) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) sum += total(r[i] * r[i]);
      const float inverse = rsqrtf(row_sum<LANES>(sum, scratch) * a.share + a.eps);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const uint32_t c = (i * LANES + lane) * 8;
        if (there) put<T>(a.normed, row * a.width, c, a.width, r[i] * inverse * pre[i]);
      }
    }
  }
}

// With i the inverse root of a norm and m the mean over a row:
//   dr = dr' + i (pre dn) - r' i^3 m(pre dn r'),   dpre = sum dn r' i,
//   dscale = sum dr v i post,  dpost = sum dr scale v i,
//   dv = i e - v i^3 m(e v) with e = dr scale post,  dout = dv silu(gate),  dgate = dv out silu'(gate).
template <class T, int LANES, int V>
__global__ __launch_bounds__(kBlock<LANES>) void norms_grad_rows(Norms a) {
  __shared__ float scratch[LANES / 64 + 1];
  __shared__ float joined[kBlock<LANES>][9];
  constexpr uint32_t kRows = kBlock<LANES> / LANES;
  const uint32_t lane = threadIdx.x % LANES;
  f32x8 post[V], scale[V], pre[V], dpost[V], dscale[V], dpre[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const uint32_t c = (i * LANES + lane) * 8;
    post[i] = param8(a.post, c, a.width, 1.0f), scale[i] = param8(a.scale, c, a.width, 1.0f), pre[i] = param8(a.pre, c, a.width, 1.0f);
    dpost[i] = dscale[i] = dpre[i] = eight(0.0f);
  }
  for (uint64_t base = (uint64_t)blockIdx.x * kRows; base < a.rows; base += (uint64_t)gridDim.x * kRows) {
    const uint64_t row = base + threadIdx.x / LANES;
    const bool there = row < a.rows;
    f32x8 r[V], v[V], u[V], z[V], d[V];
    float inverse = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const uint32_t c = (i * LANES + lane) * 8;
      r[i] = values<T>(a.residual, row * a.residual_stride, there, c, a.width);
      u[i] = values<T>(a.out, row * a.out_stride, there, c, a.width);
      z[i] = values<T>(a.gate, row * a.gate_stride, there, c, a.width);
      d[i] = values<T>(a.dresidual_out, row * a.width, there, c, a.width);
      v[i] = u[i];
      if (a.gate) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[i][e] *= z[i][e] * sigmoid_of<T>(z[i][e]);
      }
    }
    if (a.out) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) sum += total(v[i] * v[i]);
      inverse = rsqrtf(row_sum<LANES>(sum, scratch) * a.share + a.eps);
#pragma unroll
      for (int i = 0; i < V; i++) r[i] += scale[i] * (v[i] * inverse * post[i]);
    }
    if (a.dnormed) {
      f32x8 e[V];
      float sum = 0.0f, with = 0.0f;
#pragma unroll
      for (int i = 0; i < V; i++) {
        const uint32_t c = (i * LANES + lane) * 8;
        e[i] = values<T>(a.dnormed, row * a.width, there, c, a.width);
        sum += total(r[i] * r[i]);
        with += total(e[i] * pre[i] * r[i]);
      }
      const float j = rsqrtf(row_sum<LANES>(sum, scratch) * a.share + a.eps);
      const float mean = row_sum<LANES>(with, scratch) * a.share * j * j * j;
#pragma unroll
      for (int i = 0; i < V; i++) {
        if (there) dpre[i] += e[i] * r[i] * j;
        d[i] += e[i] * pre[i] * j - r[i] * mean;
      }
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const uint32_t c = (i * LANES + lane) * 8;
      if (there && a.dresidual) put<T>(a.dresidual, row * a.width, c, a.width, d[i]);
    }
    if (!a.out) continue;
    float with = 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const f32x8 p = v[i] * inverse * d[i];
      if (there) {
        dscale[i] += p * post[i];
        dpost[i] += p * scale[i];
      }
      d[i] *= scale[i] * post[i];
      with += total(d[i] * v[i]);
    }
    const float mean = row_sum<LANES>(with, scratch) * a.share * inverse * inverse * inverse;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const uint32_t c = (i * LANES + lane) * 8;
      f32x8 dv = d[i] * inverse - v[i] * mean;
      if (a.gate) {
        f32x8 dz;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float s = sigmoid_of<T>(z[i][e]);
          dz[e] = dv[e] * u[i][e] * s * (1.0f + z[i][e] * (1.0f - s));
          dv[e] *= z[i][e] * s;
        }
        if (there) put<T>(a.dgate, row * a.width, c, a.width, dz);
      }
      if (there) put<T>(a.dout, row * a.width, c, a.width, dv);
    }
  }
  // The sums of the block's rows side by side, in the order of its lanes.
#pragma unroll
  for (int k = 0; k < 3; k++) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const f32x8 s = k == 0 ? dpost[i] : k == 1 ? dscale[i] : dpre[i];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; e++) joined[threadIdx.x][e] = s[e];
      __syncthreads();
      for (uint32_t at = threadIdx.x; at < LANES * 8; at += kBlock<LANES>) {
        float v = 0.0f;
        for (uint32_t g = 0; g < kRows; g++) v += joined[g * LANES + at / 8][at % 8];
        const uint32_t c = i * LANES * 8 + at;
        if (c < a.width) a.parts[((uint64_t)blockIdx.x * 3 + k) * a.width + c] = v;
      }
    }
  }
}

__global__ __launch_bounds__(1024) void norms_grad_sums(const float *parts, uint32_t workers, uint32_t width, float *dpost,
                                                        float *dscale, float *dpre) {
  sum_columns(parts, workers, 3 * width, [&](uint32_t at, float v) {
    float *to = at < width ? dpost : at < 2 * width ? dscale : dpre;
    if (to) to[at % width] = v;
  });
}

namespace {

// Blocks of the grid. Up to a width of 512 a gradient's registers leave a compute unit three blocks of 256
// threads, so 768 of them all begin at once: 65,536 bf16 rows of 512 take 115 us, in 512 blocks 129 and in
// 1,024, which run in two turns, 142. Wider rows leave it two blocks, and over 4,096 one of 1,024 threads:
// there 768 are not the best (65,536 x 1,024: 269 us, 222 in 512 blocks; 16,384 x 4,096: 297 and 243;
// 8,192 x 8,192: 427, 402 in 256), but no rule by width has been made.
constexpr uint32_t kMostBlocks = 2048, kMostWorkers = 768;

uint32_t lanes_of(uint32_t width) {
  if (width > 4096) return 1024;
  if (width > 1024) return 256;
  uint32_t lanes = 1;
  while (lanes * 8 < width && lanes < 64) lanes *= 2;
  return lanes;
}
uint32_t blocks_of(uint32_t rows, uint32_t width, uint32_t most) {
  const uint32_t lanes = lanes_of(width), each = lanes <= 64 ? 256 / lanes : 1, n = (rows + each - 1) / each;
  return n < 1 ? 1 : n < most ? n : most;
}

template <class T, int LANES, int V>
void launch(const Norms &a, bool grad, hipStream_t stream) {
  if (grad) hipLaunchKernelGGL((norms_grad_rows<T, LANES, V>), dim3(a.workers), dim3(kBlock<LANES>), 0, stream, a);
  else hipLaunchKernelGGL((norms_rows<T, LANES, V>), dim3(a.workers), dim3(kBlock<LANES>), 0, stream, a);
}
template <class T>
int launch(const Norms &a, bool grad, hipStream_t stream) {
  switch (lanes_of(a.width)) {
    case 1: launch<T, 1, 1>(a, grad, stream); break;
    case 2: launch<T, 2, 1>(a, grad, stream); break;
    case 4: launch<T, 4, 1>(a, grad, stream); break;
    case 8: launch<T, 8, 1>(a, grad, stream); break;
    case 16: launch<T, 16, 1>(a, grad, stream); break;
    case 32: launch<T, 32, 1>(a, grad, stream); break;
    case 64:
      if (a.width <= 512) launch<T, 64, 1>(a, grad, stream);
      else launch<T, 64, 2>(a, grad, stream);
      break;
    case 256: launch<T, 256, 2>(a, grad, stream); break;
    default: launch<T, 1024, 1>(a, grad, stream);
  }
  return launched();
}

int check_norms(const uor_trunk_norms_args *s) {
  if (!s) return fail(-1, "null argument");
  if (s->dtype > UOR_TRUNK_F32) return fail(-1, "dtype %u is neither bf16 nor f32", s->dtype);
  if (s->width < 1 || s->width > UOR_TRUNK_MAX_WIDTH) return fail(-1, "width %u outside 1..8192", s->width);
  if (!(s->eps >= 0.0f)) return fail(-1, "eps is negative");
  if (!s->out && (s->gate || s->post || s->scale)) return fail(-1, "a gate, post or scale without a block's output");
  if (s->rows && !s->out && !s->residual) return fail(-1, "neither a residual nor a block's output");
  if (!s->out && !s->pre) return fail(-1, "nothing to compute: neither a block's output nor pre");
  if (s->rows > 1 && ((s->residual && s->residual_stride < s->width) || (s->out && s->out_stride < s->width) ||
                      (s->gate && s->gate_stride < s->width)))
    return fail(-1, "rows overlap: a stride is less than a row");
  return 0;
}
Norms norms_of(const uor_trunk_norms_args *s) {
  Norms a{};
  a.rows = s->rows, a.width = s->width, a.eps = s->eps, a.share = 1.0f / (float)s->width;
  a.residual_stride = s->residual_stride, a.out_stride = s->out_stride, a.gate_stride = s->gate_stride;
  a.residual = s->residual, a.out = s->out, a.gate = s->gate, a.post = s->post, a.scale = s->scale, a.pre = s->pre;
  a.residual_out = s->residual_out, a.normed = s->normed, a.dresidual_out = s->dresidual_out, a.dnormed = s->dnormed;
  a.dresidual = s->dresidual, a.dout = s->dout, a.dgate = s->dgate;
  return a;
}

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" int uor_trunk_norms_async(const uor_trunk_norms_args *s, void *stream) {
  if (const int e = check_norms(s)) return e;
  if (!s->rows) return 0;
  if ((s->out && !s->residual_out) || (s->pre && !s->normed)) return fail(-1, "null residual_out or normed");
  Norms a = norms_of(s);
  a.workers = blocks_of(s->rows, s->width, kMostBlocks);
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(a, false, (hipStream_t)stream) : launch<float>(a, false, (hipStream_t)stream);
}

extern "C" uint64_t uor_trunk_norms_backward_workspace_bytes(const uor_trunk_norms_args *s) {
  if (check_norms(s)) return 0;
  return (uint64_t)blocks_of(s->rows, s->width, kMostWorkers) * 3 * s->width * sizeof(float);
}

extern "C" int uor_trunk_norms_backward_async(const uor_trunk_norms_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_norms(s)) return e;
  if (s->rows && ((s->out && !s->dout) || (s->gate && !s->dgate))) return fail(-1, "null dout or dgate");
  if (s->dnormed && !s->pre) return fail(-1, "dnormed without pre");
  const uint64_t want = uor_trunk_norms_backward_workspace_bytes(s);
  if (!workspace || bytes < want || (uintptr_t)workspace % 16)
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)want);
  Norms a = norms_of(s);
  a.workers = blocks_of(s->rows, s->width, kMostWorkers);
  a.parts = (float *)workspace;
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  if (const int e = s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(a, true, (hipStream_t)stream) : launch<float>(a, true, (hipStream_t)stream)) return e;
  hipLaunchKernelGGL(norms_grad_sums, dim3((3 * s->width + 63) / 64), dim3(1024), 0, (hipStream_t)stream, a.parts, a.workers, s->width,
                     s->dpost, s->dscale, s->dpre);
  return launched();
}
