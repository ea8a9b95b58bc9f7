// trunk.h - what the float trunk's kernels share: types, conversions, packed rows, launch checks.
#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>
#include <stdio.h>

#include "../../../include/uor_trunk.h"

namespace trunk {

using bf16 = __bf16;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x8 = __attribute__((ext_vector_type(8))) float;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

// Four and eight values of an activation's type.
template <class T>
struct Vec;
template <>
struct Vec<bf16> {
  using x4 = bf16x4;
  using x8 = bf16x8;
};
template <>
struct Vec<float> {
  using x4 = f32x4;
  using x8 = f32x8;
};
template <class T>
using V4 = typename Vec<T>::x4;
template <class T>
using V8 = typename Vec<T>::x8;

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }
// 1 / (1 + e^-v) to 2^-21 of it: what the rounding of v log2(e) leaves goes into the exponential, which
// would be |v| 2^-24 of itself off without. Past +-87, where a float holds e^-v no more, as at 87. NUMBER:
// for NaN it may be some number, where the result is multiplied by what v is too.
template <bool NUMBER = false>
__device__ __forceinline__ float sigmoid(float v) {
  const float c = __builtin_amdgcn_fmed3f(v, -87.0f, 87.0f);
  const float t = c * -kLog2e, left = fmaf(c, -1.92596299e-8f, fmaf(c, -kLog2e, -t));
  const float e = exp2_(t), s = __builtin_amdgcn_rcpf(1.0f + fmaf(e, left * 0.693147181f, e));
  return NUMBER || v == v ? s : v;
}
// The activation's, for rows of T. Rows of bf16 go without what the rounding leaves: of a negative v the
// value is |v| 2^-24 of itself off, 2^-20 at -16, where the rows' own rounding is 2^-9. That takes five
// instructions a value less: 152,700 rows of 256 through their norms take 76 us where they took 84,
// convolutions of 300 prompts 52 where they took 55, their gradients 257 where they took 269.
template <class T>
__device__ __forceinline__ float sigmoid_of(float v) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + exp2_(-kLog2e * v));
  else return sigmoid<true>(v);
}
// e^v of v <= 0, to 2^-22 of it: what the rounding of v log2(e) leaves goes into the result.
__device__ __forceinline__ float exp_down(float v) {
  v = fmaxf(v, -120.0f);
  const float t = v * kLog2e, left = fmaf(v, 1.92596299e-8f, fmaf(v, kLog2e, -t));
  const float e = exp2_(t);
  return fmaf(e, left * 0.693147181f, e);
}
// log(1 + e^v) without overflow; its derivative is sigmoid(v). With e = e^-|v|, log(1 + e) is
// 2 artanh(z) of z = e / (2 + e) <= 1/3, whose series is z + z^3 / 3 + ... + z^15 / 15 to 2^-25 of it.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp_down(-fabsf(v)), d = 2.0f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(r, fmaf(-d, r, 1.0f), r);
  const float z = e * r, s = z * z;
  float p = 1.0f / 15.0f;
  p = fmaf(p, s, 1.0f / 13.0f);
  p = fmaf(p, s, 1.0f / 11.0f);
  p = fmaf(p, s, 1.0f / 9.0f);
  p = fmaf(p, s, 1.0f / 7.0f);
  p = fmaf(p, s, 1.0f / 5.0f);
  p = fmaf(p, s, 1.0f / 3.0f);
  p = fmaf(p * s, z, z);
  return fmaxf(v, 0.0f) + 2.0f * p + (v != v ? v : 0.0f);
}

// The packed rows of a call. Offsets are clamped to the rows that there are, and a sequence's end
// to its start, so a table of any content stays inside the arrays.
struct Rows {
  const int32_t *offsets;
  uint32_t tokens, seqs;
  __device__ __forceinline__ uint32_t at(uint32_t s) const {
    if (!offsets) return s ? tokens : 0;
    const int32_t v = offsets[s];
    return v < 0 ? 0u : (uint32_t)v < tokens ? (uint32_t)v : tokens;
  }
  __device__ __forceinline__ void of(uint32_t s, uint32_t &start, uint32_t &end) const {
    start = at(s);
    end = max(at(s + 1), start);
  }
  // The rows that some sequence may own, of offsets that ascend.
  __device__ __forceinline__ void owned(uint32_t &first, uint32_t &end) const {
    first = at(0);
    end = max(at(seqs), first);
  }
};
// Zeros in the rows of `cols` values that no sequence owns: the blocks of a grid share them.
template <class T>
__device__ __forceinline__ void clear_unowned(const Rows &rows, T *to, int64_t stride, uint32_t cols) {
  uint32_t first, end;
  rows.owned(first, end);
  for (uint64_t i = blockIdx.x; i < rows.tokens - (end - first); i += gridDim.x)
    for (uint32_t c = threadIdx.x; c < cols; c += blockDim.x) to[(int64_t)(i < first ? i : i + (end - first)) * stride + c] = (T)0.0f;
}

// Pieces of `size` rows: sequence s owns the pieces from offsets[s] / size + s on. Those places
// do not overlap, as ceil(length / size) pieces fit below the next sequence's, and all lie below
// tokens / size + seqs, so a grid of that many blocks needs no table of the pieces.
struct Piece {
  uint32_t seq, number;  // which sequence, and its how manieth piece
  uint32_t first, end;   // the piece's rows (none: first == end)
  uint32_t start, stop;  // its sequence's rows
};
__host__ __device__ __forceinline__ uint32_t pieces(uint32_t tokens, uint32_t seqs, uint32_t size) { return tokens / size + seqs; }
// The last sequence that begins at or before some place, the first if none does. WAVE: the lanes of a
// wavefront ask for the same, and look at 64 sequences at a time: what each look waits for is a read.
template <bool WAVE, class F>
__device__ __forceinline__ uint32_t last_before(uint32_t seqs, F begins_before) {
  uint32_t lo = 0, hi = seqs;
  while (hi - lo > 1) {
    if constexpr (WAVE) {
      const uint32_t step = (hi - lo + 63) / 64, mid = lo + (threadIdx.x & 63) * step;
      const uint64_t ahead = __ballot(mid < hi && begins_before(mid));
      lo += ahead ? (63 - __builtin_clzll(ahead)) * step : 0;
      hi = hi - lo > step ? lo + step : hi;
    } else {
      const uint32_t mid = (lo + hi) / 2;
      if (begins_before(mid)) lo = mid;
      else hi = mid;
    }
  }
  return lo;
}
template <bool WAVE = false>
__device__ __forceinline__ bool piece(const Rows &rows, uint32_t i, uint32_t size, Piece &p) {
  const uint32_t lo = last_before<WAVE>(rows.seqs, [&](uint32_t s) { return rows.at(s) / size + s <= i; });
  const uint32_t base = rows.at(lo) / size + lo;
  if (base > i) return false;  // only where the offsets do not ascend
  rows.of(lo, p.start, p.stop);
  p.seq = lo;
  p.number = i - base;
  const uint64_t first = p.start + (uint64_t)p.number * size;
  if (first >= p.stop && p.number) return false;
  p.first = first < p.stop ? (uint32_t)first : p.stop;
  p.end = p.stop - p.first > size ? p.first + size : p.stop;
  return true;
}

// The i-th of the places that pieces after a sequence's first have, of which there are `size`-long
// stretches of rows: sequence s has them from offsets[s] / size on. Where several sequences begin in
// one stretch only the last can have any. `which` is the piece's number less one, `count` how many
// pieces its sequence has.
template <bool WAVE>
__device__ __forceinline__ bool later_piece(const Rows &rows, uint32_t i, uint32_t size, uint32_t &seq, uint32_t &which, uint32_t &count) {
  // The last sequence that begins in the i-th stretch or before.
  const uint32_t lo = last_before<WAVE>(rows.seqs, [&](uint32_t s) { return rows.at(s) / size <= i; });
  uint32_t start, stop;
  rows.of(lo, start, stop);
  if (start / size > i || stop == start) return false;
  seq = lo;
  which = i - start / size;
  count = (stop - start - 1) / size + 1;
  return which + 1 < count;
}
__device__ __forceinline__ Piece piece_of(const Rows &rows, uint32_t seq, uint32_t number, uint32_t size) {
  Piece p;
  rows.of(seq, p.start, p.stop);
  p.seq = seq, p.number = number;
  p.first = p.start + number * size;
  p.end = p.stop - p.first > size ? p.first + size : p.stop;
  return p;
}

// N values next to each other, of which no more is known than that each is aligned: memory is read and
// written 16 bytes at a time at any address.
template <class T, int N>
struct Loose {
  using Values = __attribute__((ext_vector_type(N))) T;
  typedef Values At __attribute__((aligned(sizeof(T))));
};
template <class T, int N>
__device__ __forceinline__ typename Loose<T, N>::Values loose(const T *at) {
  return *(const typename Loose<T, N>::At *)at;
}
template <class T, int N>
__device__ __forceinline__ void loose(T *at, typename Loose<T, N>::Values v) {
  *(typename Loose<T, N>::At *)at = v;
}
// N values of a row from `col` on, zeros past `cols` or without a row.
template <class T, int N>
__device__ __forceinline__ typename Loose<T, N>::Values load_some(const T *row, bool there, uint32_t col, uint32_t cols) {
  typename Loose<T, N>::Values v;
#pragma unroll
  for (int e = 0; e < N; e++) v[e] = (T)0.0f;
  if (!there || col >= cols) return v;
  if (col + N <= cols) return loose<T, N>(row + col);
#pragma unroll
  for (int e = 0; e < N; e++)
    if (col + e < cols) v[e] = row[col + e];
  return v;
}
template <class T, int N>
__device__ __forceinline__ void store_some(T *row, uint32_t col, uint32_t cols, typename Loose<T, N>::Values v) {
  if (col + N <= cols) {
    loose<T, N>(row + col, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e++)
    if (col + e < cols) row[col + e] = v[e];
}

// The sums of the columns of parts[rows][n], each given to put(column, sum), in one order: a block
// of 1,024 threads takes 64 columns, 16 threads a column.
template <class F>
__device__ __forceinline__ void sum_columns(const float *parts, uint32_t rows, uint32_t n, F put) {
  __shared__ float part[16][64];
  const uint32_t at = blockIdx.x * 64 + threadIdx.x % 64, share = threadIdx.x / 64;
  float v = 0.0f;
  if (at < n)
#pragma unroll 8
    for (uint32_t r = share; r < rows; r += 16) v += parts[(uint64_t)r * n + at];
  part[share][threadIdx.x % 64] = v;
  __syncthreads();
  if (share || at >= n) return;
  for (int k = 1; k < 16; k++) v += part[k][threadIdx.x];
  put(at, v);
}

// Host side: the last error's text, and a call's device.
inline char *error_text() {
  static thread_local char text[256] = "";
  return text;
}
template <class... V>
inline int fail(int code, const char *format, V... v) {
  if constexpr (sizeof...(V) == 0) snprintf(error_text(), 256, "%s", format);
  else snprintf(error_text(), 256, format, v...);
  return code;
}
struct OnDevice {
  int before = -1;
  bool ok = true;
  explicit OnDevice(int device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    if (before != device) ok = hipSetDevice(device) == hipSuccess;
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};
inline int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail(-2, "launch: %s", hipGetErrorString(e));
}
// Whether rows of this stride can be read 16 bytes at a time.
inline bool aligned16(const void *p, int64_t stride, uint32_t size) {
  return ((uintptr_t)p & 15) == 0 && (stride * size) % 16 == 0;
}

}  // namespace trunk
