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
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }
// log(1 + e^v) without overflow; its derivative is sigmoid(v).
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))) + (v != v ? v : 0.0f); }

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
};

// Pieces of `size` rows: sequence s owns the pieces from offsets[s] / size + s on. Those places
// do not overlap, as ceil(length / size) pieces fit below the next sequence's, and all lie below
// tokens / size + seqs, so a grid of that many blocks needs no table of the pieces.
struct Piece {
  uint32_t seq, number;  // which sequence, and its how manieth piece
  uint32_t first, end;   // the piece's rows (none: first == end)
  uint32_t start, stop;  // its sequence's rows
};
__host__ __device__ __forceinline__ uint32_t pieces(uint32_t tokens, uint32_t seqs, uint32_t size) { return tokens / size + seqs; }
__device__ __forceinline__ bool piece(const Rows &rows, uint32_t i, uint32_t size, Piece &p) {
  uint32_t lo = 0, hi = rows.seqs;  // the last sequence whose pieces begin at or before i
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (rows.at(mid) / size + mid <= i) lo = mid;
    else hi = mid;
  }
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

// Up to eight values of a row from `col` on, zeros past `cols` or without a row.
template <class T>
__device__ __forceinline__ V8<T> load8(const T *row, bool there, uint32_t col, uint32_t cols, bool wide) {
  V8<T> v;
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = (T)0.0f;
  if (!there || col >= cols) return v;
  if (wide && col + 8 <= cols) return *(const V8<T> *)(row + col);
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (col + e < cols) v[e] = row[col + e];
  return v;
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
