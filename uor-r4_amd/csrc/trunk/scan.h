// scan.h - what the scan's kernels share: tiles on the matrix cores, chunks of rows in LDS, the
// logarithms of a chunk's decays.
//
// A sequence is taken in chunks of 64 rows. With a_t = D_t A and l_t its running sum inside the
// chunk, the recurrence over a chunk from the state h before it is
//
//   y_t = e^(l_t) h C_t + sum_(s <= t) (C_t . B_s) e^(l_t - l_s) D_s x_s,
//   h'  = e^(l_end) h + sum_s e^(l_end - l_s) D_s x_s (x) B_s,
//
// four matrix products. No factor e^(-l_s) is formed on its own: it would overflow where steps are
// long, and every exponent above is a decay between two rows.
#pragma once
#include "trunk.h"

namespace trunk {

constexpr int kChunk = 64;    // rows of a chunk: four tiles of 16
constexpr int kThreads = 256; // four wavefronts

// 16 x 16 products over 32 places. A lane holds eight values of its operand's row (lane % 16),
// places 8 (lane / 16) .. + 7, or for an operand built from two result tiles places 4 (lane / 16)
// .. + 3 of the first and of the second: any order of the places is right if both operands have
// the same. A lane's four results are rows 4 (lane / 16) + r of column lane % 16.
//
// Split is an operand that was computed in 32 bits. With bf16 it is the sum of two bf16 parts,
// 2^-18 of a value off at most: one part alone would add an error of the size of y's own rounding
// to y, and states and their sums are held to 32 bits' worth.
//
// v rounded to bf16, and v then what the rounding left of it. Two values at a time, as they are
// rounded by one instruction and lie in one register.
__device__ __forceinline__ bf16x8 round8(f32x8 &v) {
  using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
  u32x4 out;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const bf16x2 two = {(bf16)v[2 * e], (bf16)v[2 * e + 1]};
    out[e] = __builtin_bit_cast(uint32_t, two);
    asm("" : "+v"(out[e]));  // else each value is rounded once more by itself
    v[2 * e] -= __builtin_bit_cast(float, out[e] << 16);
    v[2 * e + 1] -= __builtin_bit_cast(float, out[e] & 0xffff0000u);
  }
  return __builtin_bit_cast(bf16x8, out);
}
template <class T>
struct Mma;
template <>
struct Mma<bf16> {
  struct Split {
    bf16x8 hi, lo;
  };
  static constexpr int kParts = 2;
  static __device__ __forceinline__ Split split(f32x8 v) {
    Split s;
    s.hi = round8(v);
    s.lo = round8(v);
    return s;
  }
  static __device__ __forceinline__ f32x4 mul(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mul(bf16x8 a, const Split &b, f32x4 c) { return mul(a, b.hi, mul(a, b.lo, c)); }
  static __device__ __forceinline__ f32x4 mul(const Split &a, bf16x8 b, f32x4 c) { return mul(a.hi, b, mul(a.lo, b, c)); }
};
template <>
struct Mma<float> {
  using Split = f32x8;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ Split split(f32x8 v) { return v; }
  static __device__ __forceinline__ f32x4 mul(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// The pitch of a row of `n` values in LDS: 16 bytes more, so that the 16 rows that a wavefront
// reads 16 bytes of at a time start four banks apart.
template <class T>
constexpr int pitch(int n) {
  return n + 16 / (int)sizeof(T);
}

template <class T>
__device__ __forceinline__ V8<T> operand(const T *row, int place) {
  return *(const V8<T> *)(row + place);
}
// The places of two result tiles of 16 rows (see Mma).
template <class T>
__device__ __forceinline__ V8<T> operand_tiles(const T *row, int place) {
  const V4<T> a = *(const V4<T> *)(row + place), b = *(const V4<T> *)(row + place + 16);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <class T>
__device__ __forceinline__ f32x8 widen(V8<T> v) {
  return __builtin_convertvector(v, f32x8);
}

// One head of one call.
struct Scan {
  Rows rows;
  uint32_t heads, groups, dim, state;
  uint32_t size, pieces;  // rows of a piece, and how many pieces the grid has
  uint32_t later;         // places of pieces after a sequence's first
  uint32_t tiles;         // a head's parts of dim
  int64_t x_stride, dt_stride, b_stride, c_stride, y_stride;
  const void *x, *dt, *B, *C;
  const float *A, *D, *bias;
  const float *initial;  // [seqs][heads][dim][state], or NULL
  void *y;
  float *final;
  float *starts;         // [pieces][heads][dim][state]: where a piece begins, if sequences are cut; or NULL
  double *totals;        // [pieces][heads]: log2 of a piece's whole decay
  bool x_wide, b_wide, c_wide, y_wide, state_wide;
};

// Pieces are dealt to the eight XCDs in turn, and a piece's heads run on one of them, next to each
// other: heads of a group read the same B and C, which that XCD's L2 then holds.
constexpr uint32_t kXcds = 8;
inline uint32_t grid_of(uint32_t pieces, uint32_t heads) { return (pieces + kXcds - 1) / kXcds * kXcds * heads; }
__device__ __forceinline__ void place_of(uint32_t block, uint32_t heads, uint32_t &piece, uint32_t &head) {
  const uint32_t k = block / kXcds;
  piece = k / heads * kXcds + block % kXcds;
  head = k % heads;
}

// The logarithms (base 2) of a chunk's decays. l_t is kept as a float and the float that is left
// of it: l_t - l_s then has the error of its own size and not of the sum's.
struct Decays {
  float hi[kChunk], lo[kChunk];
  float step[kChunk];  // D_t, 0 past the chunk's last row
  float from[kChunk];  // e^(l_t)
  float tail[kChunk];  // e^(l_end - l_t)
  float to[kChunk];    // D_t e^(l_end - l_t)
  double total;        // l_end
  float whole;         // e^(l_end)
};
// By one wavefront, a row a lane.
template <class T>
__device__ __forceinline__ void decays(Decays &d, const T *dt, int64_t stride, uint32_t first, uint32_t end, float A, float bias) {
  const int lane = threadIdx.x & 63;
  const uint32_t row = first + lane;
  float step = 0.0f;
  double l = 0.0;
  if (row < end) {
    step = softplus((float)dt[(int64_t)row * stride] + bias);
    l = (double)step * (double)A * 1.4426950408889634;
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const double before = __shfl_up(l, k);
    if (lane >= k) l += before;
  }
  const double last = __shfl(l, 63);
  const float hi = (float)l;
  d.hi[lane] = hi;
  d.lo[lane] = hi - hi == 0.0f ? (float)(l - (double)hi) : 0.0f;
  d.step[lane] = step;
  d.from[lane] = exp2_(hi);
  const float tail = exp2_((float)(last - l));
  d.tail[lane] = tail;
  d.to[lane] = step * tail;
  if (lane == 0) {
    d.total = last;
    d.whole = exp2_((float)last);
  }
}

// Rows of a chunk into LDS. A thread takes eight columns of two rows: in `plain` rows as they
// are, in `turned` columns as rows, two rows' values as one piece of a row.
template <class T, int COLS>
__device__ __forceinline__ bool stage(T *plain, T *turned, const T *base, int64_t stride, uint32_t first, uint32_t end,
                                      uint32_t cols, bool wide) {
  bool odd = false;
  constexpr int kJobs = kChunk / 2 * (COLS / 8);
#pragma unroll
  for (int job = threadIdx.x; job < kJobs; job += kThreads) {
    const int row = job % 32 * 2, col = job / 32 * 8;
    const T *at = base + (int64_t)(first + row) * stride;
    const V8<T> a = load8(at, first + row < end, col, cols, wide);
    const V8<T> b = load8(at + stride, first + row + 1 < end, col, cols, wide);
    if (plain) {
      *(V8<T> *)(plain + row * pitch<T>(COLS) + col) = a;
      *(V8<T> *)(plain + (row + 1) * pitch<T>(COLS) + col) = b;
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        T *to = turned + (col + e) * pitch<T>(kChunk) + row;
        to[0] = a[e];
        to[1] = b[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) odd |= !finite((float)a[e]) || !finite((float)b[e]);
  }
  return odd;
}

// A wavefront's part of the state: PW tiles of 16 over dim, NT over state, dealt to four wavefronts.
template <int NT, int PW>
struct Own {
  static constexpr int kTiles = NT * PW / 4;
  int p, n;  // its 16 values of dim, and the first of its 16s of the state's axis
  __device__ __forceinline__ Own() {
    const int wave = threadIdx.x >> 6;
    p = wave % PW;
    n = wave / PW * kTiles;
  }
};

// The state at `at` ([dim][state]) as result tiles; rows past its sizes are zeros.
template <int NT, int PW>
__device__ __forceinline__ void load_state(f32x4 (&h)[NT * PW / 4], const Own<NT, PW> &own, const float *at, uint32_t p0,
                                           uint32_t dim, uint32_t state) {
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const uint32_t p = p0 + own.p * 16 + (lane & 15);
#pragma unroll
  for (int i = 0; i < NT * PW / 4; i++) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t n = (own.n + i) * 16 + 4 * q + r;
      h[i][r] = at && p < dim && n < state ? at[(uint64_t)p * state + n] : 0.0f;
    }
  }
}
template <int NT, int PW>
__device__ __forceinline__ void store_state(const f32x4 (&h)[NT * PW / 4], const Own<NT, PW> &own, float *at, uint32_t p0,
                                            uint32_t dim, uint32_t state) {
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const uint32_t p = p0 + own.p * 16 + (lane & 15);
#pragma unroll
  for (int i = 0; i < NT * PW / 4; i++) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t n = (own.n + i) * 16 + 4 * q + r;
      if (p < dim && n < state) at[(uint64_t)p * state + n] = h[i][r];
    }
  }
}
// h' = e^(l_end) h + sum over the chunk's rows of weight * row (x) (row of the other).
template <class T, int NT, int PW>
__device__ __forceinline__ void advance(f32x4 (&h)[NT * PW / 4], const Own<NT, PW> &own, const T *x_turned, const T *b_turned,
                                        const float *weight, float whole) {
  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int i = 0; i < NT * PW / 4; i++) h[i] *= whole;
#pragma unroll
  for (int k = 0; k < kChunk; k += 32) {
    f32x8 v = widen<T>(operand(x_turned + (own.p * 16 + i16) * pitch<T>(kChunk), k + 8 * q));
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] *= weight[k + 8 * q + e];
    const auto w = Mma<T>::split(v);
#pragma unroll
    for (int i = 0; i < NT * PW / 4; i++)
      h[i] = Mma<T>::mul(operand(b_turned + ((own.n + i) * 16 + i16) * pitch<T>(kChunk), k + 8 * q), w, h[i]);
  }
}

int check_scan(const uor_trunk_scan_args *s, bool step);
Scan scan_of(const uor_trunk_scan_args *s, uint32_t size);
// A join's blocks: by sequences, or by the places of later pieces, where there are fewer.
__host__ __device__ inline uint32_t join_places(const Scan &a) { return a.rows.seqs < a.later ? a.rows.seqs : a.later; }
// The sequence of a join's block, and how many pieces it has.
__device__ __forceinline__ bool joined(const Scan &a, uint32_t i, uint32_t &seq, uint32_t &n) {
  if (a.rows.seqs < a.later) {
    uint32_t start, end;
    a.rows.of(i, start, end);
    seq = i, n = end > start ? (end - start - 1) / a.size + 1 : 1;
    return n > 1;
  }
  uint32_t which;
  return later_piece<true>(a.rows, i, a.size, seq, which, n) && !which;
}
inline dim3 join_of(const Scan &a) {
  const uint32_t states = join_places(a) * a.heads, most = (a.dim * a.state + kThreads - 1) / kThreads, even = 4096 / states + 1;
  return dim3(states, most < even ? most : even);
}
uint32_t piece_rows(uint32_t tokens, uint32_t seqs, uint32_t units, uint32_t least);
// Whether rows whose heads or groups are `part` values can be read 16 bytes at a time, and a chunk of
// them by offsets of 32 bits.
inline bool wide_rows(const void *p, int64_t stride, uint32_t part, uint32_t bytes) {
  return aligned16(p, stride, bytes) && part * bytes % 16 == 0 && stride < (1 << 22);
}

}  // namespace trunk
