// wave.h - the scan by wavefronts: one wavefront holds one head's state, or a part of its values, in
// registers, and takes its sequence in chunks of 64 rows.
//
// With a_t = D_t A and l_t its running sum inside the chunk, the recurrence over a chunk from the
// state h before it is
//
//   y_t = e^(l_t) h C_t + sum_(s <= t) (C_t . B_s) e^(l_t - l_s) D_s x_s,
//   h'  = e^(l_end) h + sum_s e^(l_end - l_s) D_s x_s (x) B_s,
//
// four matrix products. No factor e^(-l_s) is formed on its own: it would overflow where steps are
// long. With r_i the sum at the end of the chunk's i-th 16 rows, a row t of tile i and a row s of a
// tile j < i have e^(l_t - l_s) = e^(l_t - r_i) e^(r_i - r_(j+1)) e^(r_(j+1) - l_s), every factor a
// decay between two rows; only within a tile of 16 the differences are formed one by one.
//
// The wavefronts of a block are heads of one group, which share the chunk's B and C in LDS.
#pragma once
#include "scan.h"

namespace trunk {

// Tiles of 16 of an axis of the state go in pairs, so that a lane's results of a pair are eight
// values next to each other: row 4 q + r of tile i is place 32 (i / 2) + 8 q + 4 (i % 2) + r. They
// are then 16 or 32 bytes of memory, and in this order the operand of the next product.
__device__ __forceinline__ int place(int tile, int row) { return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3); }

// An operand that was computed in 32 bits. With bf16 it goes in as the sum of three bf16 parts, 2^-25 of
// a value off at most, so that the products are those of 32 bits. With two parts, 2^-18 off, one bf16
// output in a thousand rounded the other way than 32-bit sums do, and states were four times further from
// 64 bits than such sums are; 300 bf16 prompts of up to 509 took 92 us where they take 98, gradients of
// 2,048 sequences of 128 1,000 where they take 1,075.
template <class T>
struct Fine;
template <>
struct Fine<bf16> {
  bf16x8 hi, mid, lo;
  static __device__ __forceinline__ Fine of(f32x8 v) {
    Fine s;
    s.hi = round8(v);
    s.mid = round8(v);
    s.lo = round8(v);
    return s;
  }
};
template <>
struct Fine<float> {
  f32x8 v;
  static __device__ __forceinline__ Fine of(f32x8 v) { return {v}; }
};
__device__ __forceinline__ f32x4 mul(bf16x8 a, const Fine<bf16> &b, f32x4 c) {
  return Mma<bf16>::mul(a, b.hi, Mma<bf16>::mul(a, b.mid, Mma<bf16>::mul(a, b.lo, c)));
}
__device__ __forceinline__ f32x4 mul(const Fine<bf16> &a, bf16x8 b, f32x4 c) {
  return Mma<bf16>::mul(a.hi, b, Mma<bf16>::mul(a.mid, b, Mma<bf16>::mul(a.lo, b, c)));
}
__device__ __forceinline__ f32x4 mul(f32x8 a, const Fine<float> &b, f32x4 c) { return Mma<float>::mul(a, b.v, c); }
__device__ __forceinline__ f32x4 mul(const Fine<float> &a, f32x8 b, f32x4 c) { return Mma<float>::mul(a.v, b, c); }

// A lane's number, anew: what a loop computes from it is computed again each time, and does not stand
// in registers, of which these kernels have none to spare.
__device__ __forceinline__ int anew(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// The operand of column place(tile, lane % 16) of rows row0 .. + 31, of a chunk that lies in LDS row
// after row: places 4 q .. + 3 of its first 16 rows and of its second. 16 lanes read four rows of
// 16 values, each lane four of a row, and get them by columns.
template <class T, int PITCH>
__device__ __forceinline__ V8<T> column(int lane, const T *base, int row0, int tile) {
  const int q = lane >> 4, i16 = lane & 15;
  if constexpr (sizeof(T) == 2) {
    using Local = __attribute__((address_space(3))) bf16x4;
    const T *at = base + (row0 + 4 * q + (i16 >> 2)) * PITCH + 32 * (tile >> 1) + 8 * (i16 & 3) + 4 * (tile & 1);
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local *)at);
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local *)(at + 16 * PITCH));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const T *at = base + (row0 + 4 * q) * PITCH + place(tile, i16);
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = at[e * PITCH], v[e + 4] = at[(16 + e) * PITCH];
    return v;
  }
}

// 0x80000000 for a column past the last, an offset that no buffer has; nothing for others.
__device__ __forceinline__ uint32_t past(uint32_t col, uint32_t cols) { return (cols - 1 - col) & 0x80000000u; }
// Eight values of a row whose first is `offset` bytes into a buffer, 16 bytes at a time: those past
// the row's last column, or past the buffer's end, are zeros, and none of them is written.
template <class T>
__device__ __forceinline__ V8<T> load_eight(__amdgpu_buffer_rsrc_t rows, uint32_t offset, uint32_t col, uint32_t cols) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)(offset | past(col, cols)), 0, 0));
  } else {
    const f32x4 a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)(offset | past(col, cols)), 0, 0));
    const f32x4 b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)((offset + 16) | past(col + 4, cols)), 0, 0));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
template <class T>
__device__ __forceinline__ void store_eight(__amdgpu_buffer_rsrc_t rows, uint32_t offset, uint32_t col, uint32_t cols, f32x8 v) {
  using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
  if constexpr (sizeof(T) == 2) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8)), rows, (int)(offset | past(col, cols)), 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 0, 1, 2, 3)), rows, (int)(offset | past(col, cols)), 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, __builtin_shufflevector(v, v, 4, 5, 6, 7)), rows,
                                           (int)((offset + 16) | past(col + 4, cols)), 0, 0);
  }
}

// v, or 0 where it is not wanted, whatever v is.
__device__ __forceinline__ float keep(float v, bool wanted) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & (wanted ? ~0u : 0u));
}

// A chunk's rows of COLS columns on their way to LDS, row after row: THREADS threads share it, each
// eight columns of a row at a time. Rows that can be read 16 bytes at a time are fetched into
// registers long before they are put down; others are read when they are.
template <class T, int COLS, int THREADS>
struct Load {
  static constexpr int kJobs = kChunk * (COLS / 8), kN = (kJobs + THREADS - 1) / THREADS, kPitch = pitch<T>(COLS);
  V8<T> v[kN];
  const T *at;
  uint32_t rows;
  __device__ __forceinline__ void get(uint32_t thread, const T *base, int64_t stride, uint32_t first, uint32_t end, uint32_t cols, bool wide) {
    at = base + (int64_t)first * stride;
    rows = end - first;
    // Reads past the buffer's end give zeros: rows past the chunk's last, columns sent there, and
    // all that this form cannot read.
    const uint32_t pitch = (uint32_t)stride * sizeof(T), bytes = wide && rows ? (rows - 1) * pitch + cols * (uint32_t)sizeof(T) : 0;
    const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < kN; i++) {
      const uint32_t job = i * THREADS + thread, col = job % (COLS / 8) * 8;  // a job too many is a row too many
      v[i] = load_eight<T>(from, job / (COLS / 8) * pitch + col * (uint32_t)sizeof(T), col, cols);
    }
  }
  // Whether some value is infinite or no number.
  __device__ __forceinline__ bool put(uint32_t thread, T *to, int64_t stride, uint32_t cols, bool wide) const {
    bool odd = false;
    if (wide) {
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const uint32_t job = i * THREADS + thread;
        if (kJobs % THREADS == 0 || job < kJobs) *(V8<T> *)(to + job / (COLS / 8) * kPitch + job % (COLS / 8) * 8) = v[i];
      }
      if constexpr (sizeof(T) == 2) {  // the largest exponent of all
        using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
        using u16x8 = __attribute__((ext_vector_type(8))) uint16_t;
        u16x8 most = 0;
#pragma unroll
        for (int i = 0; i < kN; i++)
          most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x8, __builtin_bit_cast(u32x4, v[i]) & 0x7fff7fffu));
        odd = __builtin_reduce_max(most) >= 0x7f80;
      } else {
#pragma unroll
        for (int i = 0; i < kN; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) odd |= !finite(v[i][e]);
      }
    } else {
#pragma unroll 1
      for (uint32_t job = thread; job < kJobs; job += THREADS) {
        const uint32_t row = job / (COLS / 8), col = job % (COLS / 8) * 8;
        const V8<T> some = load_some<T, 8>(at + (int64_t)row * stride, row < rows, col, cols);
        *(V8<T> *)(to + row * kPitch + col) = some;
#pragma unroll
        for (int e = 0; e < 8; e++) odd |= !finite((float)some[e]);
      }
    }
    return odd;
  }
};

// v of the lane that a data movement between lanes names, 0 where it names none.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double moved(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The sum over the lanes of its 16 up to this one, and over lanes 0 .. this one.
template <class F>
__device__ __forceinline__ F running_sum16(F v) {
  v += moved<0x111>(v);  // from 1, 2, 4 and 8 lanes before
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  return v + moved<0x118>(v);
}
__device__ __forceinline__ double running_sum(double v) {
  v = running_sum16(v);
  v += moved<0x142, 0xa>(v);         // the first 16's sum to the second, the third's to the fourth
  return v + moved<0x143, 0xc>(v);  // the first half's to the second
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)bits, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// 2^v: what v's rounding to 32 bits leaves goes into the result, as these factors are common to whole
// rows and states and their errors do not cancel in sums.
__device__ __forceinline__ float power(double v) {
  const float hi = (float)v, e = exp2_(hi), left = hi - hi == 0.0f ? (float)(v - (double)hi) : 0.0f;
  return fmaf(e, left * 0.693147181f, e);
}
// The same with no more than the exponential's own error, for sums over many rows.
__device__ __forceinline__ double power64(double v) {
  const float hi = (float)v;
  return (double)exp2_(hi) * (1.0 + (hi - hi == 0.0f ? (v - (double)hi) * 0.6931471805599453 : 0.0));
}
__device__ __forceinline__ float between(double later, double before) { return power(later - before); }

// What a wavefront knows of its chunk's steps. The logarithms (base 2) are sums in 64 bits; l_t is
// kept as a float and the float that is left of it, so that l_t - l_s has the error of its own size.
struct Steps {
  float hi[kChunk], lo[kChunk];
  float step[kChunk];  // D_t, 0 past the chunk's last row
  float u[kChunk];     // e^(l_t - r_i), from the start of the row's tile i
  float v[kChunk];     // D_t e^(r_(i+1) - l_t), to its end
};
struct GradSteps : Steps {
  double l[kChunk];  // the logarithms themselves
  float to[4], from[4], c[3];  // as Decay's, for code that does not know which tiles it takes
  float w[kChunk];   // e^(r_(i+1) - l_t)
};
struct Decay {
  float to[4];     // from a tile's end to the chunk's
  float from[4];   // from the chunk's start to a tile's
  float whole;
  float c20, c30, c31;  // from the end of tile 0 to tile 2's start, ...
  double total;
};
// A row's step and the logarithm of its decay, nothing past the chunk's last row. -1e5 already leaves
// nothing of what was before, and differences of such sums are numbers, where infinities' are none.
struct Row {
  float step;
  double log;
};
__device__ __forceinline__ Row row_of(float raw, bool there, float A, float bias) {
  Row r;
  r.step = there ? softplus(raw + bias) : 0.0f;
  r.log = there ? (double)r.step * (double)A * 1.4426950408889634 : 0.0;
  r.log = r.log < -1e5 ? -1e5 : r.log;
  return r;
}
template <class S>
__device__ __forceinline__ Decay steps_of(int lane, S &s, Row row) {
  const float step = row.step;
  const double l = running_sum(row.log);
  const double r1 = lane_of(l, 15), r2 = lane_of(l, 31), r3 = lane_of(l, 47), r4 = lane_of(l, 63);
  const double start = lane < 16 ? 0.0 : lane < 32 ? r1 : lane < 48 ? r2 : r3, end = lane < 16 ? r1 : lane < 32 ? r2 : lane < 48 ? r3 : r4;
  const float hi = (float)l;
  s.hi[lane] = hi;
  s.lo[lane] = hi - hi == 0.0f ? (float)(l - (double)hi) : 0.0f;
  s.step[lane] = step;
  s.u[lane] = between(l, start);
  const float w = between(end, l);
  s.v[lane] = step * w;
  if constexpr (sizeof(S) > sizeof(Steps)) s.w[lane] = w, s.l[lane] = l;
  Decay d;
  d.to[0] = between(r4, r1), d.to[1] = between(r4, r2), d.to[2] = between(r4, r3), d.to[3] = 1.0f;
  d.from[0] = 1.0f, d.from[1] = power(r1), d.from[2] = power(r2), d.from[3] = power(r3);
  d.whole = power(r4);
  d.c20 = between(r2, r1), d.c30 = between(r3, r1), d.c31 = between(r3, r2);
  d.total = r4;
  if constexpr (sizeof(S) > sizeof(Steps)) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) s.to[i] = d.to[i], s.from[i] = d.from[i];
      s.c[0] = d.c20, s.c[1] = d.c30, s.c[2] = d.c31;
    }
  }
  return d;
}

// A state [dim][state] in a wavefront: NT tiles of state by PW of dim, columns of dim.
template <int NT, int PW>
__device__ __forceinline__ void get_state(f32x4 (&h)[NT][PW], const float *at, uint32_t dim, uint32_t state, bool wide) {
  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int i = 0; i < PW; i++)
#pragma unroll
    for (int n = 0; n < NT; n++) h[n][i] = f32x4{0, 0, 0, 0};
  if (!at) return;
#pragma unroll
  for (int i = 0; i < PW; i++) {
    const uint32_t p = place(i, i16);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const uint32_t first = place(n, 4 * q);
      if (p >= dim) continue;
      const float *from = at + (uint64_t)p * state + first;
      if (wide) {
        if (first < state) h[n][i] = *(const f32x4 *)from;
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (first + r < state) h[n][i][r] = from[r];
      }
    }
  }
}
template <int NT, int PW>
__device__ __forceinline__ void put_state(const f32x4 (&h)[NT][PW], float *at, uint32_t dim, uint32_t state, bool wide) {
  const int lane = threadIdx.x & 63, q = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int i = 0; i < PW; i++) {
    const uint32_t p = place(i, i16);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const uint32_t first = place(n, 4 * q);
      if (p >= dim) continue;
      float *to = at + (uint64_t)p * state + first;
      if (wide) {
        if (first < state) *(f32x4 *)to = h[n][i];
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (first + r < state) to[r] = h[n][i][r];
      }
    }
  }
}

// The weights of a k-step's eight rows (see column) from a chunk's, each tile's by its factor.
__device__ __forceinline__ f32x8 weights(int lane, const float *rows, int row0, float first, float second) {
  const int q = lane >> 4;
  const f32x4 a = *(const f32x4 *)(rows + row0 + 4 * q) * first, b = *(const f32x4 *)(rows + row0 + 16 + 4 * q) * second;
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// h' = e^(l_end) h + the sum over the chunk's rows of their weight, column of x and row of B.
template <class T, int NT, int PW>
__device__ __forceinline__ void advance(int lane, f32x4 (&h)[NT][PW], const V8<T> (&xs)[2][PW], const T *sB, const float *rows, const float (&to)[4], float whole) {
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < PW; i++) h[n][i] *= whole;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const f32x8 weight = weights(lane, rows, 32 * k, to[2 * k], to[2 * k + 1]);
    V8<T> b[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) b[n] = column<T, pitch<T>(16 * NT)>(lane, sB, 32 * k, n);
#pragma unroll
    for (int i = 0; i < PW; i++) {
      const auto w = Fine<T>::of(widen<T>(xs[k][i]) * weight);
#pragma unroll
      for (int n = 0; n < NT; n++) h[n][i] = mul(b[n], w, h[n][i]);
    }
  }
}

// The blocks of a call by wavefronts: `units` of a group are its heads' parts of dim, W to a block.
struct Unit {
  uint32_t piece, group, head, p0;
  bool idle;  // a wavefront past the group's last unit
};
template <int W>
__device__ __forceinline__ Unit unit_of(const Scan &a, uint32_t parts) {
  Unit u;
  uint32_t at;
  const uint32_t share = a.heads / a.groups, blocks = (share * a.tiles + W - 1) / W;
  place_of(blockIdx.x, a.groups * blocks, u.piece, at);
  u.group = at / blocks;
  uint32_t unit = at % blocks * W + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u.idle = unit >= share * a.tiles;
  unit = u.idle ? 0 : unit;
  u.head = u.group * share + unit / a.tiles;
  u.p0 = unit % a.tiles * parts;
  return u;
}

// A piece's end state from zeros and its whole decay, at the place of the piece after it; a sequence's last
// piece needs neither. BACK, for the pieces after a sequence's first, at their own places: the gradient at
// the state before a piece from that of y alone, with dy for x and C for B, along the piece from its end:
// the sum of e^(l_t) dy_t (x) C_t.
template <class T, int NT, int PW, int W, bool BACK>
__global__ __launch_bounds__(64 * W, W == 1 ? 1 : 2) void scan_ends(Scan a) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kNp = pitch<T>(kN), kPp = pitch<T>(kP);
  __shared__ __align__(16) T sB[kChunk * kNp], sXs[W][kChunk * kPp];
  __shared__ Steps steps[W];
  const Unit unit = unit_of<W>(a, kP);
  uint32_t seq, which, count;
  if (unit.piece >= a.later || !later_piece<true>(a.rows, unit.piece, a.size, seq, which, count)) return;
  const Piece at = piece_of(a.rows, seq, BACK ? which + 1 : which, a.size);
  const int wave = threadIdx.x >> 6, lane0 = threadIdx.x & 63;
  const uint32_t head = unit.head;
  const T *x = (const T *)a.x + head * a.dim + unit.p0, *dt = (const T *)a.dt + head, *B = (const T *)a.B + unit.group * a.state;
  const uint32_t dim = a.dim - unit.p0 < (uint32_t)kP ? a.dim - unit.p0 : kP;
  const float A = a.A[head], bias = a.bias ? a.bias[head] : 0.0f;
  f32x4 h[NT][PW];
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < PW; i++) h[n][i] = f32x4{0, 0, 0, 0};
  double total = 0.0;
  Load<T, kN, 64 * W> nextB;
  Load<T, kP, 64> nextX;
  float raw = 0.0f;
  const uint32_t chunks = (at.end - at.first + kChunk - 1) / kChunk;
  const auto fetch = [&](uint32_t i) {  // the i-th chunk on the way, none past the last
    const uint32_t first = i < chunks ? at.first + (BACK ? chunks - 1 - i : i) * kChunk : at.first;
    const uint32_t end = i < chunks ? (at.end - first > kChunk ? first + kChunk : at.end) : first;
    const int lane = anew(lane0), thread = wave * 64 + lane;
    nextB.get(thread, B, a.b_stride, first, end, a.state, a.b_wide);
    nextX.get(lane, x, a.x_stride, first, end, dim, a.x_wide);
    raw = first + lane < end ? (float)dt[(int64_t)(first + lane) * a.dt_stride] : 0.0f;
  };
  fetch(0);
  for (uint32_t i = 0; i < chunks; i++) {
    const uint32_t first = at.first + (BACK ? chunks - 1 - i : i) * kChunk, end = at.end - first > kChunk ? first + kChunk : at.end;
    const int lane = anew(lane0), thread = wave * 64 + lane;
    __syncthreads();
    nextB.put(thread, sB, a.b_stride, a.state, a.b_wide);
    nextX.put(lane, sXs[wave], a.x_stride, dim, a.x_wide);
    const Decay d = steps_of(lane, steps[wave], row_of(raw, first + lane < end, A, bias));
    __syncthreads();
    fetch(i + 1);
    if (unit.idle) continue;
    V8<T> xs[2][PW];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int i = 0; i < PW; i++) xs[k][i] = column<T, kPp>(lane, sXs[wave], 32 * k, i);
    advance<T, NT, PW>(lane, h, xs, sB, BACK ? steps[wave].u : steps[wave].v, BACK ? d.from : d.to, d.whole);
    total += d.total;
  }
  if (unit.idle) return;
  const uint64_t slot = (uint64_t)unit.piece * a.heads + head;
  put_state<NT, PW>(h, a.starts + slot * a.dim * a.state + (uint64_t)unit.p0 * a.state, dim, a.state, a.state_wide);
  if (lane0 == 0 && unit.p0 == 0) a.totals[slot] = total;
}

constexpr uint32_t kAhead = 8;  // pieces that a join reads before it sums them

}  // namespace trunk
