// scan.h - what the scan's kernels share: products on the matrix cores, a call's arguments, which block
// takes which piece, and what a cut sequence's pieces are joined by.
#pragma once
#include "trunk.h"

namespace trunk {

constexpr int kChunk = 64;    // rows of a chunk: four tiles of 16
constexpr int kThreads = 256; // four wavefronts

// 16 x 16 products over 32 places. A lane holds eight values of its operand's row (lane % 16),
// places 8 (lane / 16) .. + 7, or for an operand built from two result tiles places 4 (lane / 16)
// .. + 3 of the first and of the second: any order of the places is right if both operands have
// the same. A lane's four results are rows 4 (lane / 16) + r of column lane % 16.

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
  static __device__ __forceinline__ f32x4 mul(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
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
  float *starts;         // [later][heads][dim][state]: where a sequence's pieces after its first begin, if any are cut; or NULL
  double *totals;        // [later][heads]: log2 of a piece's whole decay
  uint32_t *order;       // the pieces, longest first: how many, and from the third on sequence and number; or NULL
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

int check_scan(const uor_trunk_scan_args *s, bool step);
Scan scan_of(const uor_trunk_scan_args *s, uint32_t size);
// The block's piece, in the pieces' order or the call's; `number` is then its place among all pieces.
__device__ __forceinline__ bool next_piece(const Scan &a, uint32_t &number, Piece &at) {
  if (number >= a.pieces) return false;
  if (!a.order) return piece<true>(a.rows, number, a.size, at);
  if (number >= a.order[0]) return false;
  const uint32_t *place = a.order + 2 + 2 * number;
  at = piece_of(a.rows, place[0], place[1], a.size);
  number = at.start / a.size + at.seq + at.number;
  return true;
}

// The place of the piece that follows in the sequence; a piece's own is one less.
__device__ __forceinline__ uint64_t next_place(const Scan &a, const Piece &at) { return (uint64_t)(at.start / a.size) + at.number; }

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
