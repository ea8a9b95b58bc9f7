// tiles.h - products of two matrices by tiles of 256 x 128: what the head's kernels share.
//
// A block of four wavefronts takes a tile of 256 x 128 sums, each wavefront 128 x 64 of it in 128
// registers a lane, as 4 x 2 results of 32 x 32 of the matrix instruction. Both operands come by
// stages of 64 bytes of the summed axis (32 bf16 or 16 f32) through LDS: 24 KB a stage, three of
// them, written by loads that go past the registers, so that two blocks share a compute unit and
// one's matrix instructions run through the other's epilogue and barriers.
//
// An operand lies along the summed axis (its values for one row or column of the result next to each
// other) or across it (a row apart). Along, a stage's rows are 64 bytes, and a lane reads the 16 bytes
// that the matrix instruction wants of it; across, they come out of LDS by transposing reads (bf16) or
// a value at a time (f32). 16-byte pieces of a row are dealt over its places by an exclusive or with
// the row's number, so that no two of the lanes that read at once meet in a bank.
//
// Any order of the summed axis is right that both operands share: an f32 lane's 16 bytes are four
// values of four matrix instructions of two.
#pragma once
#include "trunk.h"

namespace trunk {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kTileM = 256, kTileN = 128, kStages = 3;
constexpr int kStageBytes = (kTileM + kTileN) * 64, kLdsBytes = kStages * kStageBytes;
constexpr uint32_t kNowhere = 0x80000000u;  // an offset that no buffer has: the load gives zeros
template <class T>
constexpr int kVec = 16 / sizeof(T);  // values of 16 bytes
template <class T>
constexpr int kDeep = 64 / sizeof(T);  // values of the summed axis in a stage

// What a lane holds of an operand: 16 bytes.
template <class T>
struct Piece16;
template <>
struct Piece16<bf16> {
  using V = bf16x8;
};
template <>
struct Piece16<float> {
  using V = f32x4;
};
template <class T>
using Part = typename Piece16<T>::V;

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
// The row of a 32 x 32 result that a lane's r-th value has; its column is lane % 32.
__device__ __forceinline__ int row_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }
// -inf in the place of sums whose row is `limit` or more from the wavefront's first.
__device__ __forceinline__ void cut_rows(f32x16 (&z)[4][2], uint32_t limit, int half) {
  const int own = (int)limit - 4 * half;
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const bool there = 32 * i + row_of(r, 0) < own;
      z[i][0][r] = there ? z[i][0][r] : -__builtin_inff(), z[i][1][r] = there ? z[i][1][r] : -__builtin_inff();
    }
}

// The places of 16-byte pieces in a row of a stage: piece c lies at c ^ twist(row).
template <class T, bool ALONG>
__device__ __forceinline__ uint32_t twist(uint32_t row) {
  if constexpr (ALONG) return (row >> 2) & 3;          // 16 rows of 64 bytes cover the banks four times
  else if constexpr (sizeof(T) == 2) return (row & 3) << 2;  // four rows are read at once, 64 bytes each
  else return ((row >> 2) & 1) << 3;                   // two rows four apart, 128 bytes each
}

// A stage of both operands to LDS at `to` (the wavefront's own place of it), past the registers: the 256 rows'
// four loads, the 128 rows' two, each 4 KB of the block. The wait for them is the caller's. The first wait is
// between what may have written the buffers' scalar registers and the loads that read them, the others
// between m0 and the loads that take it.
__device__ __forceinline__ void to_lds(uint32_t to, u32x4 a, const uint32_t (&at)[4], u32x4 b, const uint32_t (&bt)[2]) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %7, 0 offen lds\n\t"
      "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %7, 0 offen lds\n\t"
      "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %7, 0 offen lds\n\t"
      "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %7, 0 offen lds\n\t"
      "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %8, 0 offen lds\n\t"
      "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\tbuffer_load_dwordx4 %6, %8, 0 offen lds"
      ::"s"(to), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(bt[0]), "v"(bt[1]), "s"(a), "s"(b)
      : "memory", "scc");
}
__device__ __forceinline__ u32x4 buffer_at(const char *base) {
  const uint64_t at = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  return u32x4{lo, hi & 0xffffu, 0x7fffffffu, 0x00020000u};
}

// One operand's way into LDS. Its R rows (columns of the result's, for the second operand) times the
// stage's depth; what is past `there` of them or past the summed axis's `depth` is read as zeros.
template <class T, bool ALONG, int R>
struct Feed {
  static constexpr int kJobs = R * 4 / 256;  // loads a lane and stage
  static constexpr int kRow = ALONG ? 4 : R * (int)sizeof(T) / 16, kRows = 256 / kRow;  // pieces of a row, rows a load of the block
  const char *base;
  int64_t step;
  uint32_t off[kJobs];
  int left;
  // `pitch` bytes from row to row in memory; 256 of them are under 2^31. `base` is aligned to 16.
  __device__ __forceinline__ void start(const T *from, int64_t pitch, uint32_t there, uint32_t depth) {
    base = (const char *)from;
    step = ALONG ? 64 : kDeep<T> * pitch;
    const uint32_t row = threadIdx.x / kRow, place = threadIdx.x % kRow;
    left = (int)depth - (int)(ALONG ? (place ^ twist<T, true>(row)) * kVec<T> : row);
#pragma unroll
    for (int i = 0; i < kJobs; i++) {
      const uint32_t r = row + i * kRows, c = place ^ twist<T, ALONG>(r);  // along: the same in all of them
      off[i] = (ALONG ? r : c * kVec<T>) < there ? r * (uint32_t)pitch + c * 16 : kNowhere;
    }
  }
  __device__ __forceinline__ void nothing() { left = -(1 << 30); }
  // The next stage's buffer and offsets.
  __device__ __forceinline__ u32x4 next(uint32_t (&at)[kJobs]) {
    const u32x4 from = buffer_at(base);
#pragma unroll
    for (int i = 0; i < kJobs; i++) at[i] = left > (ALONG ? 0 : i * kRows) ? off[i] : kNowhere;
    base += step;
    left -= kDeep<T>;
    return from;
  }
};

// One operand's way out of LDS: N tiles of 32 from the wavefront's first one on.
template <class T, bool ALONG, int R, int N>
struct Reader {
  static constexpr int kPitch = ALONG ? 64 : R * (int)sizeof(T);
  uint32_t at[ALONG ? 2 : N];
  __device__ __forceinline__ void start(int lane, int first) {
    const uint32_t half = lane >> 5, i32 = lane & 31, j = lane & 15;
    if constexpr (ALONG) {
#pragma unroll
      for (uint32_t s = 0; s < 2; s++) at[s] = (first * 32 + i32) * 64 + (((2 * s + half) ^ twist<T, true>(i32)) * 16);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t row = 8 * half + (j >> 2), c = (4 * (first + i) + (i32 >> 4) * 2 + ((j & 3) >> 1)) ^ twist<T, false>(row);
          at[i] = row * kPitch + c * 16 + 8 * (j & 1);
        } else {
          const uint32_t c = (8 * (first + i) + (i32 >> 2)) ^ twist<T, false>(4 * half);
          at[i] = 4 * half * kPitch + c * 16 + (i32 & 3) * 4;
        }
      }
    }
  }
  // The i-th tile's part of the stage's first or second half.
  __device__ __forceinline__ Part<T> get(const char *stage, int s, int i) const {
    if constexpr (ALONG) {
      return *(const Part<T> *)(stage + at[s] + i * 2048);
    } else if constexpr (sizeof(T) == 2) {
      using Local = __attribute__((address_space(3))) bf16x4;
      const char *from = stage + at[i] + s * 16 * kPitch;
      const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local *)from);
      const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local *)(from + 4 * kPitch));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const char *from = stage + at[i] + s * 8 * kPitch;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = *(const float *)(from + e * kPitch);
      return v;
    }
  }
};

// A block's tiles one after another. `work` says how many there are and of how many stages each
// (tiles, stages), gives the feeds of the n-th (feed(n, a, b)) and takes its sums (take(n, sums)). The loads
// run two stages ahead, over a tile's end into the next.
template <class T, bool A_ALONG, bool B_ALONG, class Work>
__device__ __forceinline__ void run_tiles(char *lds, Work &work) {
  Feed<T, A_ALONG, kTileM> fa;
  Feed<T, B_ALONG, kTileN> fb;
  Reader<T, A_ALONG, kTileM, 4> ra;
  Reader<T, B_ALONG, kTileN, 2> rb;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  ra.start(lane, 4 * (wave >> 1));
  rb.start(lane, 2 * (wave & 1));
  const uint32_t tiles = work.tiles, stages = work.stages;
  if (!stages) {  // sums over nothing
    for (uint32_t n = 0; n < tiles; n++) {
      f32x16 sums[4][2] = {};
      work.take(n, sums);
    }
    return;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  uint32_t ahead_tile = 0, ahead = 0, put = 0;
  work.feed(0, fa, fb);
  auto issue = [&]() {
    uint32_t at[4], bt[2];
    const u32x4 a = fa.next(at), b = fb.next(bt);
    to_lds(lds0 + put + wave * 1024, a, at, b, bt);
    put = put == (kStages - 1) * kStageBytes ? 0 : put + kStageBytes;
    if (++ahead == stages) {
      ahead = 0;
      if (++ahead_tile < tiles) work.feed(ahead_tile, fa, fb);
      else fa.nothing(), fb.nothing();
    }
  };
  issue();
  issue();
  uint32_t from = 0;
  for (uint32_t n = 0; n < tiles; n++) {
    f32x16 sums[4][2] = {};
    for (uint32_t k = 0; k < stages; k++) {
      // This stage's loads are all but the last six; everyone has read the stage that is written next.
      asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      issue();
      const char *stage = lds + from;
      from = from == (kStages - 1) * kStageBytes ? 0 : from + kStageBytes;
#pragma unroll
      for (int s = 0; s < 2; s++) {
        Part<T> a[4], b[2];
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = ra.get(stage, s, i);
#pragma unroll
        for (int i = 0; i < 2; i++) b[i] = rb.get(stage + kTileM * 64, s, i);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) sums[i][j] = mma32(a[i], b[j], sums[i][j]);
      }
    }
    work.take(n, sums);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the loads that run ahead of the last tile
}

}  // namespace trunk
