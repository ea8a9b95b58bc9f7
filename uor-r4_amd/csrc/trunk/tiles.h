// tiles.h - products of two matrices by tiles of 256 x 128 (or 128 x 64, or 64 x 64): what the head's kernels share.
//
// A block of four wavefronts takes a tile of 256 x 128 sums, each wavefront 128 x 64 of it in 128
// registers a lane, as 4 x 2 results of 32 x 32 of the matrix instruction. Both operands come by
// stages of 64 bytes of the summed axis (32 bf16 or 16 f32) through LDS: 24 KB a stage, three of
// them, written by loads that go past the registers, so that two blocks share a compute unit and
// one's matrix instructions run through the other's epilogue and barriers.
//
// Matrices that the kernels lay out themselves lie by panels: 64 bytes of each row, row after row, and then the rows'
// next 64 bytes. A stage's part of 256 rows is then 16 KB in one piece along the summed axis, and 2 KB pieces across.
// Rows that lie 2 KB apart are read by half lines of the caches, every line twice: 8,192 x 131,072 logits of width
// 1,024 took 333 M requests to the L2 caches as rows and 201 M as panels (2.01 and 1.92 ms).
//
// An operand lies along the summed axis (its values for one row or column of the result next to each
// other) or across it (a row apart). Along, a stage's rows are 64 bytes, and a lane reads the 16 bytes
// that the matrix instruction wants of it; across, they come out of LDS by transposing reads (bf16) or
// a value at a time (f32). 16-byte pieces of a row are dealt over its places by an exclusive or with
// the row's number, so that no two of the lanes that read at once meet in a bank.
//
// In 32 bits the sums of 128 values at a time are added to a second set of sums, so that the errors of long sums are those
// of their 128ths. Operands of 32 bits as three planes of bf16 and six products of them ran 1.4 times as fast for 4,096
// rows of 512, half as fast for up to 100, and up to 6 times further from 64 bits; they are not used.
//
// Any order of the summed axis is right that both operands share: an f32 lane's 16 bytes are four
// values of four matrix instructions of two.
#pragma once
#include "trunk.h"

namespace trunk {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kStages = 3;
// A block's tile: 2 x 2 wavefronts of M x N results of 32 x 32.
template <int M_, int N_>
struct Shape {
  static constexpr int M = M_, N = N_, kM = 64 * M, kN = 64 * N, kLoads = M + N;
  static constexpr int kStageBytes = (kM + kN) * 64, kLdsBytes = kStages * kStageBytes;
  static constexpr int kBlocks = M * N > 4 ? 2 : 4;  // that share a compute unit
};
using Large = Shape<4, 2>;
using Small = Shape<2, 1>;
using Tiny = Shape<1, 1>;
constexpr int kRound = 256;  // rows and words are rounded up to whole large tiles
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
template <int M, int N>
__device__ __forceinline__ void cut_rows(f32x16 (&z)[M][N], uint32_t limit, int half) {
  const int own = (int)limit - 4 * half;
#pragma unroll
  for (int i = 0; i < M; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const bool there = 32 * i + row_of(r, 0) < own;
#pragma unroll
      for (int j = 0; j < N; j++) z[i][j][r] = there ? z[i][j][r] : -__builtin_inff();
    }
}

// The places of 16-byte pieces in a row of a stage: piece c lies at c ^ twist(row). R: the operand's rows (columns).
template <class T, bool ALONG, int R>
__device__ __forceinline__ uint32_t twist(uint32_t row) {
  if constexpr (ALONG) return (row >> 2) & 3;                           // 16 rows of 64 bytes cover the banks four times
  else if constexpr (sizeof(T) == 4) return ((row >> 2) & 1) << 3;      // two rows four apart are read at once, 128 bytes each
  else if constexpr (R >= 128) return (row & 3) << 2;                   // four rows, 64 bytes each, that lie 256 bytes or more apart
  else return ((row >> 1) & 1) << 2;                                    // or 128
}

// A stage of both operands to LDS at `to` (the wavefront's own place of it), past the registers: the first one's
// loads, then the second one's, each 4 KB of the block. The wait for them is the caller's. The first wait is
// between what may have written the buffers' scalar registers and the loads that read them, the others
// between m0 and the loads that take it.
#define LOAD(at, buffer) "buffer_load_dwordx4 " at ", " buffer ", 0 offen lds\n\t"
#define NEXT "s_add_u32 m0, m0, 0x1000\n\ts_nop 0\n\t"
__device__ __forceinline__ void to_lds(uint32_t to, u32x4 a, const uint32_t (&at)[4], u32x4 b, const uint32_t (&bt)[2]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" LOAD("%1", "%7") NEXT LOAD("%2", "%7") NEXT LOAD("%3", "%7") NEXT LOAD("%4", "%7") NEXT LOAD(
                   "%5", "%8") NEXT LOAD("%6", "%8")
               ::"s"(to), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(bt[0]), "v"(bt[1]), "s"(a), "s"(b)
               : "memory", "scc");
}
__device__ __forceinline__ void to_lds(uint32_t to, u32x4 a, const uint32_t (&at)[2], u32x4 b, const uint32_t (&bt)[1]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" LOAD("%1", "%4") NEXT LOAD("%2", "%4") NEXT LOAD("%3", "%5")
               ::"s"(to), "v"(at[0]), "v"(at[1]), "v"(bt[0]), "s"(a), "s"(b)
               : "memory", "scc");
}
__device__ __forceinline__ void to_lds(uint32_t to, u32x4 a, const uint32_t (&at)[1], u32x4 b, const uint32_t (&bt)[1]) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" LOAD("%1", "%3") NEXT LOAD("%2", "%4")
               ::"s"(to), "v"(at[0]), "v"(bt[0]), "s"(a), "s"(b)
               : "memory", "scc");
}
#undef LOAD
#undef NEXT
__device__ __forceinline__ u32x4 buffer_at(const char *base) {
  const uint64_t at = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  return u32x4{lo, hi & 0xffffu, 0x7fffffffu, 0x00020000u};
}

// How a matrix lies in memory: row after row, `pitch` bytes apart, or by panels, which are `pitch` bytes apart.
enum Lies { ROWS, PANELS };

// One operand's way into LDS. Its R rows (columns of the result's, for the second operand) times the
// stage's depth; what is past `there` of them or past the summed axis's `depth` is read as zeros.
template <class T, bool ALONG, Lies LIES, int R>
struct Feed {
  static constexpr int kJobs = R * 4 / 256;  // loads a lane and stage
  static constexpr int kRow = ALONG ? 4 : R * (int)sizeof(T) / 16, kRows = 256 / kRow;  // pieces of a row, rows a load of the block
  const char *base;
  int64_t step;
  uint32_t off[kJobs];
  int left;
  // `from` is the operand's first value, aligned to 16 bytes (to a panel's row where panels are read across).
  // What an operand's rows (256 of them), or its panels, cover in memory is under 2^31 bytes.
  __device__ __forceinline__ void start(const char *from, int64_t pitch, uint32_t there, uint32_t depth) {
    base = from;
    step = ALONG ? (LIES == ROWS ? 64 : pitch) : kDeep<T> * (LIES == ROWS ? pitch : 64);
    const uint32_t row = threadIdx.x / kRow, place = threadIdx.x % kRow;
    left = (int)depth - (int)(ALONG ? (place ^ twist<T, true, R>(row)) * kVec<T> : row);
#pragma unroll
    for (int i = 0; i < kJobs; i++) {
      const uint32_t r = row + i * kRows, c = place ^ twist<T, ALONG, R>(r);  // along: the same in all of them
      const uint32_t at = LIES == ROWS ? r * (uint32_t)pitch + c * 16 : r * 64 + (c & 3) * 16 + (ALONG ? 0 : (c >> 2) * (uint32_t)pitch);
      off[i] = (ALONG ? r : c * kVec<T>) < there ? at : kNowhere;
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
      for (uint32_t s = 0; s < 2; s++) at[s] = (first * 32 + i32) * 64 + (((2 * s + half) ^ twist<T, true, R>(i32)) * 16);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t row = 8 * half + (j >> 2), c = (4 * (first + i) + (i32 >> 4) * 2 + ((j & 3) >> 1)) ^ twist<T, false, R>(row);
          at[i] = row * kPitch + c * 16 + 8 * (j & 1);
        } else {
          const uint32_t c = (8 * (first + i) + (i32 >> 2)) ^ twist<T, false, R>(4 * half);
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

// A block's tiles one after another. `work` says how many there are (tiles) and of how many stages each (stages(n)), gives the
// feeds of the n-th (feed(n, a, b)) and takes its sums (take(n, sums), with kStores
// stores at least to memory). The loads run two stages ahead, over a tile's end into the next. Loads and stores end in
// their order, so that behind a tile's stores the next two stages wait for loads alone: with a wait for the stores
// too, 8,192 x 16,384 logits of width 1,024 and their G took 372 us, without 348.
template <class T, class S, bool A_ALONG, Lies A_LIES, bool B_ALONG, Lies B_LIES, class Work>
__device__ __forceinline__ void run_tiles(char *lds, Work &work) {
  Feed<T, A_ALONG, A_LIES, S::kM> fa;
  Feed<T, B_ALONG, B_LIES, S::kN> fb;
  Reader<T, A_ALONG, S::kM, S::M> ra;
  Reader<T, B_ALONG, S::kN, S::N> rb;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  ra.start(lane, S::M * (wave >> 1));
  rb.start(lane, S::N * (wave & 1));
  const uint32_t tiles = work.tiles;
  if (!tiles) return;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  uint32_t ahead_tile = 0, ahead = work.stages(0), put = 0;
  work.feed(0, fa, fb);
  auto issue = [&]() {
    uint32_t at[S::M], bt[S::N];
    const u32x4 a = fa.next(at), b = fb.next(bt);
    to_lds(lds0 + put + wave * 1024, a, at, b, bt);
    put = put == (kStages - 1) * S::kStageBytes ? 0 : put + S::kStageBytes;
    if (!--ahead) {
      if (++ahead_tile < tiles) ahead = work.stages(ahead_tile), work.feed(ahead_tile, fa, fb);
      else fa.nothing(), fb.nothing();
    }
  };
  issue();
  issue();
  uint32_t from = 0, stored = 0;
  constexpr bool kFold = sizeof(T) == 4;
  static_assert(!kFold || S::M * S::N <= 4, "no registers for two sets of sums");
  for (uint32_t n = 0; n < tiles; n++) {
    f32x16 sums[S::M][S::N] = {}, folded[kFold ? S::M : 1][kFold ? S::N : 1] = {};
    const uint32_t stages = work.stages(n);
    for (uint32_t k = 0; k < stages; k++) {
      if (kFold && k && k % 8 == 0) {
#pragma unroll
        for (int i = 0; i < S::M; i++)
#pragma unroll
          for (int j = 0; j < S::N; j++) folded[kFold ? i : 0][kFold ? j : 0] += sums[i][j], sums[i][j] = f32x16{};
      }
      // This stage's loads are all but the last stage's; everyone has read the stage that is written next.
      if (Work::kStores && stored) {
        stored--;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads + Work::kStores) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads) : "memory");
      }
      issue();
      const char *stage = lds + from;
      from = from == (kStages - 1) * S::kStageBytes ? 0 : from + S::kStageBytes;
#pragma unroll
      for (int s = 0; s < 2; s++) {
        Part<T> a[S::M], b[S::N];
#pragma unroll
        for (int i = 0; i < S::M; i++) a[i] = ra.get(stage, s, i);
#pragma unroll
        for (int i = 0; i < S::N; i++) b[i] = rb.get(stage + S::kM * 64, s, i);
#pragma unroll
        for (int i = 0; i < S::M; i++)
#pragma unroll
          for (int j = 0; j < S::N; j++) sums[i][j] = mma32(a[i], b[j], sums[i][j]);
      }
    }
    if constexpr (kFold) {
#pragma unroll
      for (int i = 0; i < S::M; i++)
#pragma unroll
        for (int j = 0; j < S::N; j++) sums[i][j] += folded[i][j];
    }
    work.take(n, sums);
    stored = 2;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the loads that run ahead of the last tile
}

}  // namespace trunk
