// scan.hip - the selective state space scan over packed sequences: outputs and final states.
//
// One block takes one head of one piece of a sequence, chunk after chunk, with the head's state in
// registers (its transpose as result tiles: rows of the state's axis, a column a value of x) and a
// copy of it as operand parts in LDS. A wavefront owns 16 rows of the chunk for y and a part of the
// state's tiles for the update. The scores C_t . B_s are computed with s along the tile's rows, so
// that a lane's results are, once scaled, its operand of the next product over s.
//
// Rows are bound by time, not by products: a sequence of many rows and few heads would run on few
// blocks. Such sequences are cut into pieces: a first launch gives every piece its end state from
// zeros, a second joins them along the sequence, and the main launch runs all pieces at once.
#include "scan.h"

namespace trunk {

// The parts of the state as an operand, [part][16 PW][16 NT].
template <class T, int NT, int PW>
__device__ __forceinline__ void publish(T *to, const f32x4 (&h)[NT * PW / 4], const Own<NT, PW> &own) {
  const int lane = threadIdx.x & 63, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < NT * PW / 4; i++) {
    T *row = to + (own.p * 16 + (lane & 15)) * pitch<T>(16 * NT) + (own.n + i) * 16 + 4 * q;
    if constexpr (Mma<T>::kParts == 1) {
      *(f32x4 *)row = h[i];
    } else {
      bf16x4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; r++) hi[r] = (bf16)h[i][r];
#pragma unroll
      for (int r = 0; r < 4; r++) lo[r] = (bf16)(h[i][r] - (float)hi[r]);
      *(bf16x4 *)row = hi;
      *(bf16x4 *)(row + 16 * PW * pitch<T>(16 * NT)) = lo;
    }
  }
}

template <class T, int NT, int PW>
__global__ __launch_bounds__(kThreads) void scan_rows(Scan a) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kNp = pitch<T>(kN), kLp = pitch<T>(kChunk);
  __shared__ __align__(16) T sB[kChunk * kNp], sC[kChunk * kNp], sBt[kN * kLp], sXt[kP * kLp], sH[Mma<T>::kParts * kP * kNp];
  __shared__ Decays d;
  __shared__ int odd;

  uint32_t number, head;
  place_of(blockIdx.x, a.heads * a.tiles, number, head);
  const uint32_t p0 = head % a.tiles * kP;
  head /= a.tiles;
  Piece at;
  if (number >= a.pieces || !piece(a.rows, number, a.size, at)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
  const uint32_t group = head / (a.heads / a.groups);
  const T *x = (const T *)a.x + head * a.dim + p0, *dt = (const T *)a.dt + head;
  const T *B = (const T *)a.B + group * a.state, *C = (const T *)a.C + group * a.state;
  T *y = (T *)a.y + head * a.dim + p0;
  const uint32_t dim = a.dim - p0 < (uint32_t)kP ? a.dim - p0 : kP;
  const float A = a.A[head], skip = a.D ? a.D[head] : 0.0f, bias = a.bias ? a.bias[head] : 0.0f;
  const uint64_t whole = (uint64_t)a.dim * a.state;
  const Own<NT, PW> own;
  f32x4 h[NT * PW / 4];
  load_state<NT, PW>(h, own,
                     a.starts ? a.starts + ((uint64_t)number * a.heads + head) * whole
                              : a.initial ? a.initial + ((uint64_t)at.seq * a.heads + head) * whole : nullptr,
                     p0, a.dim, a.state);

  for (uint32_t first = at.first; first < at.end; first += kChunk) {
    const uint32_t end = at.end - first > kChunk ? first + kChunk : at.end;
    __syncthreads();  // the chunk before has been read
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    stage<T, kN>(sB, sBt, B, a.b_stride, first, end, a.state, a.b_wide);
    stage<T, kN>(sC, (T *)nullptr, C, a.c_stride, first, end, a.state, a.c_wide);
    if (stage<T, kP>((T *)nullptr, sXt, x, a.x_stride, first, end, dim, a.x_wide)) odd = 1;
    publish<T, NT, PW>(sH, h, own);
    if (wave == 0) decays(d, dt, a.dt_stride, first, end, A, bias);
    __syncthreads();

    // y's rows of this wavefront, transposed: what comes from the state before the chunk.
    const int t = wave * 16 + i16;
    f32x4 acc[PW];
#pragma unroll
    for (int i = 0; i < PW; i++) acc[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kN; k += 32) {
      const V8<T> c = operand(sC + t * kNp, k + 8 * q);
#pragma unroll
      for (int i = 0; i < PW; i++)
#pragma unroll
        for (int part = Mma<T>::kParts - 1; part >= 0; part--)
          acc[i] = Mma<T>::mul(operand(sH + (part * kP + i * 16 + i16) * kNp, k + 8 * q), c, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < PW; i++) acc[i] *= d.from[t];
    // What comes from the chunk's own rows, two tiles of 16 at a time.
    const float hi = d.hi[t], lo = d.lo[t];
#pragma unroll
    for (int pair = 0; pair < 2; pair++) {
      if (2 * pair > wave) break;
      f32x8 m;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int s0 = (2 * pair + half) * 16;
        f32x4 score = {0, 0, 0, 0};
        if (2 * pair + half <= wave) {
#pragma unroll
          for (int k = 0; k < kN; k += 32)
            score = Mma<T>::mul(operand(sB + (s0 + i16) * kNp, k + 8 * q), operand(sC + t * kNp, k + 8 * q), score);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int s = s0 + 4 * q + r;
          const float decay = exp2_((hi - d.hi[s]) + (lo - d.lo[s])) * d.step[s];
          m[4 * half + r] = s < t ? score[r] * decay : s == t ? score[r] * d.step[s] + skip : 0.0f;
        }
      }
      const auto w = Mma<T>::split(m);
      if (odd == 0) {
#pragma unroll
        for (int i = 0; i < PW; i++)
          acc[i] = Mma<T>::mul(operand_tiles(sXt + (i * 16 + i16) * kLp, pair * 32 + 4 * q), w, acc[i]);
      } else {
        // Some x of the chunk is infinite or no number: its products with the zeros above the
        // diagonal would reach rows before it. Such values are left out of the product, and added to
        // the rows from their own on one by one.
#pragma unroll
        for (int i = 0; i < PW; i++) {
          V8<T> v = operand_tiles(sXt + (i * 16 + i16) * kLp, pair * 32 + 4 * q);
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = finite((float)v[e]) ? v[e] : (T)0.0f;
          acc[i] = Mma<T>::mul(v, w, acc[i]);
        }
#pragma unroll 1
        for (int s = pair * 32; s < pair * 32 + 32; s++) {
          const int from = ((s & 15) >> 2) * 16 + i16, at = (s & 16 ? 4 : 0) + (s & 3);
          float mine = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) mine = e == at ? __shfl(m[e], from) : mine;
          if (s > t) continue;
#pragma unroll
          for (int i = 0; i < PW; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const float v = (float)sXt[(i * 16 + 4 * q + r) * kLp + s];
              if (!finite(v)) acc[i][r] += mine * v;
            }
        }
      }
    }
    if (first + t < end) {
      T *row = y + (int64_t)(first + t) * a.y_stride;
#pragma unroll
      for (int i = 0; i < PW; i++) {
        const uint32_t p = i * 16 + 4 * q;
        V4<T> v;
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = (T)acc[i][r];
        if (a.y_wide && p + 4 <= dim) {
          *(V4<T> *)(row + p) = v;
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (p + r < dim) row[p + r] = v[r];
        }
      }
    }
    advance<T, NT, PW>(h, own, sXt, sBt, d.to, d.whole);
  }
  if (a.final && at.end == at.stop)
    store_state<NT, PW>(h, own, a.final + ((uint64_t)at.seq * a.heads + head) * whole, p0, a.dim, a.state);
}

// A piece's end state from zeros and its whole decay; a sequence's last piece needs neither.
template <class T, int NT, int PW>
__global__ __launch_bounds__(kThreads) void scan_ends(Scan a) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kLp = pitch<T>(kChunk);
  __shared__ __align__(16) T sBt[kN * kLp], sXt[kP * kLp];
  __shared__ Decays d;
  uint32_t number, head;
  place_of(blockIdx.x, a.heads * a.tiles, number, head);
  const uint32_t p0 = head % a.tiles * kP;
  head /= a.tiles;
  Piece at;
  if (number >= a.pieces || !piece(a.rows, number, a.size, at) || at.end == at.stop) return;
  const int wave = threadIdx.x >> 6;
  const uint32_t group = head / (a.heads / a.groups);
  const T *x = (const T *)a.x + head * a.dim + p0, *dt = (const T *)a.dt + head, *B = (const T *)a.B + group * a.state;
  const uint32_t dim = a.dim - p0 < (uint32_t)kP ? a.dim - p0 : kP;
  const float A = a.A[head], bias = a.bias ? a.bias[head] : 0.0f;
  const Own<NT, PW> own;
  f32x4 h[NT * PW / 4];
#pragma unroll
  for (int i = 0; i < NT * PW / 4; i++) h[i] = f32x4{0, 0, 0, 0};
  double total = 0.0;
  for (uint32_t first = at.first; first < at.end; first += kChunk) {
    const uint32_t end = at.end - first > kChunk ? first + kChunk : at.end;
    __syncthreads();
    stage<T, kN>((T *)nullptr, sBt, B, a.b_stride, first, end, a.state, a.b_wide);
    stage<T, kP>((T *)nullptr, sXt, x, a.x_stride, first, end, dim, a.x_wide);
    if (wave == 0) decays(d, dt, a.dt_stride, first, end, A, bias);
    __syncthreads();
    advance<T, NT, PW>(h, own, sXt, sBt, d.to, d.whole);
    total += d.total;
  }
  const uint64_t slot = (uint64_t)number * a.heads + head;
  store_state<NT, PW>(h, own, a.starts + slot * a.dim * a.state, p0, a.dim, a.state);
  if (threadIdx.x == 0 && p0 == 0) a.totals[slot] = total;
}

// The pieces' end states into their start states, along each sequence.
__global__ __launch_bounds__(kThreads) void scan_join(Scan a) {
  const uint32_t seq = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  uint32_t start, end;
  a.rows.of(seq, start, end);
  const uint32_t n = end > start ? (end - start - 1) / a.size + 1 : 1;
  const uint64_t base = start / a.size + seq, whole = (uint64_t)a.dim * a.state;
  for (uint64_t e = blockIdx.y * kThreads + threadIdx.x; e < whole; e += (uint64_t)gridDim.y * kThreads) {
    float h = a.initial ? a.initial[((uint64_t)seq * a.heads + head) * whole + e] : 0.0f;
    for (uint32_t j = 0; j < n; j++) {
      const uint64_t slot = (base + j) * a.heads + head;
      float *at = a.starts + slot * whole + e;
      if (j + 1 == n) {
        *at = h;
        break;
      }
      const float own = *at;
      *at = h;
      h = exp2_((float)a.totals[slot]) * h + own;
    }
  }
}

// How many rows a piece has: sequences are cut where heads alone would leave the card idle. The
// grid then has about 1,024 blocks; pieces under 256 rows cost more to join than they gain.
uint32_t piece_rows(uint32_t tokens, uint32_t heads) {
  const uint64_t want = ((uint64_t)tokens * heads + 1023) / 1024;
  const uint64_t size = (want < 256 ? 256 : want) + kChunk - 1;
  const uint64_t rows = size / kChunk * kChunk;
  return rows < tokens ? (uint32_t)rows : (tokens + kChunk) / kChunk * kChunk;
}

namespace {

template <class T, int NT, int PW>
int launch(const Scan &a, uint32_t seqs, hipStream_t stream) {
  const uint32_t blocks = grid_of(a.pieces, a.heads * a.tiles);
  if (a.starts) {
    hipLaunchKernelGGL((scan_ends<T, NT, PW>), dim3(blocks), dim3(kThreads), 0, stream, a);
    const uint32_t parts = (a.dim * a.state + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(scan_join, dim3(seqs * a.heads, parts), dim3(kThreads), 0, stream, a);
  }
  hipLaunchKernelGGL((scan_rows<T, NT, PW>), dim3(blocks), dim3(kThreads), 0, stream, a);
  return launched();
}
template <class T, int NT>
int launch(const Scan &a, uint32_t seqs, hipStream_t stream) {
  return a.dim <= 32 ? launch<T, NT, 2>(a, seqs, stream) : launch<T, NT, 4>(a, seqs, stream);
}
template <class T>
int launch(const Scan &a, uint32_t seqs, hipStream_t stream) {
  return a.state <= 32 ? launch<T, 2>(a, seqs, stream) : a.state <= 64 ? launch<T, 4>(a, seqs, stream) : launch<T, 8>(a, seqs, stream);
}

uint64_t starts_bytes(uint64_t pieces, const uor_trunk_scan_args *s) {
  return (pieces * s->heads * s->dim * s->state * 4 + 15) / 16 * 16;
}

}  // namespace

// What every call of the scan asks of its sizes and rows.
int check_scan(const uor_trunk_scan_args *s, bool step) {
  if (!s) return fail(-1, "null argument");
  if (s->dtype > UOR_TRUNK_F32) return fail(-1, "dtype %u is neither bf16 nor f32", s->dtype);
  if (s->heads < 1 || s->groups < 1 || s->heads % s->groups) return fail(-1, "%u heads are not whole groups of %u", s->heads, s->groups);
  if (s->heads > 65535) return fail(-1, "%u heads: at most 65535", s->heads);
  if (s->dim < 1 || s->dim > UOR_TRUNK_MAX_DIM) return fail(-1, "dim %u outside 1..128", s->dim);
  if (s->state < 1 || s->state > UOR_TRUNK_MAX_STATE) return fail(-1, "state %u outside 1..128", s->state);
  if (s->tokens > 0x7fffffffu - 64) return fail(-1, "%u rows: too many", s->tokens);
  if (!step && (s->seqs < 1 || s->seqs > 0x7fffffffu / s->heads)) return fail(-1, "%u sequences", s->seqs);
  if (!step && !s->offsets && s->seqs != 1) return fail(-1, "%u sequences without offsets", s->seqs);
  if (s->tokens && (!s->x || !s->dt || !s->B || !s->C)) return fail(-1, "null rows");
  if (!s->A) return fail(-1, "null A");
  const int64_t inner = (int64_t)s->heads * s->dim, shared = (int64_t)s->groups * s->state;
  if (s->tokens > 1 && (s->x_stride < inner || s->y_stride < inner || s->dt_stride < s->heads || s->b_stride < shared || s->c_stride < shared))
    return fail(-1, "rows overlap: a stride is less than a row");
  return 0;
}
// A call's arguments as the kernels take them, cut into pieces of `size` rows.
Scan scan_of(const uor_trunk_scan_args *s, uint32_t size) {
  const uint32_t bytes = s->dtype == UOR_TRUNK_BF16 ? 2 : 4;
  const auto wide = [&](const void *p, int64_t stride, uint32_t part) { return aligned16(p, stride, bytes) && part * bytes % 16 == 0; };
  Scan a{};
  a.rows = Rows{s->offsets, s->tokens, s->seqs};
  a.heads = s->heads, a.groups = s->groups, a.dim = s->dim, a.state = s->state;
  a.size = size, a.pieces = pieces(s->tokens, s->seqs, size), a.tiles = tiles_of(s->dim);
  a.x_stride = s->x_stride, a.dt_stride = s->dt_stride, a.b_stride = s->b_stride, a.c_stride = s->c_stride, a.y_stride = s->y_stride;
  a.x = s->x, a.dt = s->dt, a.B = s->B, a.C = s->C, a.A = s->A, a.D = s->D, a.bias = s->dt_bias;
  a.initial = s->initial, a.y = s->y, a.final = s->final;
  a.x_wide = wide(s->x, s->x_stride, s->dim), a.b_wide = wide(s->B, s->b_stride, s->state), a.c_wide = wide(s->C, s->c_stride, s->state);
  a.y_wide = wide(s->y, s->y_stride, s->dim);
  return a;
}

}  // namespace trunk

using namespace trunk;

extern "C" uint32_t uor_trunk_abi_version(void) { return UOR_TRUNK_ABI_VERSION; }
extern "C" const char *uor_trunk_last_error(void) { return error_text(); }
extern "C" uint64_t uor_trunk_sizeof_scan(void) { return sizeof(uor_trunk_scan_args); }
extern "C" uint64_t uor_trunk_sizeof_conv(void) { return sizeof(uor_trunk_conv_args); }
extern "C" uint64_t uor_trunk_sizeof_norms(void) { return sizeof(uor_trunk_norms_args); }

extern "C" uint64_t uor_trunk_scan_workspace_bytes(const uor_trunk_scan_args *s) {
  if (check_scan(s, false)) return 0;
  const uint32_t size = piece_rows(s->tokens, s->heads * tiles_of(s->dim));
  if (size >= s->tokens) return 0;
  const uint64_t n = pieces(s->tokens, s->seqs, size);
  return starts_bytes(n, s) + n * s->heads * sizeof(double);
}

extern "C" int uor_trunk_scan_async(const uor_trunk_scan_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_scan(s, false)) return e;
  if (s->tokens && !s->y) return fail(-1, "null y");
  const uint64_t want = uor_trunk_scan_workspace_bytes(s);
  if (want && (!workspace || bytes < want || (uintptr_t)workspace % 16))
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)want);
  Scan a = scan_of(s, piece_rows(s->tokens, s->heads * tiles_of(s->dim)));
  if (want) {
    a.starts = (float *)workspace;
    a.totals = (double *)((char *)workspace + starts_bytes(a.pieces, s));
  }
  if ((uint64_t)(a.pieces + kXcds) * a.heads * a.tiles > 0x7fffffffu) return fail(-1, "too many sequences and heads for one call");
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(a, s->seqs, (hipStream_t)stream) : launch<float>(a, s->seqs, (hipStream_t)stream);
}
