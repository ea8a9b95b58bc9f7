// scan.hip - the selective state space scan over packed sequences: outputs and final states.
//
// One wavefront takes 32 values of one head of one piece of a sequence, chunk after chunk, with their
// state in registers: as columns of values of x, so that pairs of its tiles are the operand of the
// product with C as they lie. The scores C_t . B_s are computed with s along the tile's rows, so that
// a lane's results are, once scaled, its operand of the next product over s. The blocks' four
// wavefronts are of one group and share B and C; x is each wavefront's own.
//
// Rows are bound by instructions and by time, not by bytes or products: 300 bf16 prompts of up to 509,
// 8 heads of 64 by a state of 64, take 90 us (98 with the launches around), of which their bytes would
// take 41, the vector instructions 54 and the products 20. Two pairs of tiles of x a wavefront compute
// scores and decays once for both, but leave half the wavefronts, two a SIMD instead of three: 130 us
// against 112, before the longest went first.
//
// A sequence of many rows and few heads would run on few wavefronts. Such sequences are cut into
// pieces: a first launch gives every piece its end state from zeros, a second joins them along the
// sequence, and the main launch runs all pieces at once. One of 65,536 rows, 16 heads of 64 by 128:
// 84 + 26 + 230 us.
#include "wave.h"

namespace trunk {

// The values of x that are infinite or no number, times their weights, onto y of their rows and of
// those after them: a row a lane. Rounding y before it changes nothing, as no such sum is finite.
template <class T, int NP, int PP>
__device__ __forceinline__ void add_odd(T *y, int64_t y_stride, uint32_t first, uint32_t end, uint32_t dim, uint32_t state, const T *sB,
                                     const T *sC, const T *sX, const Steps &s, float skip) {
  __threadfence_block();  // y has been written by other lanes
  const uint32_t t = threadIdx.x & 63;
  if (first + t >= end) return;
  T *row = y + (int64_t)(first + t) * y_stride;
  for (uint32_t from = 0; from <= t; from++) {
    float weight = 0.0f;
    bool known = false;
    for (uint32_t p = 0; p < dim; p++) {
      const float v = (float)sX[from * PP + p];
      if (finite(v)) continue;
      if (!known) {
        for (uint32_t n = 0; n < state; n++) weight += (float)sC[t * NP + n] * (float)sB[from * NP + n];
        weight *= from < t ? exp2_((s.hi[t] - s.hi[from]) + (s.lo[t] - s.lo[from])) * s.step[from] : s.step[from];
        if (from == t) weight += skip;
        known = true;
      }
      row[p] = (T)((float)row[p] + weight * v);
    }
  }
}

template <class T, int NT, int PW, int W>
__global__ __launch_bounds__(64 * W, W == 1 ? 1 : 2) void scan_rows(Scan a) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kNp = pitch<T>(kN), kPp = pitch<T>(kP), kThreads_ = 64 * W;
  __shared__ __align__(16) T sB[kChunk * kNp], sC[kChunk * kNp], sXs[W][kChunk * kPp];
  __shared__ Steps steps[W];

  clear_unowned(a.rows, (T *)a.y, a.y_stride, a.heads * a.dim);
  Unit unit = unit_of<W>(a, kP);
  Piece at;
  if (!next_piece(a, unit.piece, at)) return;
  const int wave = threadIdx.x >> 6, lane0 = threadIdx.x & 63;
  const uint32_t head = unit.head;
  const T *x = (const T *)a.x + head * a.dim + unit.p0, *dt = (const T *)a.dt + head;
  const T *B = (const T *)a.B + unit.group * a.state, *C = (const T *)a.C + unit.group * a.state;
  T *y = (T *)a.y + head * a.dim + unit.p0, *sX = sXs[wave];
  Steps &s = steps[wave];
  const uint32_t dim = a.dim - unit.p0 < (uint32_t)kP ? a.dim - unit.p0 : kP;
  const float A = a.A[head], skip = a.D ? a.D[head] : 0.0f, bias = a.bias ? a.bias[head] : 0.0f;
  const uint64_t whole = (uint64_t)a.dim * a.state, part = (uint64_t)unit.p0 * a.state;
  f32x4 h[NT][PW];
  get_state<NT, PW>(h,
                    at.number ? a.starts + ((next_place(a, at) - 1) * a.heads + head) * whole + part
                              : a.initial ? a.initial + ((uint64_t)at.seq * a.heads + head) * whole + part : nullptr,
                    dim, a.state, a.state_wide);

  // A chunk's rows are fetched into registers while the state goes past the chunk before.
  Load<T, kN, kThreads_> nextB, nextC;
  Load<T, kP, 64> nextX;
  float raw = 0.0f;
  const auto fetch = [&](uint32_t first) {
    const uint32_t end = at.end - first > kChunk ? first + kChunk : at.end;
    const int lane = anew(lane0), thread = wave * 64 + lane;
    nextB.get(thread, B, a.b_stride, first, end, a.state, a.b_wide);
    nextC.get(thread, C, a.c_stride, first, end, a.state, a.c_wide);
    nextX.get(lane, x, a.x_stride, first, end, dim, a.x_wide);
    raw = first + lane < end ? (float)dt[(int64_t)(first + lane) * a.dt_stride] : 0.0f;
  };
  fetch(at.first);  // past the last chunk nothing is read: rows that are always fetched need no register before

  for (uint32_t first = at.first; first < at.end; first += kChunk) {
    const uint32_t end = at.end - first > kChunk ? first + kChunk : at.end;
    const int lane = anew(lane0), thread = wave * 64 + lane, q = lane >> 4, i16 = lane & 15;
    __syncthreads();  // the chunk before has been read
    nextB.put(thread, sB, a.b_stride, a.state, a.b_wide);
    nextC.put(thread, sC, a.c_stride, a.state, a.c_wide);
    const bool odd = __any(nextX.put(lane, sX, a.x_stride, dim, a.x_wide));
    const Decay d = steps_of(lane, s, row_of(raw, first + lane < end, A, bias));
    __syncthreads();
    if (unit.idle) {
      fetch(end);
      continue;
    }

    // y, transposed: what comes from the state before the chunk.
    f32x4 acc[4][PW];
#pragma unroll
    for (int tile = 0; tile < 4; tile++)
#pragma unroll
      for (int i = 0; i < PW; i++) acc[tile][i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NT / 2; k++) {
      V8<T> c[4];
#pragma unroll
      for (int tile = 0; tile < 4; tile++) c[tile] = operand(sC + (tile * 16 + i16) * kNp, 32 * k + 8 * q);
#pragma unroll
      for (int i = 0; i < PW; i++) {
        const auto hs = Fine<T>::of(__builtin_shufflevector(h[2 * k][i], h[2 * k + 1][i], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int tile = 0; tile < 4; tile++) acc[tile][i] = mul(hs, c[tile], acc[tile][i]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    V8<T> xs[2][PW];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int i = 0; i < PW; i++) xs[k][i] = column<T, kPp>(lane, sX, 32 * k, i);
    // Some x of the chunk is infinite or no number: its products with the zeros above the diagonal
    // would reach rows before it. Such values are left out of the products, and added afterwards.
    if (odd) {
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < PW; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) xs[k][i][e] = finite((float)xs[k][i][e]) ? xs[k][i][e] : (T)0.0f;
    }

    // And what comes from the chunk's own rows, 16 at a time.
#pragma unroll
    for (int tile = 0; tile < 4; tile++) {
      const int t = tile * 16 + i16;
      __builtin_amdgcn_sched_barrier(0);  // tiles taken together would not fit the registers
      if (first + tile * 16 >= end) break;
      V8<T> c[NT / 2];
#pragma unroll
      for (int k = 0; k < NT / 2; k++) c[k] = operand(sC + t * kNp, 32 * k + 8 * q);
      const float u = s.u[t];
      const auto score = [&](int other) {
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < NT / 2; k++) v = Mma<T>::mul(operand(sB + (other * 16 + i16) * kNp, 32 * k + 8 * q), c[k], v);
        return v;
      };
      const auto before = [&](int other) {  // a tile before this one: its rows' weight at this one's start
        const float c = other + 1 == tile ? 1.0f : tile == 2 ? d.c20 : other == 0 ? d.c30 : d.c31;
        return score(other) * (*(const f32x4 *)(s.v + other * 16 + 4 * q) * c);
      };
#pragma unroll
      for (int i = 0; i < PW; i++) acc[tile][i] *= tile < 2 ? d.from[tile] * u : d.from[tile];
      const auto add = [&](int pair, f32x8 m) {
        const auto w = Fine<T>::of(m);
#pragma unroll
        for (int i = 0; i < PW; i++) acc[tile][i] = mul(xs[pair][i], w, acc[tile][i]);
      };
      if (tile >= 2) {
        add(0, __builtin_shufflevector(before(0), before(1), 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < PW; i++) acc[tile][i] *= u;
      }
      // The tile's own rows, and the tile before it in the same pair.
      f32x4 own = score(tile);
      const f32x4 step = *(const f32x4 *)(s.step + tile * 16 + 4 * q), hi = *(const f32x4 *)(s.hi + tile * 16 + 4 * q),
                  lo = *(const f32x4 *)(s.lo + tile * 16 + 4 * q);
      const float hi_t = s.hi[t], lo_t = s.lo[t];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int other = 4 * q + r;
        const float decay = exp2_((hi_t - hi[r]) + (lo_t - lo[r])) * step[r];
        own[r] = keep(own[r] * decay, other < i16) + keep(own[r] * step[r] + skip, other == i16);
      }
      if (tile & 1) add(tile >> 1, __builtin_shufflevector(before(tile - 1) * u, own, 0, 1, 2, 3, 4, 5, 6, 7));
      else add(tile >> 1, __builtin_shufflevector(own, f32x4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7));
      if (a.y_wide) {  // rows past the last and columns past dim are dropped
        const uint32_t pitch = (uint32_t)a.y_stride * sizeof(T);
        const auto to = __builtin_amdgcn_make_buffer_rsrc((void *)(y + (int64_t)first * a.y_stride), 0,
                                                          (int)((end - first - 1) * pitch + dim * (uint32_t)sizeof(T)), 0x00020000);
#pragma unroll
        for (int i = 0; i < PW; i += 2) {
          const uint32_t p = place(i, 4 * q);
          store_eight<T>(to, t * pitch + p * (uint32_t)sizeof(T), p, dim, __builtin_shufflevector(acc[tile][i], acc[tile][i + 1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
      } else if (first + t < end) {
        T *row = y + (int64_t)(first + t) * a.y_stride;
#pragma unroll
        for (int i = 0; i < PW; i++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (place(i, 4 * q + r) < (int)dim) row[place(i, 4 * q + r)] = (T)acc[tile][i][r];
      }
    }
    if (odd) {
      add_odd<T, kNp, kPp>(y, a.y_stride, first, end, dim, a.state, sB, sC, sX, s, skip);
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < PW; i++) xs[k][i] = column<T, kPp>(lane, sX, 32 * k, i);
    }
    fetch(end);  // now that y's registers are free
    advance<T, NT, PW>(lane, h, xs, sB, s.v, d.to, d.whole);
  }
  if (a.final && at.end == at.stop && !unit.idle)
    put_state<NT, PW>(h, a.final + ((uint64_t)at.seq * a.heads + head) * whole + part, dim, a.state, a.state_wide);
}

// The end states of pieces from zeros into the start states of those after them, along each sequence that
// has more than one.
__global__ __launch_bounds__(kThreads) void scan_join(Scan a) {
  const uint32_t head = blockIdx.x % a.heads;
  uint32_t seq, n;
  if (!joined(a, blockIdx.x / a.heads, seq, n)) return;
  const uint64_t base = a.rows.at(seq) / a.size, whole = (uint64_t)a.dim * a.state, step = a.heads * whole;
  for (uint64_t e = blockIdx.y * kThreads + threadIdx.x; e < whole; e += (uint64_t)gridDim.y * kThreads) {
    float h = a.initial ? a.initial[((uint64_t)seq * a.heads + head) * whole + e] : 0.0f;
    float *at = a.starts + (base * a.heads + head) * whole + e;
    const double *totals = a.totals + base * a.heads + head;
    for (uint32_t j = 0; j < n; j += kAhead) {
      float own[kAhead], decay[kAhead];  // of the next pieces: what is read does not wait for the sums
#pragma unroll
      for (uint32_t k = 0; k < kAhead; k++) {
        const uint32_t place = j + k + 1 < n ? j + k : 0;
        own[k] = at[place * step];
        decay[k] = (float)totals[(uint64_t)place * a.heads];
      }
#pragma unroll
      for (uint32_t k = 0; k < kAhead; k++) {
        if (j + k >= n) break;
        if (j + k) at[(j + k - 1) * step] = h;
        h = exp2_(decay[k]) * h + own[k];
      }
    }
  }
}

// The pieces by their chunks, the longest first, so that none begins when the others end: 300 prompts of
// up to 509 take 129 us in their own order and 95 in this, 5 of them for the order. Which of two alike comes
// first may differ from call to call; no result depends on it.
__global__ __launch_bounds__(1024) void scan_order(Scan a) {
  constexpr uint32_t kBuckets = 64;
  __shared__ uint32_t next[kBuckets + 1];
  for (uint32_t b = threadIdx.x; b <= kBuckets; b += 1024) next[b] = 0;
  __syncthreads();
  const auto bucket = [](uint32_t rows) {
    const uint32_t chunks = (rows + kChunk - 1) / kChunk;
    return kBuckets - (chunks < kBuckets ? chunks : kBuckets);
  };
  const auto each = [&](auto put) {
    for (uint32_t seq = threadIdx.x; seq < a.rows.seqs; seq += 1024) {
      uint32_t start, stop;
      a.rows.of(seq, start, stop);
      const uint32_t n = stop > start ? (stop - start - 1) / a.size + 1 : 1;
      if (n > 1) put(seq, 0, n - 1, bucket(a.size));
      put(seq, n - 1, 1, bucket(stop - start - (n - 1) * a.size));
    }
  };
  each([&](uint32_t, uint32_t, uint32_t count, uint32_t b) { atomicAdd(&next[b], count); });
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t sum = 0;
    for (uint32_t b = 0; b <= kBuckets; b++) {
      const uint32_t here = next[b];
      next[b] = sum;
      sum += here;
    }
    a.order[0] = sum < a.pieces ? sum : a.pieces;  // more only where the offsets do not ascend
  }
  __syncthreads();
  each([&](uint32_t seq, uint32_t number, uint32_t count, uint32_t b) {
    const uint32_t at = atomicAdd(&next[b], count);
    for (uint32_t i = 0; i < count && at + i < a.pieces; i++) {
      a.order[2 + 2 * (at + i)] = seq;
      a.order[3 + 2 * (at + i)] = number + i;
    }
  });
}

// How many rows a piece has: sequences are cut where they alone would leave the card idle. The grid
// then has about 4,096 wavefronts, two for each place; pieces under `least` rows cost more to join
// than they gain: one head over 9 bf16 prompts of 2,580 rows takes 69 us in pieces of 512 and 31 in pieces
// of 128, f32 gradients of 37 of up to 301 102 us in pieces of 128 and 70 in pieces of 64. Where there are
// sequences for every place only those are cut that would still run when the others have long ended.
uint32_t piece_rows(uint32_t tokens, uint32_t seqs, uint32_t units, uint32_t least) {
  const uint64_t even = ((uint64_t)tokens * units + 4095) / 4096, want = (uint64_t)seqs * units < 2048 ? even : 4 * even;
  const uint64_t size = (want < least ? least : want) + kChunk - 1;
  const uint64_t rows = size / kChunk * kChunk;
  return rows < tokens ? (uint32_t)rows : (tokens + kChunk) / kChunk * kChunk;
}

namespace {

template <class T, int NT, int PW, int W>
int launch(const Scan &a, hipStream_t stream) {
  const uint32_t units = a.heads / a.groups * a.tiles, blocks = a.groups * ((units + W - 1) / W);
  if (a.starts) {
    hipLaunchKernelGGL((scan_ends<T, NT, PW, W, false>), dim3(grid_of(a.later, blocks)), dim3(64 * W), 0, stream, a);
    hipLaunchKernelGGL(scan_join, join_of(a), dim3(kThreads), 0, stream, a);
  }
  if (a.order) hipLaunchKernelGGL(scan_order, dim3(1), dim3(1024), 0, stream, a);
  hipLaunchKernelGGL((scan_rows<T, NT, PW, W>), dim3(grid_of(a.pieces, blocks)), dim3(64 * W), 0, stream, a);
  return launched();
}
template <class T, int NT, int PW>
int launch(const Scan &a, hipStream_t stream) {
  const uint32_t units = a.heads / a.groups * a.tiles;
  return units == 1 ? launch<T, NT, PW, 1>(a, stream) : units == 2 ? launch<T, NT, PW, 2>(a, stream) : launch<T, NT, PW, 4>(a, stream);
}
template <class T>
int launch(const Scan &a, hipStream_t stream) {
  return a.state <= 32 ? launch<T, 2, 2>(a, stream) : a.state <= 64 ? launch<T, 4, 2>(a, stream) : launch<T, 8, 2>(a, stream);
}

// 512 rows are never cut: two more launches cost what a chain of eight chunks does.
uint32_t rows_of(const uor_trunk_scan_args *s) {
  return s->tokens <= 512 ? 512 + kChunk : piece_rows(s->tokens, s->seqs, s->heads * ((s->dim + 31) / 32), 128);
}
// Where a call's scratch memory begins, and how much there is.
struct Plan {
  uint32_t size;
  bool cut, ordered;
  uint64_t totals, order, bytes;
};
Plan plan_of(const uor_trunk_scan_args *s) {
  Plan p{};
  p.size = rows_of(s);
  p.cut = p.size < s->tokens;
  const uint64_t n = pieces(s->tokens, s->seqs, p.size), waves = n * s->heads * ((s->dim + 31) / 32);
  // One launch more, where more wavefronts are wanted than the card holds and each has long to go; the
  // launch looks at 1,024 sequences at a time. Without and with it, bf16, 8 heads of 64 by a state of 64:
  // 200 prompts of up to 340 (3,200 wavefronts, 35,342 rows) 78 and 59 us, 300 of up to 250 72 and 61, 600
  // of up to 110 (33,321 rows) 69 and 64, 8,000 of up to 40 491 and 486. Below the borders it gains where
  // lengths are long (190 of up to 340: 75 and 56) and not where they are short (600 of up to 60: 50 and 52),
  // and with many sequences it costs more than it gives (20,000 of up to 10: 1,033 and 1,077).
  p.ordered = s->seqs > 1 && s->seqs <= 8192 && waves > 3072 && s->tokens >= 32768;
  if (p.cut) {
    const uint64_t later = s->tokens / p.size + 1;
    p.totals = (later * s->heads * s->dim * s->state * 4 + 15) / 16 * 16;
    p.bytes = p.totals + later * s->heads * sizeof(double);
  }
  if (p.ordered) {
    p.order = (p.bytes + 15) / 16 * 16;
    p.bytes = p.order + (n + 1) * 8;
  }
  return p;
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
  const auto wide = [&](const void *p, int64_t stride, uint32_t part) { return wide_rows(p, stride, part, bytes); };
  Scan a{};
  a.rows = Rows{s->offsets, s->tokens, s->seqs};
  a.heads = s->heads, a.groups = s->groups, a.dim = s->dim, a.state = s->state;
  a.size = size, a.pieces = pieces(s->tokens, s->seqs, size), a.later = s->tokens / size + 1, a.tiles = (s->dim + 31) / 32;
  // One row has no stride; chunks go by one all the same.
  const int64_t inner = (int64_t)s->heads * s->dim, shared = (int64_t)s->groups * s->state;
  const bool one = s->tokens <= 1;
  a.x_stride = one ? inner : s->x_stride, a.dt_stride = one ? s->heads : s->dt_stride, a.y_stride = one ? inner : s->y_stride;
  a.b_stride = one ? shared : s->b_stride, a.c_stride = one ? shared : s->c_stride;
  a.x = s->x, a.dt = s->dt, a.B = s->B, a.C = s->C, a.A = s->A, a.D = s->D, a.bias = s->dt_bias;
  a.initial = s->initial, a.y = s->y, a.final = s->final;
  a.x_wide = wide(s->x, a.x_stride, s->dim), a.b_wide = wide(s->B, a.b_stride, s->state), a.c_wide = wide(s->C, a.c_stride, s->state);
  a.y_wide = wide(s->y, a.y_stride, s->dim);
  a.state_wide = s->state % 4 == 0 && aligned16(s->initial, 0, 4) && aligned16(s->final, 0, 4);
  return a;
}

}  // namespace trunk

using namespace trunk;

extern "C" uint32_t uor_trunk_abi_version(void) { return UOR_TRUNK_ABI_VERSION; }
extern "C" const char *uor_trunk_last_error(void) { return error_text(); }
extern "C" uint64_t uor_trunk_sizeof_scan(void) { return sizeof(uor_trunk_scan_args); }
extern "C" uint64_t uor_trunk_sizeof_conv(void) { return sizeof(uor_trunk_conv_args); }
extern "C" uint64_t uor_trunk_sizeof_norms(void) { return sizeof(uor_trunk_norms_args); }

extern "C" uint64_t uor_trunk_scan_workspace_bytes(const uor_trunk_scan_args *s) { return check_scan(s, false) ? 0 : plan_of(s).bytes; }

extern "C" int uor_trunk_scan_async(const uor_trunk_scan_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_scan(s, false)) return e;
  if (s->tokens && !s->y) return fail(-1, "null y");
  const Plan p = plan_of(s);
  if (p.bytes && (!workspace || bytes < p.bytes || (uintptr_t)workspace % 16))
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)p.bytes);
  Scan a = scan_of(s, p.size);
  if (p.cut) {
    a.starts = (float *)workspace;
    a.totals = (double *)((char *)workspace + p.totals);
  }
  if (p.ordered) a.order = (uint32_t *)((char *)workspace + p.order);
  if ((uint64_t)(a.pieces + kXcds) * a.heads * a.tiles > 0x7fffffffu) return fail(-1, "too many sequences and heads for one call");
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(a, (hipStream_t)stream) : launch<float>(a, (hipStream_t)stream);
}
