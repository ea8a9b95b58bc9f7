// scan_grad.hip - the scan's gradients over packed sequences.
//
// With g the gradient at the state after a chunk, from what comes later, and h the state before it,
// W_ts = dy_t . x_s, S_ts = C_t . B_s and e_ts = e^(l_t - l_s) for s <= t, all inside the chunk:
//
//   dx_s = D_s [ e^(l_end - l_s) g B_s + sum_(t >= s) S_ts e_ts dy_t ] + skip dy_s,
//   dB_s = D_s [ e^(l_end - l_s) g^T x_s + sum_(t >= s) W_ts e_ts C_t ],
//   dC_t = e^(l_t) h^T dy_t + sum_(s <= t) W_ts e_ts D_s B_s,
//   g'   = e^(l_end) g + sum_t e^(l_t) dy_t (x) C_t   for the chunk before.
//
// With E_ts = W_ts S_ts e_ts D_s, q_t = e^(l_t) C_t . h^T dy_t and r_s = D_s e^(l_end - l_s) x_s . g B_s, the
// gradient at the logarithm of row u's decay is
//
//   da_u = e^(l_end) <g, h> + sum_(t >= u) q_t + sum_(s < u) r_s + sum_(t >= u, s < u) E_ts,
//
// whose last sum is taken tile by tile: rows' sums over the tiles before u's, columns' over those
// after it, and within u's own tile its rows' running sums. (The sum over t >= u of E's row t less its
// column t is the same, but what cancels there is many times what is left.) At the step itself the
// gradient is (r_u + column u of E) / D_u + A da_u, where what D_u divides is summed without it.
//
// A block takes one group of one piece of a sequence, a wavefront one of its heads (or 32 of a head's
// values), with g in registers. It goes along the piece once for h, and writes the states before its
// chunks down but for the last, which it still holds; then back, chunk after chunk. Both states are
// wanted in two layouts: h is summed as columns of the state's axis, and g, held as columns of x's
// values, is turned by products with parts of the unit matrix, which are exact. dB and dC are summed
// over the block's wavefronts through LDS, in their order. Long sequences are cut into pieces as in
// the scan; one launch more gives every piece's gradient at its start.
//
// Bound by instructions: 2,048 bf16 sequences of 128, 8 heads of 64 by a state of 64, take 1,041 us,
// of which the vector instructions alone would take 539, the products 166 and the bytes 184. Two blocks
// of four wavefronts share a compute unit, two wavefronts a SIMD with 256 registers each; one a SIMD
// with 512 took 1,750 us where this took 980, one block of eight wavefronts 1,027.
#include "wave.h"

namespace trunk {

struct Grad {
  Scan s;               // s.tiles: parts of dim, rounded up to a power of two
  const void *dy;
  const float *dfinal;
  uint32_t subs, parts; // a group's wavefronts are taken in so many turns, shared by so many blocks
  float *h;             // [tokens / 64 + 1][heads * tiles][NT * 2][64][4]: states before chunks
  float *g_starts;      // like s.starts: the gradients at the starts of pieces after their sequence's first
  double *sums;         // [pieces][heads][3]: dA, dD, ddt_bias
  float *dBparts, *dCparts;  // [parts][tokens][groups][state], with more than one turn
  void *dx, *ddt, *dB, *dC;
  float *dA, *dD, *dbias, *dinitial;
  bool dy_wide, dx_wide, shared_wide, mid_wide;
};

// The 32 x 16 part `which` of the unit matrix as an operand.
template <class T>
__device__ __forceinline__ V8<T> ones(int lane, int which) {
  V8<T> v;
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = (T)(e >> 2 == which && 4 * (lane >> 4) + (e & 3) == (lane & 15) ? 1.0f : 0.0f);
  return v;
}
// The turned parts: two operands of a row's 32 places each, as one of the places' rows `which`.
__device__ __forceinline__ bf16x8 turn(bf16x8 a, bf16x8 b, bf16x8 unit) {
  const f32x4 zero = {0, 0, 0, 0};
  const f32x4 x = Mma<bf16>::mul(a, unit, zero), y = Mma<bf16>::mul(b, unit, zero);
  return __builtin_convertvector(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7), bf16x8);
}
__device__ __forceinline__ Fine<bf16> turn(const Fine<bf16> &a, const Fine<bf16> &b, bf16x8 unit) {
  return {turn(a.hi, b.hi, unit), turn(a.mid, b.mid, unit), turn(a.lo, b.lo, unit)};
}
__device__ __forceinline__ Fine<float> turn(const Fine<float> &a, const Fine<float> &b, f32x8 unit) {
  const f32x4 zero = {0, 0, 0, 0};
  return {__builtin_shufflevector(Mma<float>::mul(a.v, unit, zero), Mma<float>::mul(b.v, unit, zero), 0, 1, 2, 3, 4, 5, 6, 7)};
}
__device__ __forceinline__ float dot(f32x8 a, f32x8 b) {
  const f32x4 v = __builtin_shufflevector(a, a, 0, 1, 2, 3) * __builtin_shufflevector(b, b, 0, 1, 2, 3) +
                  __builtin_shufflevector(a, a, 4, 5, 6, 7) * __builtin_shufflevector(b, b, 4, 5, 6, 7);
  return (v[0] + v[1]) + (v[2] + v[3]);
}
// The sum of a row's 16 lanes, to all of them: from 8, 4, 2 and 1 lanes on, around the row.
__device__ __forceinline__ float row_sum(float v) {
  v += moved<0x128>(v);
  v += moved<0x124>(v);
  v += moved<0x122>(v);
  return v + moved<0x121>(v);
}
// The sum of a column's four lanes.
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// h as columns of the state's axis: h[n][i] holds rows place(i, 4 q + r) of dim, column place(n, lane % 16).
template <int NT>
__device__ __forceinline__ void get_turned(int lane, f32x4 (&h)[NT][2], const float *at, uint32_t dim, uint32_t state) {
  const int q = lane >> 4, i16 = lane & 15;
#pragma unroll
  for (int n = 0; n < NT; n++) h[n][0] = h[n][1] = f32x4{0, 0, 0, 0};
  if (!at) return;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t p = place(i, 4 * q + r), c = place(n, i16);
        h[n][i][r] = p < dim && c < state ? at[(uint64_t)p * state + c] : 0.0f;
      }
}
// advance, for a state that lies so.
template <class T, int NT>
__device__ __forceinline__ void advance_turned(int lane, f32x4 (&h)[NT][2], const T *sX, const T *sB, const float *rows, const float (&to)[4],
                                               float whole) {
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 2; i++) h[n][i] *= whole;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const f32x8 weight = weights(lane, rows, 32 * k, to[2 * k], to[2 * k + 1]);
    Fine<T> w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) w[i] = Fine<T>::of(widen<T>(column<T, pitch<T>(32)>(lane, sX, 32 * k, i)) * weight);
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const V8<T> b = column<T, pitch<T>(16 * NT)>(lane, sB, 32 * k, n);
#pragma unroll
      for (int i = 0; i < 2; i++) h[n][i] = mul(w[i], b, h[n][i]);
    }
  }
}

// What a loop computes from these values is computed again each time (see anew).
template <int NT>
__device__ __forceinline__ void hold(f32x4 (&h)[NT][2]) {
#pragma unroll
  for (int n = 0; n < NT; n++) asm volatile("" : "+v"(h[n][0]), "+v"(h[n][1]));
}

// Values that are infinite or no number (odd) meet zeros in the products: of rows that come before or after,
// of the parts of the unit matrix. What is not finite by the definition then is none here, but more may
// be: in the chunk, rows on the other side. A piece where that was (some ddt of it is not finite) is taken once more by
// a second form, whose products leave such values out, and which then writes NaN where they reach:
//   dx_s: an odd dy_t of the same value or any C_t of t >= s, B_s, a step's NaN after s, D_s;
//   dB_s: an odd dy_t, the same value of C_t of t >= s, x_s, a step's NaN after s, D_s, the same value of g;
//   dC_t: an odd x_s or D_s, the same value of B_s of s <= t, dy_t;
//   da_u: an odd dy_t or C_t of t >= u, x_s, B_s or D_s of s < u, any of g, any step's NaN.
// Where all is finite that is one launch more: 37 f32 sequences of up to 301 take 71 us where they took 68,
// 2,048 bf16 sequences of 128 1,090 where they took 1,075.
template <bool ODD, class V>
__device__ __forceinline__ V clean(V v) {
  if constexpr (ODD) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (!finite((float)v[e])) v[e] = 0.0f;
  }
  return v;
}
constexpr float kNone = __builtin_nanf("");
// The odd rows of a wavefront's chunk, a bit a row. `decays`: those whose decay is odd, `steps`: D_t.
struct Odd {
  uint64_t dy, x, B, C, steps, decays;
  bool g;
};
__device__ __forceinline__ bool from_row(uint64_t rows, int s) { return rows >> s; }
__device__ __forceinline__ bool after_row(uint64_t rows, int s) { return rows >> s >> 1; }
__device__ __forceinline__ bool before_row(uint64_t rows, int s) { return rows & ((1ull << s) - 1); }
__device__ __forceinline__ bool up_to_row(uint64_t rows, int s) { return rows << (63 - s); }
__device__ __forceinline__ bool at_row(uint64_t rows, int s) { return rows >> s & 1; }

// Wavefronts that a SIMD is to hold: with states of more than 64 a wavefront needs all its registers.
template <int NT, int W>
constexpr int kHeld = NT > 4 || W == 1 ? 1 : 2;

template <class T, int NT, int W, bool ODD>
__global__ __launch_bounds__(64 * W, (kHeld<NT, W>)) void grad_rows(Grad k) {
  constexpr int kN = 16 * NT, kP = 32, kNp = pitch<T>(kN), kPp = pitch<T>(kP), G = 2;
  __shared__ __align__(16) T sB[kChunk * kNp], sC[kChunk * kNp], sYs[W][kChunk * kPp];
  __shared__ __align__(16) float sRed[W][G * 2 * 256];
  __shared__ GradSteps steps[W];
  // q and r / D without their decays; of E its tiles' own part of da, the rows' sums over the tiles
  // before, the columns' over those after / D, and the columns' whole sums / D.
  __shared__ float sSum[W][6][kChunk];
  __shared__ float sDa[W][kChunk], sDirect[W][kChunk], sDiag[W];
  const Scan &a = k.s;
  const uint32_t share = a.heads / a.groups, units = share * a.tiles;
  if constexpr (!ODD) {
    clear_unowned(a.rows, (T *)k.dx, (int64_t)a.heads * a.dim, a.heads * a.dim);
    clear_unowned(a.rows, (T *)k.ddt, a.heads, a.heads);
    clear_unowned(a.rows, (T *)k.dB, (int64_t)a.groups * a.state, a.groups * a.state);
    clear_unowned(a.rows, (T *)k.dC, (int64_t)a.groups * a.state, a.groups * a.state);
  }
  uint32_t number, block;
  place_of(blockIdx.x, a.groups * k.parts, number, block);
  Piece at;
  if (!next_piece(a, number, at)) return;
  const uint32_t group = block / k.parts, part = block % k.parts;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane0 = threadIdx.x & 63;
  const T *B = (const T *)a.B + group * a.state, *C = (const T *)a.C + group * a.state;
  const uint64_t whole = (uint64_t)a.dim * a.state;
  const uint32_t chunks = (at.end - at.first + kChunk - 1) / kChunk;
  T *sY = sYs[wave];
  GradSteps &s = steps[wave];
  const uint32_t sub0 = k.subs * part / k.parts, sub1 = k.subs * (part + 1) / k.parts;
  if constexpr (ODD) {  // of the block's own heads, whose sums the block itself writes anew
    bool any = false;
    for (uint32_t unit = sub0 * W + lane0 * a.tiles; unit < sub1 * W && unit < units; unit += 64 * a.tiles)
      any |= !(fabs(k.sums[((uint64_t)number * a.heads + group * share + unit / a.tiles) * 3 + 2]) < __builtin_inf());
    if (!__any(any)) return;  // each wavefront looks at all of them
  }

#pragma unroll 1
  for (uint32_t sub = sub0; sub < sub1; sub++) {
    uint32_t unit = sub * W + wave;
    bool idle = unit >= units;
    if (idle) unit = 0;
    const uint32_t head = group * share + unit / a.tiles, tile = unit % a.tiles, p0 = tile * kP;
    idle = idle || p0 >= a.dim;
    const uint32_t dim = idle ? 0 : a.dim - p0 < (uint32_t)kP ? a.dim - p0 : kP;
    const T *x = (const T *)a.x + head * a.dim + p0, *dy = (const T *)k.dy + head * a.dim + p0, *dt = (const T *)a.dt + head;
    const float A = a.A[head], skip = a.D ? a.D[head] : 0.0f, bias = a.bias ? a.bias[head] : 0.0f;
    const uint64_t cell = (uint64_t)p0 * a.state;
    const float *start = at.number ? a.starts + ((next_place(a, at) - 1) * a.heads + head) * whole + cell
                                   : a.initial ? a.initial + ((uint64_t)at.seq * a.heads + head) * whole + cell : nullptr;
    const float *finish = at.end != at.stop ? k.g_starts + (next_place(a, at) * a.heads + head) * whole + cell
                                            : k.dfinal ? k.dfinal + ((uint64_t)at.seq * a.heads + head) * whole + cell : nullptr;
    // Where the state before the piece's j-th chunk is kept.
    const auto kept = [&](uint32_t j) {
      return k.h + (((uint64_t)(at.first / kChunk + j) * a.heads + head) * a.tiles + tile) * (NT * 2 * 256);
    };

    // Along the piece, but for its last chunk.
    f32x4 h[NT][2];
    get_turned<NT>(lane0, h, idle ? nullptr : start, dim, a.state);
    {
      Load<T, kN, 64 * W> nextB;
      Load<T, kP, 64> nextX;
      float raw = 0.0f;
      const auto fetch = [&](uint32_t j) {
        const uint32_t first = at.first + j * kChunk, rows = j + 1 < chunks ? kChunk : 0;
        const int lane = anew(lane0), thread = wave * 64 + lane;
        nextB.get(thread, B, a.b_stride, first, first + rows, a.state, a.b_wide);
        nextX.get(lane, x, a.x_stride, first, first + rows, dim, a.x_wide && dim);
        raw = rows ? (float)dt[(int64_t)(first + lane) * a.dt_stride] : 0.0f;
      };
      fetch(0);
#pragma unroll 1
      for (uint32_t j = 0; j + 1 < chunks; j++) {
        const int lane = anew(lane0), thread = wave * 64 + lane;
        __syncthreads();
        nextB.put(thread, sB, a.b_stride, a.state, a.b_wide);
        nextX.put(lane, sY, a.x_stride, dim, a.x_wide && dim);
        const Decay d = steps_of(lane, s, row_of(raw, true, A, bias));
        __syncthreads();
        fetch(j + 1);
        if (idle) continue;
        advance_turned<T, NT>(lane, h, sY, sB, s.v, d.to, d.whole);
        if (j + 2 < chunks) {
          float *to = kept(j + 1) + lane * 4;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) *(f32x4 *)(to + (n * 2 + i) * 256) = h[n][i];
        }
      }
    }

    // And back.
    f32x4 g[NT][2];
    get_state<NT, 2>(g, idle ? nullptr : finish, dim, a.state, a.state_wide);
    double sumA = 0.0, sumD = 0.0, sumBias = 0.0;
    const bool x_wide = a.x_wide && dim;
    Load<T, kN, 64 * W> nextB, nextC;
    Load<T, kP, 64> nextY;
    float raw = 0.0f;
    const auto fetch = [&](uint32_t j) {  // none where j is past the first chunk
      const bool more = j < chunks;
      const uint32_t first = more ? at.first + j * kChunk : at.first;
      const uint32_t end = !more ? first : at.end - first > kChunk ? first + kChunk : at.end;
      const int lane = anew(lane0), thread = wave * 64 + lane;
      nextB.get(thread, B, a.b_stride, first, end, a.state, a.b_wide);
      nextC.get(thread, C, a.c_stride, first, end, a.state, a.c_wide);
      nextY.get(lane, dy, a.y_stride, first, end, dim, k.dy_wide && dim);
      raw = first + lane < end ? (float)dt[(int64_t)(first + lane) * a.dt_stride] : 0.0f;
    };
    fetch(chunks - 1);
#pragma unroll 1
    for (uint32_t j = chunks; j-- > 0;) {
      const uint32_t first = at.first + j * kChunk, end = at.end - first > kChunk ? first + kChunk : at.end;
      const bool has_h = start || j, has_g = finish || j + 1 < chunks, more = end - first > 32;
      __syncthreads();
      const float raw_now = raw;
      Decay d;
      Odd odd = {};
      {
        const int lane = anew(lane0), thread = wave * 64 + lane;
        nextB.put(thread, sB, a.b_stride, a.state, a.b_wide);
        nextC.put(thread, sC, a.c_stride, a.state, a.c_wide);
        nextY.put(lane, sY, a.y_stride, dim, k.dy_wide && dim);
        Row row = row_of(raw, first + lane < end, A, bias);
        if constexpr (ODD) {
          odd.steps = __ballot(!finite(row.step));
          odd.decays = __ballot(!(fabs(row.log) < __builtin_inf()));
          row.step = finite(row.step) ? row.step : 0.0f;
          row.log = fabs(row.log) < __builtin_inf() ? row.log : 0.0;
        }
        d = steps_of(lane, s, row);
        if (!idle && j + 1 < chunks) {
          if (j) {
            const float *from = kept(j) + lane * 4;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int i = 0; i < 2; i++) h[n][i] = *(const f32x4 *)(from + (n * 2 + i) * 256);
          } else {
            get_turned<NT>(lane, h, start, dim, a.state);
          }
        }
      }
      __syncthreads();
      if constexpr (ODD) {
        const int lane = anew(lane0);
        bool dy_odd = false, x_odd = false, B_odd = false, C_odd = false, g_odd = false;
        for (uint32_t p = 0; p < dim; p++) {
          dy_odd |= !finite((float)sY[lane * kPp + p]);
          x_odd |= first + lane < end && !finite((float)x[(int64_t)(first + lane) * a.x_stride + p]);
        }
        for (uint32_t n = 0; n < a.state; n++) {
          B_odd |= !finite((float)sB[lane * kNp + n]);
          C_odd |= !finite((float)sC[lane * kNp + n]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int r = 0; r < 4; r++) g_odd |= !finite(g[n][0][r]) || !finite(g[n][1][r]);
        odd.dy = __ballot(dy_odd), odd.x = __ballot(x_odd), odd.B = __ballot(B_odd), odd.C = __ballot(C_odd);
        odd.g = __any(has_g && g_odd);
      }

      // Rows s by pairs of tiles, and for each the rows t of the pair after and of its own: (1, 1),
      // (0, 1), (0, 0). accB and dx are the rows s', accC the rows t's. One copy of the code serves all
      // three, as with one each the loop would not stay in the instruction cache.
      f32x4 accB[2][NT], accC[2][NT], dx[2][2];
      V8<T> X[2];  // x's rows s, as operands over dim
      // A lane's parts of E's columns below and in their own tile, and of its parts on both sides of
      // the second and of the third tile.
      float inner = 0.0f, diag = 0.0f, col[2], own[2], around[2] = {0, 0};
#pragma unroll 1
      for (int step_ = more ? 0 : 2; step_ < 3; step_++) {
        const int sp = step_ == 0, tp = step_ < 2;
        const int lane = anew(lane0), q = lane >> 4, i16 = lane & 15, s0 = 32 * sp + i16, t0 = 32 * tp + i16;
        if (step_ != 2 || !more) {
          // What comes through the state after the chunk: dx, and with g turned dB.
          col[0] = col[1] = own[0] = own[1] = 0.0f;
#pragma unroll
          for (int w = 0; w < 2; w++) {
            dx[w][0] = dx[w][1] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NT; n++) accB[w][n] = f32x4{0, 0, 0, 0};
          }
          if (x_wide) {
            const uint32_t pitch = (uint32_t)a.x_stride * sizeof(T), bytes = (end - first - 1) * pitch + dim * (uint32_t)sizeof(T);
            const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)(x + (int64_t)first * a.x_stride), 0, (int)bytes, 0x00020000);
#pragma unroll
            for (int w = 0; w < 2; w++) X[w] = clean<ODD>(load_eight<T>(from, (s0 + 16 * w) * pitch + 8 * q * (uint32_t)sizeof(T), 8 * q, dim));
          } else {
            T *rows = (T *)sRed[wave];
#pragma unroll 1
            for (uint32_t e = lane * 8; e < 32 * kP; e += 512) {
              const uint32_t row = first + 32 * sp + e / kP;
              *(V8<T> *)(rows + e) = load_some<T, 8>(x + (int64_t)row * a.x_stride, row < end, e % kP, dim);
            }
#pragma unroll
            for (int w = 0; w < 2; w++) X[w] = clean<ODD>(operand(rows + (w * 16 + i16) * kP, 8 * q));
          }
          if (!idle && has_g) {
            hold(g);
#pragma unroll
            for (int kk = 0; kk < NT / 2; kk++) {
              Fine<T> gp[2];
#pragma unroll
              for (int i = 0; i < 2; i++) gp[i] = Fine<T>::of(__builtin_shufflevector(g[2 * kk][i], g[2 * kk + 1][i], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
              for (int w = 0; w < 2; w++) {
                const V8<T> b = clean<ODD>(operand(sB + (s0 + 16 * w) * kNp, 32 * kk + 8 * q));
#pragma unroll
                for (int i = 0; i < 2; i++) dx[w][i] = mul(gp[i], b, dx[w][i]);
              }
              if constexpr (ODD) {
#pragma unroll
                for (int i = 0; i < 2; i++)
                  gp[i] = Fine<T>::of(clean<true>(__builtin_shufflevector(g[2 * kk][i], g[2 * kk + 1][i], 0, 1, 2, 3, 4, 5, 6, 7)));
              }
#pragma unroll
              for (int half = 0; half < 2; half++) {
                const int n = 2 * kk + half;
                const V8<T> unit_part = ones<T>(lane, half);
                const f32x4 zero = {0, 0, 0, 0};  // the parts' sum is the value itself
                const f32x8 turned = __builtin_shufflevector(mul(gp[0], unit_part, zero), mul(gp[1], unit_part, zero), 0, 1, 2, 3, 4, 5, 6, 7);
                if (has_h && (step_ == 0 || !more)) inner += dot(turned, __builtin_shufflevector(h[n][0], h[n][1], 0, 1, 2, 3, 4, 5, 6, 7));
                const auto gt = Fine<T>::of(turned);
#pragma unroll
                for (int w = 0; w < 2; w++) accB[w][n] = mul(gt, X[w], accB[w][n]);
                if constexpr (ODD) {
#pragma unroll
                  for (int r = 0; r < 4; r++) {
                    const float none = row_sum(finite(g[n][0][r]) && finite(g[n][1][r]) ? 0.0f : kNone);
                    accB[0][n][r] += none, accB[1][n][r] += none;
                  }
                }
              }
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int w = 0; w < 2; w++) {
              const float into = column_sum(dot(widen<T>(X[w]), __builtin_shufflevector(dx[w][0], dx[w][1], 0, 1, 2, 3, 4, 5, 6, 7)));
              if (q == 0) sSum[wave][1][s0 + 16 * w] = into;
              const float tail = s.w[s0 + 16 * w] * s.to[2 * sp + w], weight = s.v[s0 + 16 * w] * s.to[2 * sp + w];
#pragma unroll
              for (int i = 0; i < 2; i++) dx[w][i] *= tail;
#pragma unroll
              for (int n = 0; n < NT; n++) accB[w][n] *= weight;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (step_ != 1) {
          // What comes through the state before the chunk: dC.
#pragma unroll
          for (int v = 0; v < 2; v++)
#pragma unroll
            for (int n = 0; n < NT; n++) accC[v][n] = f32x4{0, 0, 0, 0};
          if (!idle && has_h) {
            hold(h);
            V8<T> y[2];
#pragma unroll
            for (int v = 0; v < 2; v++) y[v] = clean<ODD>(operand(sY + (t0 + 16 * v) * kPp, 8 * q));
#pragma unroll
            for (int n = 0; n < NT; n++) {
              const auto hp = Fine<T>::of(__builtin_shufflevector(h[n][0], h[n][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
              for (int v = 0; v < 2; v++) accC[v][n] = mul(hp, y[v], accC[v][n]);
            }
#pragma unroll
            for (int v = 0; v < 2; v++) {
              const int t = t0 + 16 * v;
              float through = 0.0f;
#pragma unroll
              for (int kk = 0; kk < NT / 2; kk++)
                through += dot(widen<T>(clean<ODD>(operand(sC + t * kNp, 32 * kk + 8 * q))),
                               __builtin_shufflevector(accC[v][2 * kk], accC[v][2 * kk + 1], 0, 1, 2, 3, 4, 5, 6, 7));
              through = column_sum(through);
              if (q == 0) sSum[wave][0][t] = through;
              const float weight = s.u[t] * s.from[2 * tp + v];
#pragma unroll
              for (int n = 0; n < NT; n++) accC[v][n] *= weight;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!idle) {
          // What comes from the chunk's own rows.
          Fine<T> Z[2];
          float rows[2][4] = {};  // a lane's part of E's rows, over the tiles before theirs
#pragma unroll
          for (int w = 0; w < 2; w++) {
            const int mine = s0 + 16 * w;
            const float step = s.step[mine], to_end = s.w[mine];
            V8<T> b[NT / 2];
#pragma unroll
            for (int kk = 0; kk < NT / 2; kk++) b[kk] = clean<ODD>(operand(sB + mine * kNp, 32 * kk + 8 * q));
            f32x4 M[2], z[2];
#pragma unroll
            for (int v = 0; v < 2; v++) {
              M[v] = z[v] = f32x4{0, 0, 0, 0};
              if (v < w && sp == tp) continue;
              f32x4 S = {0, 0, 0, 0};
#pragma unroll
              for (int kk = 0; kk < NT / 2; kk++) S = Mma<T>::mul(clean<ODD>(operand(sC + (t0 + 16 * v) * kNp, 32 * kk + 8 * q)), b[kk], S);
              const f32x4 Wt = Mma<T>::mul(clean<ODD>(operand(sY + (t0 + 16 * v) * kPp, 8 * q)), X[w], f32x4{0, 0, 0, 0});
              const int t4 = 32 * tp + 16 * v + 4 * q;
              if (v > w || sp != tp) {
                // Tiles 2 and 1 are next to each other, and so are those of one pair.
                const float c = sp == tp || (v == 0 && w == 1) ? 1.0f : s.c[v ? 1 + w : 0];
                const f32x4 e = *(const f32x4 *)(s.u + t4) * (c * to_end);
                M[v] = S * e;
                z[v] = Wt * e;
                float all = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                  const float both = z[v][r] * S[r], e_ts = both * step;
                  col[w] += both;
                  rows[v][r] += e_ts;
                  all += e_ts;
                }
                if (sp != tp && w == 0) around[0] += all;
                if (sp != tp && v == 1) around[1] += all;
              } else {
                const float hi_s = s.hi[mine], lo_s = s.lo[mine];
                const f32x4 hi = *(const f32x4 *)(s.hi + t4), lo = *(const f32x4 *)(s.lo + t4);
                float inside = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                  const int row = 4 * q + r;
                  const float e = exp2_((hi[r] - hi_s) + (lo[r] - lo_s)), at_s = keep(Wt[r], row == i16);
                  const float below = keep(Wt[r] * e, row > i16);
                  M[v][r] = keep(S[r] * e, row > i16) + keep(S[r], row == i16);
                  z[v][r] = below + at_s;
                  const float both = keep(below * S[r], row > i16);
                  own[w] += both + keep(at_s * S[r], row == i16);
                  diag += at_s;
                  inside += keep(running_sum16(moved<0x111>(both * step)), row >= i16);
                }
                inside = column_sum(inside);
                if (q == 0) sSum[wave][2][mine] = inside;
              }
              z[v] *= step;
            }
            const auto m = Fine<T>::of(__builtin_shufflevector(M[0], M[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int i = 0; i < 2; i++) dx[w][i] = mul(clean<ODD>(column<T, kPp>(lane, sY, 32 * tp, i)), m, dx[w][i]);
            Z[w] = Fine<T>::of(__builtin_shufflevector(z[0], z[1], 0, 1, 2, 3, 4, 5, 6, 7));
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int v = 0; v < 2; v++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const float sum = row_sum(rows[v][r]);
              float *to = &sSum[wave][3][32 * tp + 16 * v + 4 * q + r];
              if (i16 == 0) *to = sp == tp ? sum : *to + sum;  // (1, 1) comes before (0, 1)
            }
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const V8<T> c = clean<ODD>(column<T, kNp>(lane, sC, 32 * tp, n));
#pragma unroll
            for (int w = 0; w < 2; w++) accB[w][n] = mul(c, Z[w], accB[w][n]);
          }
          __builtin_amdgcn_sched_barrier(0);
          Fine<T> Zt[2];
#pragma unroll
          for (int v = 0; v < 2; v++) Zt[v] = turn(Z[0], Z[1], ones<T>(lane, v));
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const V8<T> b = clean<ODD>(column<T, kNp>(lane, sB, 32 * sp, n));
#pragma unroll
            for (int v = 0; v < 2; v++) accC[v][n] = mul(b, Zt[v], accC[v][n]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (!idle && step_ != 1) {
#pragma unroll
          for (int w = 0; w < 2; w++) {
            const int mine = s0 + 16 * w;
            const float below = column_sum(col[w]), in = column_sum(own[w]);
            if (q == 0) sSum[wave][4][mine] = below, sSum[wave][5][mine] = below + in;
            if (first + mine >= end) continue;
            f32x8 v = __builtin_shufflevector(dx[w][0], dx[w][1], 0, 1, 2, 3, 4, 5, 6, 7) * s.step[mine] +
                      widen<T>(operand(sY + mine * kPp, 8 * q)) * skip;
            if constexpr (ODD) {
              const bool row = from_row(odd.C, mine) || at_row(odd.B | odd.steps, mine) || after_row(odd.decays, mine);
              for (int e = 0; e < 8; e++) {
                bool none = row;
                for (int t = mine; t < kChunk; t++) none |= !finite((float)sY[t * kPp + 8 * q + e]);
                v[e] = none ? kNone : v[e];
              }
            }
            const V8<T> o = __builtin_convertvector(v, V8<T>);
            T *to = (T *)k.dx + ((uint64_t)(first + mine) * a.heads + head) * a.dim + p0 + 8 * q;
            if (k.dx_wide) {  // whole pieces of eight values, or four of 32 bits
              if (8 * q + 8 <= (int)dim) *(V8<T> *)to = o;
              else if (8 * q < (int)dim) *(V4<T> *)to = __builtin_shufflevector(o, o, 0, 1, 2, 3);
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (8 * q + e < (int)dim) to[e] = o[e];
            }
          }
        }

        if constexpr (ODD) {
          for (int w = 0; w < 2; w++)
            for (int n = 0; n < NT; n++)
              for (int r = 0; r < 4; r++) {
                const int s_ = s0 + 16 * w, t_ = t0 + 16 * w, c = place(n, 4 * q + r);
                if (!idle && step_ != 1) {  // dB of these rows is whole
                  bool none = at_row(odd.x | odd.steps, s_) || after_row(odd.decays, s_) || from_row(odd.dy, s_);
                  for (int t = s_; t < kChunk; t++) none |= !finite((float)sC[t * kNp + c]);
                  accB[w][n][r] = none ? kNone : accB[w][n][r];
                }
                if (!idle && step_ != 0) {  // and dC
                  bool none = at_row(odd.dy, t_) || up_to_row(odd.x | odd.steps | odd.decays, t_);
                  for (int s = 0; s <= t_; s++) none |= !finite((float)sB[s * kNp + c]);
                  accC[w][n][r] = none ? kNone : accC[w][n][r];
                }
              }
        }

        // dB's and dC's sums over the block's wavefronts, of two tiles of rows, and out: turns after the
        // first add to what the turn before wrote, by the same threads.
#pragma unroll 1
        for (int which = step_ == 0; which < 2; which++) {  // dC after (0, 1) and (0, 0), dB after (1, 1) and (0, 0)
          if (which && step_ == 1) break;
          const int pair = which ? sp : tp;
          T *out = (T *)(which ? k.dB : k.dC);
          float *mid = (which ? k.dBparts : k.dCparts) + (uint64_t)part * a.rows.tokens * a.groups * a.state;
#pragma unroll
          for (int n0 = 0; n0 < NT; n0 += G) {
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
              for (int n = 0; n < G; n++)
                if (which) *(f32x4 *)(sRed[wave] + ((w * G + n) * 64 + lane) * 4) = accB[w][n0 + n];
                else *(f32x4 *)(sRed[wave] + ((w * G + n) * 64 + lane) * 4) = accC[w][n0 + n];
            __syncthreads();
#pragma unroll
            for (uint32_t item = wave * 64 + lane; item < G * 128; item += 64 * W) {
              const uint32_t of = item & 63, w = item >> 6 & 1, n = item >> 7;
              const uint32_t row = first + (2 * pair + w) * 16 + (of & 15), c = place(n0 + n, 4 * (of >> 4));
              const bool there = row < end && c < a.state;
              const uint64_t to = ((uint64_t)row * a.groups + group) * a.state + c;
              const bool adds = sub > sub0, keeps = sub + 1 < sub1 || k.parts > 1;
              f32x4 v = {0, 0, 0, 0};
              if (there && adds) {
                if (k.mid_wide) {
                  v = *(const f32x4 *)(mid + to);
                } else {
#pragma unroll
                  for (int e = 0; e < 4; e++) v[e] = c + e < a.state ? mid[to + e] : 0.0f;
                }
              }
#pragma unroll
              for (int i = 0; i < W; i++) v += *(const f32x4 *)(sRed[i] + ((w * G + n) * 64 + of) * 4);
              if (!there) continue;
              const V4<T> o = __builtin_convertvector(v, V4<T>);
              if (k.mid_wide && keeps) *(f32x4 *)(mid + to) = v;
              else if (k.shared_wide && !keeps) *(V4<T> *)(out + to) = o;
              else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  if (c + e >= a.state) break;
                  if (keeps) mid[to + e] = v[e];
                  else out[to + e] = o[e];
                }
              }
            }
            __syncthreads();
          }
        }
      }

      // A row a lane: the gradients at its decay and its step, of all the head's wavefronts.
      const int lane = anew(lane0);
      if (!idle) {
        const bool there = first + lane < end && (more || lane < 32);
        const float step = s.step[lane];
        const float(&sum)[6][kChunk] = sSum[wave];
        // Their decays' errors would be common to all rows that the sums reach.
        const double l = s.l[lane], r = there && has_g ? (double)sum[1][lane] * power64(d.total - l) : 0.0;
        const double into = r * (double)step, before = running_sum(into);
        const double q_t = there && has_h ? (double)sum[0][lane] * power64(l) : 0.0, through = running_sum(q_t);
        const double base = has_g && has_h ? power64(d.total) * (double)wave_sum(inner) : 0.0;
        const double row = there ? (double)sum[3][lane] : 0.0, rows_to = running_sum16(row);
        const double col_s = there ? (double)(sum[4][lane] * step) : 0.0, cols_to = running_sum16(col_s);
        const float second = wave_sum(around[0]), third = wave_sum(around[1]);
        double inside = there ? (double)sum[2][lane] : 0.0;
        inside += (__shfl(rows_to, lane | 15) - (rows_to - row)) + (cols_to - col_s);
        inside += (double)(lane >> 4 == 1 ? second : lane >> 4 == 2 ? third : 0.0f);
        sDa[wave][lane] = (float)(base + (before - into) + (lane_of(through, 63) - (through - q_t)) + inside);
        sDirect[wave][lane] = there ? (float)r + sum[5][lane] : 0.0f;
        const float all = wave_sum(diag);
        if (lane == 0) sDiag[wave] = all;
        if constexpr (ODD) {
          if (from_row(odd.dy | odd.C, lane) || before_row(odd.x | odd.B | odd.steps, lane) || odd.decays || odd.g) sDa[wave][lane] = kNone;
          if (from_row(odd.dy | odd.C, lane) || at_row(odd.x | odd.B, lane) || after_row(odd.decays, lane)) sDirect[wave][lane] = kNone;
          if (lane == 0 && (odd.dy | odd.x)) sDiag[wave] = kNone;
        }
      } else {
        sDa[wave][lane] = sDirect[wave][lane] = 0.0f;
        if (lane == 0) sDiag[wave] = 0.0f;
      }
      __syncthreads();
      if (!idle && tile == 0) {
        float da = 0.0f, direct = 0.0f, all = 0.0f;
        for (uint32_t i = 0; i < a.tiles; i++) {
          da += sDa[wave + i][lane];
          direct += sDirect[wave + i][lane];
          all += sDiag[wave + i];
        }
        if (lane == 0) sumD += (double)all;
        if (first + lane < end) {
          const float dstep = (direct + A * da) * sigmoid<>(raw_now + bias);
          sumA += (double)((ODD && at_row(odd.steps, lane) ? kNone : s.step[lane]) * da);
          sumBias += (double)dstep;
          ((T *)k.ddt)[(uint64_t)(first + lane) * a.heads + head] = (T)dstep;
        }
      }
      fetch(j - 1);
      if (!idle && (j || (!at.number && k.dinitial))) {
        V8<T> ys[2][2];
#pragma unroll
        for (int kk = 0; kk < 2; kk++)
#pragma unroll
          for (int i = 0; i < 2; i++) ys[kk][i] = column<T, kPp>(lane, sY, 32 * kk, i);
        advance<T, NT, 2>(lane, g, ys, sC, s.u, d.from, d.whole);
        if (ODD && odd.decays) {
#pragma unroll
          for (int n = 0; n < NT; n++) g[n][0] = g[n][1] = f32x4{kNone, kNone, kNone, kNone};
        }
      }
    }
    if (idle) continue;
    if (!at.number && k.dinitial)
      put_state<NT, 2>(g, k.dinitial + ((uint64_t)at.seq * a.heads + head) * whole + cell, dim, a.state, a.state_wide);
    if (tile == 0) {
      sumA = wave_sum(sumA), sumD = wave_sum(sumD), sumBias = wave_sum(sumBias);
      if (lane0 == 0) {
        double *to = k.sums + ((uint64_t)number * a.heads + head) * 3;
        to[0] = sumA, to[1] = sumD, to[2] = sumBias;
      }
    }
  }
}

// The parts' sums of dB and dC, in their order.
template <class T>
__global__ __launch_bounds__(256) void grad_parts(Grad k) {
  const uint64_t n = (uint64_t)k.s.rows.tokens * k.s.groups * k.s.state, at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  uint32_t first, end;
  k.s.rows.owned(first, end);
  const uint32_t row = (uint32_t)(at / (k.s.groups * k.s.state));
  if (row < first || row >= end) return;  // cleared, and there are no parts
  float b = 0.0f, c = 0.0f;
  for (uint32_t p = 0; p < k.parts; p++) {
    b += k.dBparts[p * n + at];
    c += k.dCparts[p * n + at];
  }
  ((T *)k.dB)[at] = (T)b;
  ((T *)k.dC)[at] = (T)c;
}

// The pieces' sums of the parameters' gradients, a block a head.
__global__ __launch_bounds__(1024) void grad_sums(Grad k) {
  __shared__ double part[3][1024];
  const uint32_t head = blockIdx.x;
  double v[3] = {0.0, 0.0, 0.0};
  for (uint32_t seq = threadIdx.x; seq < k.s.rows.seqs; seq += 1024) {
    uint32_t start, stop;
    k.s.rows.of(seq, start, stop);
    const uint32_t n = stop > start ? (stop - start - 1) / k.s.size + 1 : 1;
    const double *from = k.sums + ((uint64_t)(start / k.s.size + seq) * k.s.heads + head) * 3;
    for (uint32_t j = 0; j < n; j++)
      for (int i = 0; i < 3; i++) v[i] += from[(uint64_t)j * k.s.heads * 3 + i];
  }
  for (int i = 0; i < 3; i++) part[i][threadIdx.x] = v[i];
  for (int m = 512; m; m >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < m)
      for (int i = 0; i < 3; i++) part[i][threadIdx.x] += part[i][threadIdx.x + m];
  }
  if (threadIdx.x) return;
  k.dA[head] = (float)part[0][0];
  if (k.dD) k.dD[head] = (float)part[1][0];
  if (k.dbias) k.dbias[head] = (float)part[2][0];
}

// The gradients at the starts of pieces after their sequence's first, from those of their own y, from each
// cut sequence's end.
__global__ __launch_bounds__(kThreads) void grad_join(Grad k) {
  const Scan &a = k.s;
  const uint32_t head = blockIdx.x % a.heads;
  uint32_t seq, n;
  if (!joined(a, blockIdx.x / a.heads, seq, n)) return;
  const uint64_t base = a.rows.at(seq) / a.size, whole = (uint64_t)a.dim * a.state, step = a.heads * whole;
  for (uint64_t e = blockIdx.y * kThreads + threadIdx.x; e < whole; e += (uint64_t)gridDim.y * kThreads) {
    float g = k.dfinal ? k.dfinal[((uint64_t)seq * a.heads + head) * whole + e] : 0.0f;
    float *at = k.g_starts + (base * a.heads + head) * whole + e;
    const double *totals = a.totals + base * a.heads + head;
    for (uint32_t j = 0; j < n; j += kAhead) {  // from the end
      float own[kAhead], decay[kAhead];
#pragma unroll
      for (uint32_t i = 0; i < kAhead; i++) {
        const uint32_t place = j + i + 1 < n ? n - 2 - j - i : n - 2;
        own[i] = at[place * step];
        decay[i] = (float)totals[(uint64_t)place * a.heads];
      }
#pragma unroll
      for (uint32_t i = 0; i < kAhead; i++) {
        if (j + i >= n) break;
        if (j + i) at[(n - 1 - j - i) * step] = g;
        g = exp2_(decay[i]) * g + own[i];
      }
    }
  }
}
__global__ __launch_bounds__(kThreads) void scan_join(Scan a);
__global__ __launch_bounds__(1024) void scan_order(Scan a);

namespace {

uint32_t tiles_of(uint32_t dim) { return dim <= 32 ? 1 : dim <= 64 ? 2 : 4; }

// Where a gradient's scratch memory begins, and how much there is.
struct Plan {
  uint32_t size, pieces, waves, subs, parts;
  bool ordered;
  uint64_t cut, back, totals, order, h, sums, dB, dC, bytes;
};
Plan plan_of(const uor_trunk_scan_args *s) {
  Plan p{};
  const uint32_t tiles = tiles_of(s->dim), share = s->heads / s->groups, units = share * tiles;
  const uint64_t n16 = s->state <= 32 ? 32 : s->state <= 64 ? 64 : 128;
  p.size = piece_rows(s->tokens, s->seqs, s->heads * tiles, 64);
  p.pieces = pieces(s->tokens, s->seqs, p.size);
  // As many wavefronts to a block as its LDS has room for, whole heads each turn.
  const uint32_t most = 4;
  p.waves = 1;
  while (p.waves < units && p.waves < most) p.waves *= 2;
  p.subs = (units + p.waves - 1) / p.waves;
  // Blocks of a group share its turns where the pieces alone do not fill the card.
  const uint64_t blocks = (uint64_t)p.pieces * s->groups;
  p.parts = blocks >= 512 ? 1 : (uint32_t)((511 + blocks) / blocks);
  if (p.parts > p.subs) p.parts = p.subs;
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t begin = at;
    at += (bytes + 255) / 256 * 256;
    return begin;
  };
  const bool cut = p.size < s->tokens;
  const uint64_t later = cut ? s->tokens / p.size + 1 : 0, starts = later * s->heads * s->dim * s->state * 4;
  p.cut = take(starts), p.back = take(starts);
  // As in the scan; two wavefronts a SIMD, and each chunk takes several times as long. Without and with it:
  // 520 sequences of up to 128 (2,080 wavefronts) 308 and 250 us, 520 of up to 64 (16,710 rows) 180 and 180,
  // 2,000 of up to 20 303 and 277, 8,000 of up to 20 1,043 and 1,037; below the borders 300 of up to 200 would
  // gain (292 and 248), 300 of up to 60 not (116 and 117).
  p.ordered = s->seqs > 1 && s->seqs <= 8192 && (uint64_t)p.pieces * s->groups * p.parts * p.waves > 2048 && s->tokens >= 16384;
  p.order = take(p.ordered ? ((uint64_t)p.pieces + 1) * 8 : 0);
  p.totals = take(later * s->heads * 8);
  // States are kept of chunks that have one before them and one after them in their piece.
  p.h = take(p.size > 2 * kChunk && s->tokens > 2 * kChunk ? ((uint64_t)s->tokens / kChunk + 1) * s->heads * tiles * n16 * 32 * 4 : 0);
  p.sums = take((uint64_t)p.pieces * s->heads * 3 * 8);
  const uint64_t rows = p.subs > 1 ? (uint64_t)p.parts * s->tokens * s->groups * s->state * 4 : 0;
  p.dB = take(rows), p.dC = take(rows);
  p.bytes = at;
  return p;
}

template <class T, int NT, int W>
int launch(const Grad &k, hipStream_t stream) {
  const Scan &a = k.s;
  if (a.starts) {
    constexpr int E = W < 4 ? W : 4;
    Scan s = a;
    s.tiles = (a.dim + 31) / 32;
    const uint32_t units = a.heads / a.groups * s.tiles;
    const dim3 grid(grid_of(a.later, a.groups * ((units + E - 1) / E))), join = join_of(a);
    hipLaunchKernelGGL((scan_ends<T, NT, 2, E, false>), grid, dim3(64 * E), 0, stream, s);
    hipLaunchKernelGGL(scan_join, join, dim3(kThreads), 0, stream, s);
    s.x = k.dy, s.x_stride = a.y_stride, s.x_wide = k.dy_wide;
    s.B = a.C, s.b_stride = a.c_stride, s.b_wide = a.c_wide;
    s.starts = k.g_starts;
    hipLaunchKernelGGL((scan_ends<T, NT, 2, E, true>), grid, dim3(64 * E), 0, stream, s);
    hipLaunchKernelGGL(grad_join, join, dim3(kThreads), 0, stream, k);
  }
  if (a.order) hipLaunchKernelGGL(scan_order, dim3(1), dim3(1024), 0, stream, a);
  hipLaunchKernelGGL((grad_rows<T, NT, W, false>), dim3(grid_of(a.pieces, a.groups * k.parts)), dim3(64 * W), 0, stream, k);
  hipLaunchKernelGGL((grad_rows<T, NT, W, true>), dim3(grid_of(a.pieces, a.groups * k.parts)), dim3(64 * W), 0, stream, k);
  if (k.parts > 1 && a.rows.tokens) {
    const uint64_t n = (uint64_t)a.rows.tokens * a.groups * a.state;
    hipLaunchKernelGGL(grad_parts<T>, dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, stream, k);
  }
  hipLaunchKernelGGL(grad_sums, dim3(a.heads), dim3(1024), 0, stream, k);
  return launched();
}
template <class T, int NT>
int launch(const Grad &k, uint32_t waves, hipStream_t stream) {
  return waves == 1 ? launch<T, NT, 1>(k, stream) : waves == 2 ? launch<T, NT, 2>(k, stream) : launch<T, NT, 4>(k, stream);
}
template <class T>
int launch(const Grad &k, uint32_t waves, hipStream_t stream) {
  return k.s.state <= 32 ? launch<T, 2>(k, waves, stream)
                         : k.s.state <= 64 ? launch<T, 4>(k, waves, stream) : launch<T, 8>(k, waves, stream);
}

}  // namespace
}  // namespace trunk

using namespace trunk;

extern "C" uint64_t uor_trunk_scan_backward_workspace_bytes(const uor_trunk_scan_args *s) {
  return check_scan(s, false) ? 0 : plan_of(s).bytes;
}

extern "C" int uor_trunk_scan_backward_async(const uor_trunk_scan_args *s, void *workspace, uint64_t bytes, void *stream) {
  if (const int e = check_scan(s, false)) return e;
  if (s->tokens && (!s->dy || !s->dx || !s->ddt || !s->dB || !s->dC)) return fail(-1, "null dy, dx, ddt, dB or dC");
  if (!s->dA) return fail(-1, "null dA");
  const Plan p = plan_of(s);
  if (!workspace || bytes < p.bytes || (uintptr_t)workspace % 16)
    return fail(-1, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)p.bytes);
  const uint32_t tiles = tiles_of(s->dim);
  if (((uint64_t)p.pieces + kXcds) * s->heads * tiles > 0x7fffffffu) return fail(-1, "too many rows and heads for one call");
  const uint32_t size = s->dtype == UOR_TRUNK_BF16 ? 2 : 4;
  char *base = (char *)workspace;
  Grad k{};
  k.s = scan_of(s, p.size);
  k.s.tiles = tiles;
  if (p.size < s->tokens) {
    k.s.starts = (float *)(base + p.cut);
    k.g_starts = (float *)(base + p.back);
    k.s.totals = (double *)(base + p.totals);
  }
  if (p.ordered) k.s.order = (uint32_t *)(base + p.order);
  k.s.state_wide = s->state % 4 == 0 && aligned16(s->initial, 0, 4) && aligned16(s->dfinal, 0, 4) && aligned16(s->dinitial, 0, 4);
  k.dy = s->dy, k.dfinal = s->dfinal, k.subs = p.subs, k.parts = p.parts;
  k.h = (float *)(base + p.h), k.sums = (double *)(base + p.sums);
  k.dBparts = (float *)(base + p.dB), k.dCparts = (float *)(base + p.dC);
  k.dx = s->dx, k.ddt = s->ddt, k.dB = s->dB, k.dC = s->dC, k.dA = s->dA, k.dD = s->dD, k.dbias = s->ddt_bias, k.dinitial = s->dinitial;
  k.dy_wide = wide_rows(s->dy, k.s.y_stride, s->dim, size);
  k.dx_wide = aligned16(s->dx, 0, size) && s->dim * size % 16 == 0;
  k.shared_wide = aligned16(s->dB, 0, size) && aligned16(s->dC, 0, size) && s->state % 4 == 0;
  k.mid_wide = s->state % 4 == 0;
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(k, p.waves, (hipStream_t)stream) : launch<float>(k, p.waves, (hipStream_t)stream);
}
