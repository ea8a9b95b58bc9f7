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
// W_ts e_ts D_s is summed over a group's heads before its two products with B and C. With
// E_ts = W_ts S_ts e_ts D_s, q_t = e^(l_t) C_t . h^T dy_t and r_s = D_s e^(l_end - l_s) B_s . g^T x_s,
// the gradient at the logarithm of row u's decay is
//
//   da_u = e^(l_end) <g, h> + sum_(t >= u) q_t + sum_(s < u) r_s + sum_(t >= u, s < u) E_ts,
//
// whose last sum is the sum over t >= u of E's row t less its column t. At the step itself it is
// (r_u + column u of E) / D_u + A da_u, where what D_u divides is summed without it.
//
// First all chunks' h and g are written by two launches that go along the sequences and back (cut
// into pieces where those are long, as in the scan); then every chunk of every group is a block.
#include "scan.h"

namespace trunk {

struct Grad {
  Scan s;               // pieces of the sweeps; s.starts as there, for the sweep that runs
  const void *dy;
  const float *dfinal;
  uint32_t chunks;      // places of chunks
  uint32_t parts;       // blocks that share a group's heads
  float *h, *g, *gt;    // [chunks][heads * tiles][16 NT x 16 PW]: h and gt by rows of state, g by rows of dim
  float *sums;          // [chunks][heads][3]: dA, dD, ddt_bias
  float *dBparts, *dCparts;  // [parts][tokens][groups][state], with more than one part
  void *dx, *ddt, *dB, *dC;
  float *dA, *dD, *dbias, *dinitial;
  bool dy_wide, dx_wide;
};

// The states along a piece: forward from its start, or back from its end (x then is dy, B is C).
// STORE: every chunk's is written; otherwise only the piece's last, for the join.
template <class T, int NT, int PW, bool BACK, bool STORE>
__global__ __launch_bounds__(kThreads) void grad_states(Grad k) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kLp = pitch<T>(kChunk), kTiles = NT * PW / 4;
  __shared__ __align__(16) T sBt[kN * kLp], sXt[kP * kLp];
  __shared__ Decays d;
  const Scan &a = k.s;
  uint32_t number, place;
  place_of(blockIdx.x, a.heads * a.tiles, number, place);
  const uint32_t tile = place % a.tiles, head = place / a.tiles, p0 = tile * kP;
  Piece at;
  if (number >= a.pieces || !piece(a.rows, number, a.size, at)) return;
  // The sequence's last piece this way has nothing after it to start.
  const bool last = BACK ? at.first == at.start : at.end == at.stop;
  if (!STORE && last) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
  const uint32_t group = head / (a.heads / a.groups);
  const T *x = (const T *)(BACK ? k.dy : a.x) + head * a.dim + p0, *dt = (const T *)a.dt + head;
  const T *B = (const T *)(BACK ? a.C : a.B) + group * a.state;
  const int64_t x_stride = BACK ? a.y_stride : a.x_stride, b_stride = BACK ? a.c_stride : a.b_stride;
  const bool x_wide = BACK ? k.dy_wide : a.x_wide, b_wide = BACK ? a.c_wide : a.b_wide;
  const uint32_t dim = a.dim - p0 < (uint32_t)kP ? a.dim - p0 : kP;
  const float A = a.A[head], bias = a.bias ? a.bias[head] : 0.0f;
  const uint64_t whole = (uint64_t)a.dim * a.state;
  const Own<NT, PW> own;
  f32x4 h[kTiles];
  const float *from = BACK ? k.dfinal : a.initial;
  const uint64_t slot = (uint64_t)number * a.heads + head;
  load_state<NT, PW>(h, own, !STORE ? nullptr : a.starts && (BACK || at.number) ? a.starts + slot * whole : from ? from + ((uint64_t)at.seq * a.heads + head) * whole : nullptr,
                     p0, a.dim, a.state);
  const uint32_t chunks = (at.end - at.first + kChunk - 1) / kChunk;
  const uint64_t base = at.start / kChunk + at.seq + (at.first - at.start) / kChunk;
  double total = 0.0;
  for (uint32_t i = 0; i < chunks; i++) {
    const uint32_t j = BACK ? chunks - 1 - i : i;
    const uint32_t first = at.first + j * kChunk, end = at.end - first > kChunk ? first + kChunk : at.end;
    if constexpr (STORE) {
      const bool zeros = !from && (BACK ? end == at.stop : first == at.start);  // never read
      if (!zeros) {
        const uint64_t to = ((base + j) * a.heads * a.tiles + place) * (kN * kP);
#pragma unroll
        for (int e = 0; e < kTiles; e++) {
          const int n = (own.n + e) * 16 + 4 * q, p = own.p * 16 + i16;
          float *turned = (BACK ? k.gt : k.h) + to;
#pragma unroll
          for (int r = 0; r < 4; r++) turned[(n + r) * kP + p] = h[e][r];
          if (BACK) *(f32x4 *)(k.g + to + p * kN + n) = h[e];
        }
      }
      // The state after the sequence's last chunk this way is read by no chunk.
      if (last && i + 1 == chunks && !(BACK && k.dinitial)) break;
    }
    __syncthreads();
    stage<T, kN>((T *)nullptr, sBt, B, b_stride, first, end, a.state, b_wide);
    stage<T, kP>((T *)nullptr, sXt, x, x_stride, first, end, dim, x_wide);
    if (wave == 0) decays(d, dt, a.dt_stride, first, end, A, bias);
    __syncthreads();
    advance<T, NT, PW>(h, own, sXt, sBt, BACK ? d.from : d.to, d.whole);
    total += d.total;
  }
  if constexpr (STORE) {
    if (BACK && k.dinitial && last)
      store_state<NT, PW>(h, own, k.dinitial + ((uint64_t)at.seq * a.heads + head) * whole, p0, a.dim, a.state);
  } else {
    store_state<NT, PW>(h, own, a.starts + slot * whole, p0, a.dim, a.state);
    if (threadIdx.x == 0 && p0 == 0) a.totals[slot] = total;
  }
}

template <class T, int NT, int PW>
__global__ __launch_bounds__(kThreads) void grad_rows(Grad k) {
  constexpr int kN = 16 * NT, kP = 16 * PW, kNp = pitch<T>(kN), kPp = pitch<T>(kP), kLp = pitch<T>(kChunk);
  constexpr int kZp = kChunk + 4;
  // W summed over heads is handed over where x and dy were.
  constexpr int kRowsBytes = 2 * kChunk * kPp * (int)sizeof(T), kZBytes = kChunk * kZp * 4;
  __shared__ __align__(16) T sB[kChunk * kNp], sC[kChunk * kNp], sYt[kP * kLp];
  __shared__ __align__(16) char sRows[kRowsBytes > kZBytes ? kRowsBytes : kZBytes];
  __shared__ Decays d;
  __shared__ float sQ[kChunk], sR[kChunk], sCol[kChunk], sDirect[kChunk], sRow[4][kChunk], sBase[4], sDiag[4];
  T *sX = (T *)sRows, *sY = sX + kChunk * kPp;
  float *sZ = (float *)sRows;
  const Scan &a = k.s;
  uint32_t number, place;
  place_of(blockIdx.x, a.groups * k.parts, number, place);
  Piece at;
  if (number >= k.chunks || !piece(a.rows, number, kChunk, at) || at.first == at.end) return;
  const uint32_t group = place / k.parts, part = place % k.parts, share = a.heads / a.groups;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
  const bool has_h = a.initial || at.first != at.start, has_g = k.dfinal || at.end != at.stop;
  const int mine = wave * 16 + i16;  // this lane's column: its row s, and its row t
  const uint32_t row = at.first + mine;

  stage<T, kN>(sB, (T *)nullptr, (const T *)a.B + group * a.state, a.b_stride, at.first, at.end, a.state, a.b_wide);
  stage<T, kN>(sC, (T *)nullptr, (const T *)a.C + group * a.state, a.c_stride, at.first, at.end, a.state, a.c_wide);
  __syncthreads();
  f32x4 S[4], Z[4], accB[NT], accC[NT];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    S[t] = Z[t] = f32x4{0, 0, 0, 0};
    if (t < wave) continue;
#pragma unroll
    for (int n = 0; n < kN; n += 32)
      S[t] = Mma<T>::mul(operand(sC + (t * 16 + i16) * kNp, n + 8 * q), operand(sB + mine * kNp, n + 8 * q), S[t]);
  }
#pragma unroll
  for (int n = 0; n < NT; n++) accB[n] = accC[n] = f32x4{0, 0, 0, 0};

  for (uint32_t head = group * share + share * part / k.parts; head < group * share + share * (part + 1) / k.parts; head++) {
    const float A = a.A[head], bias = a.bias ? a.bias[head] : 0.0f, skip = a.D ? a.D[head] : 0.0f;
    double da = 0.0;             // of row `lane`, on the first wavefront
    float direct = 0.0f, diag = 0.0f;
    for (uint32_t tile = 0; tile < a.tiles; tile++) {
      const uint32_t p0 = tile * kP, dim = a.dim - p0 < (uint32_t)kP ? a.dim - p0 : kP;
      __syncthreads();
      stage<T, kP>(sX, (T *)nullptr, (const T *)a.x + head * a.dim + p0, a.x_stride, at.first, at.end, dim, a.x_wide);
      stage<T, kP>(sY, sYt, (const T *)k.dy + head * a.dim + p0, a.y_stride, at.first, at.end, dim, k.dy_wide);
      if (wave == 0 && tile == 0) decays(d, (const T *)a.dt + head, a.dt_stride, at.first, at.end, A, bias);
      __syncthreads();
      const uint64_t held = ((uint64_t)number * a.heads * a.tiles + head * a.tiles + tile) * (kN * kP);
      const float step = d.step[mine], tail = d.tail[mine], from = d.from[mine], hi = d.hi[mine], lo = d.lo[mine];

      // dx: what comes through the state after the chunk.
      f32x4 dx[PW];
#pragma unroll
      for (int i = 0; i < PW; i++) dx[i] = f32x4{0, 0, 0, 0};
      if (has_g) {
#pragma unroll
        for (int n = 0; n < kN; n += 32) {
          const V8<T> b = operand(sB + mine * kNp, n + 8 * q);
#pragma unroll
          for (int i = 0; i < PW; i++)
            dx[i] = Mma<T>::mul(Mma<T>::split(*(const f32x8 *)(k.g + held + (i * 16 + i16) * kN + n + 8 * q)), b, dx[i]);
        }
#pragma unroll
        for (int i = 0; i < PW; i++) dx[i] *= tail;
      }
      // W, and through it the chunk's own part of dx and of the sums.
      float col = 0.0f, own = 0.0f;
      f32x4 M[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        M[t] = f32x4{0, 0, 0, 0};
        if (t < wave) continue;
        f32x4 w = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kP; p += 32)
          w = Mma<T>::mul(operand(sY + (t * 16 + i16) * kPp, p + 8 * q), operand(sX + mine * kPp, p + 8 * q), w);
        float rows[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int tt = t * 16 + 4 * q + r;
          const float e = tt > mine ? exp2_((d.hi[tt] - hi) + (d.lo[tt] - lo)) : 1.0f;
          const float z = tt >= mine ? w[r] * e : 0.0f;
          M[t][r] = tt >= mine ? S[t][r] * e : 0.0f;
          Z[t][r] += z * step;
          const float both = tt >= mine ? z * S[t][r] : 0.0f;
          own += tt == mine ? both : 0.0f;
          diag += tt == mine ? w[r] : 0.0f;
          const float off = tt > mine ? both : 0.0f;
          col += off;
          rows[r] = off * step;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
#pragma unroll
          for (int m = 1; m < 16; m <<= 1) rows[r] += __shfl_xor(rows[r], m);
          if (i16 == 0) sRow[wave][t * 16 + 4 * q + r] = rows[r];
        }
      }
#pragma unroll
      for (int t = 0; t < 4; t++)
        if (t < wave && lane < 16) sRow[wave][t * 16 + lane] = 0.0f;
#pragma unroll
      for (int pair = 0; pair < 2; pair++) {
        if (2 * pair + 1 < wave) continue;
        const auto m = Mma<T>::split(__builtin_shufflevector(M[2 * pair], M[2 * pair + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int i = 0; i < PW; i++) dx[i] = Mma<T>::mul(operand_tiles(sYt + (i * 16 + i16) * kLp, pair * 32 + 4 * q), m, dx[i]);
      }
      if (row < at.end) {
        T *to = (T *)k.dx + ((uint64_t)row * a.heads + head) * a.dim + p0;
#pragma unroll
        for (int i = 0; i < PW; i++) {
          const uint32_t p = i * 16 + 4 * q;
          const V4<T> y = *(const V4<T> *)(sY + mine * kPp + p);
          V4<T> v;
#pragma unroll
          for (int r = 0; r < 4; r++) v[r] = (T)(step * dx[i][r] + skip * (float)y[r]);
          if (k.dx_wide && p + 4 <= dim) {
            *(V4<T> *)(to + p) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 4; r++)
              if (p + r < dim) to[p + r] = v[r];
          }
        }
      }
      // dB and dC: what comes through the states.
      float through = 0.0f, into = 0.0f, inner = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        f32x4 vb = {0, 0, 0, 0}, vc = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < kP; p += 32) {
          const uint64_t place8 = held + (n * 16 + i16) * kP + p + 8 * q;
          f32x8 g, h;
          if (has_g) {
            g = *(const f32x8 *)(k.gt + place8);
            vb = Mma<T>::mul(Mma<T>::split(g), operand(sX + mine * kPp, p + 8 * q), vb);
          }
          if (has_h) {
            h = *(const f32x8 *)(k.h + place8);
            vc = Mma<T>::mul(Mma<T>::split(h), operand(sY + mine * kPp, p + 8 * q), vc);
          }
          if (has_g && has_h && n % 4 == wave) {
#pragma unroll
            for (int e = 0; e < 8; e++) inner += g[e] * h[e];
          }
        }
        vb *= tail;
        vc *= from;
        const V4<T> b = *(const V4<T> *)(sB + mine * kNp + n * 16 + 4 * q), c = *(const V4<T> *)(sC + mine * kNp + n * 16 + 4 * q);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          into += vb[r] * (float)b[r];
          through += vc[r] * (float)c[r];
        }
        accB[n] += vb * step;
        accC[n] += vc;
      }
      // A column's sums over its four lanes, and the wavefront's part of <g, h>.
#pragma unroll
      for (int m = 16; m < 64; m <<= 1) {
        into += __shfl_xor(into, m);
        through += __shfl_xor(through, m);
        col += __shfl_xor(col, m);
        own += __shfl_xor(own, m);
      }
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) inner += __shfl_xor(inner, m);
      if (q == 0) {
        sQ[mine] = through;
        sR[mine] = into;
        sCol[mine] = col;
        sDirect[mine] = into + col + own;
      }
      if (lane == 0) sBase[wave] = inner;
      __syncthreads();
      if (wave == 0) {
        // da of row u = lane: sums over t >= u less those over s >= u, as one sum from the end, and the
        // r of the rows before.
        const float at_step = d.step[lane];
        const double r = (double)(sR[lane] * at_step);
        double later = (double)sQ[lane] + ((double)((sRow[0][lane] + sRow[1][lane]) + (sRow[2][lane] + sRow[3][lane])) - (double)(sCol[lane] * at_step));
        double before = r;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
          const double l = __shfl_down(later, m), b = __shfl_up(before, m);
          if (lane + m < 64) later += l;
          if (lane >= m) before += b;
        }
        const double base = (double)d.whole * (double)((sBase[0] + sBase[1]) + (sBase[2] + sBase[3]));
        da += later + (before - r) + base;
        direct += sDirect[lane];
      }
    }
    // The head's parameters and its steps.
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) diag += __shfl_xor(diag, m);
    if (lane == 0) sDiag[wave] = diag;
    __syncthreads();
    if (wave == 0) {
      float dstep = 0.0f, dA = 0.0f;
      if (at.first + lane < at.end) {
        const float raw = (float)((const T *)a.dt)[(int64_t)(at.first + lane) * a.dt_stride + head] + bias;
        dstep = (direct + A * (float)da) * sigmoid(raw);
        dA = d.step[lane] * (float)da;
        ((T *)k.ddt)[(uint64_t)(at.first + lane) * a.heads + head] = (T)dstep;
      }
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        dstep += __shfl_xor(dstep, m);
        dA += __shfl_xor(dA, m);
      }
      if (lane == 0) {
        float *to = k.sums + ((uint64_t)number * a.heads + head) * 3;
        to[0] = dA;
        to[1] = (sDiag[0] + sDiag[1]) + (sDiag[2] + sDiag[3]);
        to[2] = dstep;
      }
    }
  }

  // The chunk's own part of dB and dC, of all heads at once.
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 4; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) sZ[(t * 16 + 4 * q + r) * kZp + mine] = Z[t][r];
  __syncthreads();
#pragma unroll
  for (int pair = 0; pair < 2; pair++) {
    const auto zb = Mma<T>::split(__builtin_shufflevector(Z[2 * pair], Z[2 * pair + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    const auto zc = Mma<T>::split(*(const f32x8 *)(sZ + mine * kZp + pair * 32 + 8 * q));
#pragma unroll
    for (int n = 0; n < NT; n++) {
      V8<T> c, b;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        c[e] = sC[(pair * 32 + (e >> 2) * 16 + 4 * q + (e & 3)) * kNp + n * 16 + i16];
        b[e] = sB[(pair * 32 + 8 * q + e) * kNp + n * 16 + i16];
      }
      accB[n] = Mma<T>::mul(c, zb, accB[n]);
      accC[n] = Mma<T>::mul(b, zc, accC[n]);
    }
  }
  if (row >= at.end) return;
  const uint64_t to = ((uint64_t)row * a.groups + group) * a.state;
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t c = n * 16 + 4 * q + r;
      if (c >= a.state) continue;
      if (k.parts == 1) {
        ((T *)k.dB)[to + c] = (T)accB[n][r];
        ((T *)k.dC)[to + c] = (T)accC[n][r];
      } else {
        const uint64_t plane = (uint64_t)part * a.rows.tokens * a.groups * a.state;
        k.dBparts[plane + to + c] = accB[n][r];
        k.dCparts[plane + to + c] = accC[n][r];
      }
    }
}

// The parts' sums of dB and dC, in their order.
template <class T>
__global__ __launch_bounds__(256) void grad_parts(Grad k) {
  const uint64_t n = (uint64_t)k.s.rows.tokens * k.s.groups * k.s.state, at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  float b = 0.0f, c = 0.0f;
  for (uint32_t p = 0; p < k.parts; p++) {
    b += k.dBparts[p * n + at];
    c += k.dCparts[p * n + at];
  }
  ((T *)k.dB)[at] = (T)b;
  ((T *)k.dC)[at] = (T)c;
}

// The chunks' sums of the parameters' gradients, a block a head. Places of chunks that no sequence
// has hold nothing, and are left out as they were in grad_rows.
__global__ __launch_bounds__(256) void grad_sums(Grad k) {
  __shared__ double part[3][256];
  const uint32_t head = blockIdx.x;
  double v[3] = {0.0, 0.0, 0.0};
  for (uint32_t c = threadIdx.x; c < k.chunks; c += 256) {
    Piece at;
    if (!piece(k.s.rows, c, kChunk, at) || at.first == at.end) continue;
    for (int i = 0; i < 3; i++) v[i] += (double)k.sums[((uint64_t)c * k.s.heads + head) * 3 + i];
  }
  for (int i = 0; i < 3; i++) part[i][threadIdx.x] = v[i];
  for (int m = 128; m; m >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < m)
      for (int i = 0; i < 3; i++) part[i][threadIdx.x] += part[i][threadIdx.x + m];
  }
  if (threadIdx.x) return;
  k.dA[head] = (float)part[0][0];
  if (k.dD) k.dD[head] = (float)part[1][0];
  if (k.dbias) k.dbias[head] = (float)part[2][0];
}

// The pieces' end states into their start states, from each sequence's end.
__global__ __launch_bounds__(kThreads) void grad_join(Grad k) {
  const Scan &a = k.s;
  const uint32_t seq = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  uint32_t start, end;
  a.rows.of(seq, start, end);
  const uint32_t n = end > start ? (end - start - 1) / a.size + 1 : 1;
  const uint64_t base = start / a.size + seq, whole = (uint64_t)a.dim * a.state;
  for (uint64_t e = blockIdx.y * kThreads + threadIdx.x; e < whole; e += (uint64_t)gridDim.y * kThreads) {
    float g = k.dfinal ? k.dfinal[((uint64_t)seq * a.heads + head) * whole + e] : 0.0f;
    for (uint32_t j = n; j-- > 0;) {
      const uint64_t slot = (base + j) * a.heads + head;
      float *at = a.starts + slot * whole + e;
      const float own = j ? *at : 0.0f, decay = j ? exp2_((float)a.totals[slot]) : 0.0f;
      *at = g;
      g = decay * g + own;
    }
  }
}
__global__ __launch_bounds__(kThreads) void scan_join(Scan a);

namespace {

// Where a gradient's scratch memory begins, and how much there is.
struct Plan {
  uint32_t size, pieces, chunks, parts;
  uint64_t cut, totals, h, g, gt, sums, dB, dC, bytes;
};
Plan plan_of(const uor_trunk_scan_args *s) {
  Plan p{};
  const uint32_t tiles = tiles_of(s->dim), share = s->heads / s->groups;
  const uint64_t n16 = s->state <= 32 ? 32 : s->state <= 64 ? 64 : 128, p16 = s->dim <= 32 ? 32 : 64;
  p.size = piece_rows(s->tokens, s->seqs, s->heads * tiles);
  p.pieces = pieces(s->tokens, s->seqs, p.size);
  p.chunks = pieces(s->tokens, s->seqs, kChunk);
  // Blocks of a group share its heads where the chunks alone do not fill the card.
  const uint64_t blocks = (uint64_t)p.chunks * s->groups;
  p.parts = blocks >= 512 ? 1 : (uint32_t)((511 + blocks) / blocks);
  if (p.parts > share) p.parts = share;
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t begin = at;
    at += (bytes + 255) / 256 * 256;
    return begin;
  };
  const bool cut = p.size < s->tokens;
  p.cut = take(cut ? (uint64_t)p.pieces * s->heads * s->dim * s->state * 4 : 0);
  p.totals = take(cut ? (uint64_t)p.pieces * s->heads * 8 : 0);
  const uint64_t states = (uint64_t)p.chunks * s->heads * tiles * n16 * p16 * 4;
  p.h = take(states), p.g = take(states), p.gt = take(states);
  p.sums = take((uint64_t)p.chunks * s->heads * 3 * 4);
  const uint64_t rows = p.parts > 1 ? (uint64_t)p.parts * s->tokens * s->groups * s->state * 4 : 0;
  p.dB = take(rows), p.dC = take(rows);
  p.bytes = at;
  return p;
}

template <class T, int NT, int PW>
int launch(const Grad &k, uint32_t seqs, hipStream_t stream) {
  const Scan &a = k.s;
  const dim3 block(kThreads), sweep(grid_of(a.pieces, a.heads * a.tiles));
  const dim3 join = join_of(a, seqs);
  if (a.starts) {
    hipLaunchKernelGGL((grad_states<T, NT, PW, false, false>), sweep, block, 0, stream, k);
    hipLaunchKernelGGL(scan_join, join, block, 0, stream, a);
  }
  hipLaunchKernelGGL((grad_states<T, NT, PW, false, true>), sweep, block, 0, stream, k);
  if (a.starts) {
    hipLaunchKernelGGL((grad_states<T, NT, PW, true, false>), sweep, block, 0, stream, k);
    hipLaunchKernelGGL(grad_join, join, block, 0, stream, k);
  }
  hipLaunchKernelGGL((grad_states<T, NT, PW, true, true>), sweep, block, 0, stream, k);
  hipLaunchKernelGGL((grad_rows<T, NT, PW>), dim3(grid_of(k.chunks, a.groups * k.parts)), block, 0, stream, k);
  if (k.parts > 1 && a.rows.tokens) {
    const uint64_t n = (uint64_t)a.rows.tokens * a.groups * a.state;
    hipLaunchKernelGGL(grad_parts<T>, dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, stream, k);
  }
  hipLaunchKernelGGL(grad_sums, dim3(a.heads), dim3(256), 0, stream, k);
  return launched();
}
template <class T, int NT>
int launch(const Grad &k, uint32_t seqs, hipStream_t stream) {
  return k.s.dim <= 32 ? launch<T, NT, 2>(k, seqs, stream) : launch<T, NT, 4>(k, seqs, stream);
}
template <class T>
int launch(const Grad &k, uint32_t seqs, hipStream_t stream) {
  return k.s.state <= 32 ? launch<T, 2>(k, seqs, stream) : k.s.state <= 64 ? launch<T, 4>(k, seqs, stream) : launch<T, 8>(k, seqs, stream);
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
  if (((uint64_t)p.chunks + kXcds) * s->heads * tiles > 0x7fffffffu) return fail(-1, "too many rows and heads for one call");
  const uint32_t size = s->dtype == UOR_TRUNK_BF16 ? 2 : 4;
  char *base = (char *)workspace;
  Grad k{};
  k.s = scan_of(s, p.size);
  if (p.size < s->tokens) {
    k.s.starts = (float *)(base + p.cut);
    k.s.totals = (double *)(base + p.totals);
  }
  k.dy = s->dy, k.dfinal = s->dfinal, k.chunks = p.chunks, k.parts = p.parts;
  k.h = (float *)(base + p.h), k.g = (float *)(base + p.g), k.gt = (float *)(base + p.gt), k.sums = (float *)(base + p.sums);
  k.dBparts = (float *)(base + p.dB), k.dCparts = (float *)(base + p.dC);
  k.dx = s->dx, k.ddt = s->ddt, k.dB = s->dB, k.dC = s->dC, k.dA = s->dA, k.dD = s->dD, k.dbias = s->ddt_bias, k.dinitial = s->dinitial;
  k.dy_wide = aligned16(s->dy, s->y_stride, size) && s->dim * size % 16 == 0;
  k.dx_wide = aligned16(s->dx, 0, size) && s->dim * size % 16 == 0;
  const OnDevice on(s->device);
  if (!on.ok) return fail(-2, "hipSetDevice(%d) failed", s->device);
  return s->dtype == UOR_TRUNK_BF16 ? launch<bf16>(k, s->seqs, (hipStream_t)stream) : launch<float>(k, s->seqs, (hipStream_t)stream);
}
