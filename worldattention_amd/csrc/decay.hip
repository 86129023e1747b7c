// Causal linear attention with a decay for each head (lambda = exp(log_decay)):
//   S_t = lambda S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t.
// No reference counterpart; the non-causal elu(x) + 1 heads are in elu1.hip.
//
// One product form serves the output and all three gradients. With tokens i, j counted from the start
// of a segment and X the state carried into it,
//   y_i = s_intra sum_{j <= i} lambda^(i - j) (a_i . b_j) c_j + s_inter lambda^(i + lag) a_i X
//   out: (a, b, c) = (q, k, v),   X = S,   lag 1;     dq: (dO, v, k), X = S^T, lag 1;
//   dv:  (k, q, dO),  X = Y,      lag 0;              dk: (v, dO, q), X = Y^T, lag 0,
// the last two with time running backwards, Y being the gradient of the state after the segment:
// Y = lambda^n Y' + scale sum_j lambda^(j + 1) q_j dO_j^T, which ends as the initial state's gradient.
//
// Three launches: every segment's own state, the carried states (in place), the rows (64-token chunks in
// sequence, the running state on chip).
//
// The decay's gradient, d/d log(lambda), counts the steps of every path from a token j to a token i. With
// T = dS/d log(lambda), carried as T <- lambda^n (T + n S) + sum_j (n - 1 - j) lambda^(n - 1 - j) k_j v_j^T,
// a segment adds
//   scale sum_{j < i} (i - j) lambda^(i - j) (q_i . k_j)(dO_i . v_j)                    pairs inside it
// + <S, scale sum_i (i + 1) lambda^(i + 1) q_i dO_i^T> + <T, scale sum_i lambda^(i + 1) q_i dO_i^T>,
// and the sequence's end <T, dS>. The sums over i are the segment's own gradient state and its derivative,
// so the state kernels, asked for derivatives, hold all but the pairs.
//
// Roundings. States, derivatives and all sums are fp32 (the decay's gradient is summed in fp64 across
// workgroups). Operands of bf16 products whose results leave in fp32 (states, derivatives) enter cut in three
// exact parts. In the rows of bf16 tensors, whose results leave in bf16, the decayed q.k and the running
// state's weighted operand round to bf16 once; the state itself enters in two parts (2^-17).
#include <algorithm>
#include <cmath>

#include "tile.h"

namespace {

constexpr int kChunk = 64;      // tokens a step of the running state takes
constexpr int kThreads = 256;

// Accumulator register r of lane (l32, g) of a 32 x 32 product is row 8 (r / 4) + 4 g + r % 4, column l32.
__device__ __forceinline__ int acc_row(int r, int g) { return 8 * (r >> 2) + 4 * g + (r & 3); }

struct View {
  const void* p; int64_t sb, st, sh;
};

// Geometry shared by all kernels. Segment c holds n = clamp(length - c seg, 0, seg) tokens.
struct Shape {
  int B, L, H, seg, n_seg;
  const float* log_decay;
  const int32_t* lengths;
};

__device__ __forceinline__ int length_of(const Shape& s, int b) {
  return s.lengths ? max(0, min(s.L, s.lengths[b])) : s.L;
}
__device__ __forceinline__ int tokens_of(const Shape& s, int b, int c) {
  return max(0, min(s.seg, length_of(s, b) - c * s.seg));
}
// log2 of the decay; -inf becomes a number so that 0 steps of it are 0 (lambda^0 = 1)
__device__ __forceinline__ float log2_decay(const Shape& s, int h) {
  const float g = s.log_decay[h];
  return (g < -1e30f ? -1e30f : g) * WA_LOG2E;
}
// lambda^steps: the bare exponential instruction (1 ulp; what would be below 2^-126 is 0)
__device__ __forceinline__ float power(float g2, int steps) { return __builtin_amdgcn_exp2f(g2 * (float)steps); }

// A segment's own state, sum_j w_j b_j c_j^T with w_j = w_scale lambda^steps(j), forwards steps = n - 1 - j,
// backwards (rev) j + 1. With derivatives (derivs not null) also sum_j steps w_j b_j c_j^T: forwards written
// to derivs; backwards the segment's part of the decay's gradient instead, <S, that> + <T, the state>.
struct StateParams {
  Shape s;
  View b, c;
  float* states;        // [B, H, n_seg, D, D]
  float* derivs;        // forwards: [B, H, n_seg + 1, D, D]
  const float* S;       // backwards: the carried states
  const float* T;       //            and their derivatives [B, H, n_seg + 1, D, D]
  double* part;         // [B, H, n_part], the segments' parts first
  int n_part;
  int rev;
  float w_scale;
};

// Rows: one workgroup per (segment, batch and head, job). The jobs of a segment read the same tensors: they are dealt
// eight workgroups apart, to one XCD at about one time, so that its L2 serves the second and third (three gradients
// of 32,760 tokens of 12 x 128: 387 us; one job after the other over all segments 403).
struct Job {
  View a, b, c;
  void* y; int64_t y_sb, y_st, y_sh;
  const float* x;     // carried states
  bool x_trans, rev;
  float s_intra, s_inter;
  float w_scale;                  // of the state's own tokens: s_inter X sums s_intra b c^T
  float unit, in_unit, x_in_unit; // bf16 rows sum y / unit: s_intra and s_inter in it
  float in_log2;                  // log2 of s_intra in the unit, for weights formed as one exponential
};
// time forwards, the carried state holds bare sums: both parts take the scale; backwards it holds scaled ones.
// The unit is the scale, which then stays out of the products. One of 0, or so small or large that its
// reciprocal times a row of the state could leave fp32, cannot be divided by: the unit is then 1 with its sign.
Job rows_job(const View& a, const View& b, const View& c, void* y, int64_t y_sb, int64_t y_st, int64_t y_sh, const float* x, bool x_trans,
             bool rev, float scale) {
  const float s_inter = rev ? 1.f : scale, size = scale < 0.f ? -scale : scale;
  const float unit = size >= 0x1p-32f && size <= 0x1p32f ? scale : scale < 0.f ? -1.f : 1.f;
  return Job{a, b, c, y, y_sb, y_st, y_sh, x, x_trans, rev, scale, s_inter, rev ? scale : 1.f, unit, scale / unit, s_inter / unit, std::log2(scale / unit)};
}
struct RowsParams {
  Shape s;
  Job job[3];
};

// The heads run from the last one, whose keys and values the launch before has left in the last-level cache (a
// training call of that size 823 us against 831).
__device__ __forceinline__ void place_of(const RowsParams& p, int& seg, int& bh, int& job) {
  bh = gridDim.y - 1 - blockIdx.y;
  const int n = p.s.n_seg, jobs = gridDim.x / n, whole = n / 8 * 8;
  int u = blockIdx.x;
  if (u < jobs * whole) {
    job = u % (8 * jobs) / 8;
    seg = u / (8 * jobs) * 8 + u % 8;
  } else {
    u -= jobs * whole;
    job = u / (n - whole);
    seg = whole + u % (n - whole);
  }
}

// Pairs inside the segments, for the decay's gradient.
struct PairsParams {
  Shape s;
  View q, k, v, d;
  double* part;         // [B, H, n_part] from part_at on
  int n_part, part_at;
  float scale;
};

// ---------------------------------------------------------------------------------------------
// fp32 tensors: v_mfma_f32_32x32x2 on tiles staged through registers, four waves. Time runs backwards by
// staging the rows in the other order.
// ---------------------------------------------------------------------------------------------
typedef float f32x8 __attribute__((ext_vector_type(8)));

// 32 x 32 += (32 x 16) (16 x 32): lane (l32, g) holds slots 8 g .. 8 g + 7 of the contraction.
__device__ __forceinline__ f32x16 mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// Row-major LDS tiles of W columns, rows padded by one 16-byte slot.
template <int W> struct Tile {
  static constexpr int kRow = W + 4;
  static __device__ __forceinline__ f32x8 row8(const float* t, int row, int chunk) {
    const f32x4 a = *(const f32x4*)(t + row * kRow + chunk * 8), b = *(const f32x4*)(t + row * kRow + chunk * 8 + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  static __device__ __forceinline__ f32x8 col8(const float* t, int c, int col0, int lane) {
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = t[(16 * c + 8 * (lane >> 5) + e) * kRow + col0 + (lane & 31)];
    return v;
  }
  static __device__ __forceinline__ void put8(float* t, int row, int chunk, const f32x8& v) {
    *(f32x4*)(t + row * kRow + chunk * 8) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)(t + row * kRow + chunk * 8 + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
  static __device__ __forceinline__ void put(float* t, int row, int col, float v) { t[row * kRow + col] = v; }
};

__device__ __forceinline__ f32x8 load8(const float* p) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
  return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// Rows [c0, c0 + 64) of a segment's n, in time's direction, into a tile; rows from n on are zeros.
template <int D>
__device__ __forceinline__ void stage_rows(float* tile, const float* base, int64_t st, int c0, int n, bool rev) {
  constexpr int CPR = D / 8;
#pragma unroll
  for (int i = 0; i < kChunk * CPR / kThreads; ++i) {
    const int u = threadIdx.x + i * kThreads, row = u / CPR, ch = u % CPR, t = c0 + row;
    f32x8 v{};
    if (t < n) v = load8(base + (int64_t)(rev ? n - 1 - t : t) * st + ch * 8);
    Tile<D>::put8(tile, row, ch, v);
  }
}

// Tiles of the D x D state that a wave holds. D = 128: wave w rows 32 w .. + 31 in four column tiles; D = 64:
// tile (w / 2, w % 2).
template <int D> struct Held {
  static constexpr int N = D / 32 * D / 32 / 4;
  static __device__ __forceinline__ int row0(int w) { return 32 * (D == 128 ? w : w >> 1); }
  static __device__ __forceinline__ int col0(int w, int i) { return 32 * (D == 128 ? i : w & 1); }
};

// The state after a chunk of m tokens (and its derivative): acc = lambda^m acc + sum_j w_j b_j c_j^T.
template <int D, bool DERIV>
__device__ __forceinline__ void state_update(f32x16 (&acc)[Held<D>::N], f32x16 (&dacc)[Held<D>::N], const float* tb,
                                             const float* tc, int m, float g2, int ahead, float w_scale, int w, int lane) {
  const int g = lane >> 5;
  const float keep = power(g2, m);
#pragma unroll
  for (int i = 0; i < Held<D>::N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (DERIV) dacc[i][r] = keep * (dacc[i][r] + (float)m * acc[i][r]);
      acc[i][r] *= keep;
    }
#pragma unroll
  for (int jc = 0; jc < kChunk / 16; ++jc) {
    f32x8 bw = Tile<D>::col8(tb, jc, Held<D>::row0(w), lane), bd;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int steps = max(0, m - 1 - (16 * jc + 8 * g + e) + ahead);
      bw[e] *= w_scale * power(g2, steps);
      bd[e] = bw[e] * (float)steps;
    }
#pragma unroll
    for (int i = 0; i < Held<D>::N; ++i) {
      const f32x8 c = Tile<D>::col8(tc, jc, Held<D>::col0(w, i), lane);
      acc[i] = mma(bw, c, acc[i]);
      if (DERIV) dacc[i] = mma(bd, c, dacc[i]);
    }
  }
}

// The sum over a workgroup of NW waves, valid on thread 0. `red`: NW doubles of LDS, free of other use.
template <int NW>
__device__ __forceinline__ double workgroup_sum(double x, double* red) {
  x = wa_wave_sum_d(x);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < NW; ++w) s += red[w];
  return s;
}

template <int D, bool DERIV>
__global__ void __launch_bounds__(kThreads) segment_state_f32_kernel(StateParams p) {
  __shared__ __attribute__((aligned(16))) float tb[kChunk * Tile<D>::kRow];
  __shared__ __attribute__((aligned(16))) float tc[kChunk * Tile<D>::kRow];
  __shared__ double red[4];
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 5, l32 = lane & 31;
  const int n = tokens_of(p.s, b, seg);
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  const float* bb = (const float*)p.b.p + (int64_t)b * p.b.sb + (int64_t)h * p.b.sh + first * p.b.st;
  const float* cb = (const float*)p.c.p + (int64_t)b * p.c.sb + (int64_t)h * p.c.sh + first * p.c.st;
  f32x16 acc[Held<D>::N], dacc[Held<D>::N];
#pragma unroll
  for (int i = 0; i < Held<D>::N; ++i) acc[i] = dacc[i] = f32x16{};
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    stage_rows<D>(tb, bb, p.b.st, c0, n, p.rev);
    stage_rows<D>(tc, cb, p.c.st, c0, n, p.rev);
    __syncthreads();
    state_update<D, DERIV>(acc, dacc, tb, tc, min(kChunk, n - c0), g2, p.rev, p.w_scale, w, lane);
    __syncthreads();
  }
  const int64_t at = ((int64_t)bh * p.s.n_seg + seg) * D * D, dat = ((int64_t)bh * (p.s.n_seg + 1) + seg) * D * D;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < Held<D>::N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int e = (Held<D>::row0(w) + acc_row(r, g)) * D + Held<D>::col0(w, i) + l32;
      p.states[at + e] = acc[i][r];
      if (DERIV && !p.rev) p.derivs[dat + e] = dacc[i][r];
      if (DERIV && p.rev) sum += (double)(p.S[at + e] * dacc[i][r] + p.T[dat + e] * acc[i][r]);
    }
  if (DERIV && p.rev) {
    sum = workgroup_sum<4>(sum, red);
    if (threadIdx.x == 0) p.part[(int64_t)bh * p.n_part + seg] = sum;
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) rows_f32_kernel(RowsParams p) {
  constexpr int YT = D / 64;                // output tiles of a wave: 32 rows x D / 2 columns
  __shared__ __attribute__((aligned(16))) float tb[kChunk * Tile<D>::kRow];
  __shared__ __attribute__((aligned(16))) float tc[kChunk * Tile<D>::kRow];
  __shared__ __attribute__((aligned(16))) float tp[kChunk * Tile<kChunk>::kRow];
  __shared__ __attribute__((aligned(16))) float tx[D * Tile<D>::kRow];
  int seg, bh, job;
  place_of(p, seg, bh, job);
  const Job& jb = p.job[job];
  const int b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, l32 = lane & 31;
  const int rh = w >> 1, ch = w & 1;
  const int n = tokens_of(p.s, b, seg), lag = jb.rev ? 0 : 1;
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  const float* ab = (const float*)jb.a.p + (int64_t)b * jb.a.sb + (int64_t)h * jb.a.sh + first * jb.a.st;
  const float* bb = (const float*)jb.b.p + (int64_t)b * jb.b.sb + (int64_t)h * jb.b.sh + first * jb.b.st;
  const float* cb = (const float*)jb.c.p + (int64_t)b * jb.c.sb + (int64_t)h * jb.c.sh + first * jb.c.st;
  float* yb = (float*)jb.y + (int64_t)b * jb.y_sb + (int64_t)h * jb.y_sh + first * jb.y_st;

  // tokens past the sequence's end
  const int rows = (int)min((int64_t)p.s.seg, p.s.L - first);
  for (int u = tid; u < (rows - n) * (D / 4); u += kThreads)
    *(f32x4*)(yb + (int64_t)(n + u / (D / 4)) * jb.y_st + (u % (D / 4)) * 4) = f32x4{0.f, 0.f, 0.f, 0.f};
  if (n == 0) return;

  const float* x0 = jb.x + ((int64_t)bh * p.s.n_seg + seg) * D * D;
  f32x16 acc[Held<D>::N], none[Held<D>::N];
#pragma unroll
  for (int i = 0; i < Held<D>::N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = Held<D>::row0(w) + acc_row(r, g), col = Held<D>::col0(w, i) + l32;
      acc[i][r] = jb.x_trans ? x0[col * D + row] : x0[row * D + col];
    }

  for (int c0 = 0; c0 < n; c0 += kChunk) {
    stage_rows<D>(tb, bb, jb.b.st, c0, n, jb.rev);
    stage_rows<D>(tc, cb, jb.c.st, c0, n, jb.rev);
#pragma unroll
    for (int i = 0; i < Held<D>::N; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) Tile<D>::put(tx, Held<D>::row0(w) + acc_row(r, g), Held<D>::col0(w, i) + l32, acc[i][r]);
    f32x8 a[D / 16];
    const int ta = c0 + 32 * rh + l32;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      a[k] = f32x8{};
      if (ta < n) a[k] = load8(ab + (int64_t)(jb.rev ? n - 1 - ta : ta) * jb.a.st + 16 * k + 8 * g);
    }
    __syncthreads();
    // decayed products of this wave's 32 x 32 rows and columns of the chunk
    f32x16 s{};
    if (ch <= rh) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) s = mma(a[k], Tile<D>::row8(tb, 32 * ch + l32, 2 * k + g), s);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = 32 * rh + acc_row(r, g), j = 32 * ch + l32;
      Tile<kChunk>::put(tp, i, j, j <= i ? s[r] * power(g2, i - j) : 0.f);
    }
    __syncthreads();
#pragma unroll
    for (int yt = 0; yt < YT; ++yt) {
      const int col0 = ch * (D / 2) + 32 * yt;
      f32x16 intra{}, inter{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) inter = mma(a[k], Tile<D>::col8(tx, k, col0, lane), inter);
#pragma unroll
      for (int jc = 0; jc < kChunk / 16; ++jc)
        intra = mma(Tile<kChunk>::row8(tp, 32 * rh + l32, 2 * jc + g), Tile<D>::col8(tc, jc, col0, lane), intra);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 32 * rh + acc_row(r, g), t = c0 + i;
        if (t < n)
          yb[(int64_t)(jb.rev ? n - 1 - t : t) * jb.y_st + col0 + l32] = jb.s_intra * intra[r] + jb.s_inter * power(g2, i + lag) * inter[r];
      }
    }
    state_update<D, false>(acc, none, tb, tc, min(kChunk, n - c0), g2, 1 - lag, jb.w_scale, w, lane);
    __syncthreads();
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) pairs_f32_kernel(PairsParams p) {
  __shared__ __attribute__((aligned(16))) float tk[kChunk * Tile<D>::kRow];
  __shared__ __attribute__((aligned(16))) float tv[kChunk * Tile<D>::kRow];
  __shared__ double red[4];
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 5, l32 = lane & 31, rh = w >> 1, ch = w & 1;
  const int n = tokens_of(p.s, b, seg);
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  const float* qb = (const float*)p.q.p + (int64_t)b * p.q.sb + (int64_t)h * p.q.sh + first * p.q.st;
  const float* kb = (const float*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh + first * p.k.st;
  const float* vb = (const float*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh + first * p.v.st;
  const float* db = (const float*)p.d.p + (int64_t)b * p.d.sb + (int64_t)h * p.d.sh + first * p.d.st;
  double sum = 0.0;
  for (int i0 = 0; i0 < n; i0 += kChunk) {
    f32x8 aq[D / 16], ad[D / 16];
    const int ta = i0 + 32 * rh + l32;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      aq[k] = ad[k] = f32x8{};
      if (ta < n) {
        aq[k] = load8(qb + (int64_t)ta * p.q.st + 16 * k + 8 * g);
        ad[k] = load8(db + (int64_t)ta * p.d.st + 16 * k + 8 * g);
      }
    }
    for (int j0 = 0; j0 <= i0; j0 += kChunk) {
      __syncthreads();
      stage_rows<D>(tk, kb, p.k.st, j0, n, false);
      stage_rows<D>(tv, vb, p.v.st, j0, n, false);
      __syncthreads();
      f32x16 a{}, e{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        a = mma(aq[k], Tile<D>::row8(tk, 32 * ch + l32, 2 * k + g), a);
        e = mma(ad[k], Tile<D>::row8(tv, 32 * ch + l32, 2 * k + g), e);
      }
      float part = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int steps = i0 + 32 * rh + acc_row(r, g) - (j0 + 32 * ch + l32);
        if (steps > 0) part += (float)steps * power(g2, steps) * (a[r] * e[r]);
      }
      sum += (double)part;
    }
  }
  sum = workgroup_sum<4>(sum * (double)p.scale, red);
  if (threadIdx.x == 0) p.part[(int64_t)bh * p.n_part + p.part_at + seg] = sum;
}

// ---------------------------------------------------------------------------------------------
// bf16 forms. Tiles of 64 tokens stream into a ring of LDS stages by direct loads, two steps ahead; rows
// past the segment's last token read as zeros. Time runs backwards by taking the chunks in the other
// order, with weights and masks mirrored inside a chunk; memory order inside a tile stays.
//
// All products run transposed so that operands stay where they are. A column permutation of the
// transpose reads makes it fit: the accumulator's row (register r, lane group g) is 8 (r / 4) + 4 g + r % 4;
// feeding rows in the order pi (bits 2 and 3 swapped) leaves lane group g holding, in registers
// 8 h .. 8 h + 7, rows 16 h + 8 g .. + 7: eight consecutive channels, which is both a 16-byte store and
// the natural operand order of the next product.
// ---------------------------------------------------------------------------------------------
// A lane's byte offsets into swizzled tiles of D columns. The swizzle takes no bit of a row above the
// fourth and turns a column step of 16 (a contraction step) or 32 (a tile) into one exclusive or, so four
// offsets serve every read.
template <int D>
struct TileReads {
  int row, rowpi;    // 128-bit reads: row l32 (pi(l32)), chunk g
  int tr[2];         // transpose reads in order pi: tokens of the first 16, columns of the first 32
  __device__ __forceinline__ void init(int lane) {
    const int g = lane >> 5, l32 = lane & 31, lp = (l32 & 0x13) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
    row = (l32 * D + ((g ^ dual_swizzle<D>(l32)) * 8)) * 2;
    rowpi = (lp * D + ((g ^ dual_swizzle<D>(lp)) * 8)) * 2;
    const int G = lane >> 4, r = (lane & 15) >> 2, q = ((lane & 1) << 1) | ((lane >> 1) & 1);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int t = 4 * (G >> 1) + 8 * hf + r, col = 16 * (G & 1) + 4 * q;
      tr[hf] = (t * D + (((col >> 3) ^ dual_swizzle<D>(t)) * 8) + (col & 7)) * 2;
    }
  }
  // Hides from the compiler that the offsets stay the same from step to step: the sums it would keep of
  // them take the registers that hold operands ahead of their products.
  __device__ __forceinline__ void renew_rows() { asm volatile("" : "+v"(row)); }
  __device__ __forceinline__ void renew_cols() { asm volatile("" : "+v"(tr[0]), "+v"(tr[1])); }
  __device__ __forceinline__ void renew() {
    asm volatile("" : "+v"(rowpi));
    renew_rows();
    renew_cols();
  }
  // rows 32 tile + l32, channels 16 k + 8 g .. + 7
  __device__ __forceinline__ bf16x8 rows(const bf16_t* t, int tile, int k) const {
    return *(const bf16x8*)((const char*)t + (row ^ (k << 5)) + tile * (32 * D * 2));
  }
  __device__ __forceinline__ bf16x8 rows_pi(const bf16_t* t, int tile, int k) const {
    return *(const bf16x8*)((const char*)t + (rowpi ^ (k << 5)) + tile * (32 * D * 2));
  }
  // tile_tr8 of tokens 16 c .. with lane l32 at column 32 tile + pi(l32)
  __device__ __forceinline__ bf16x8 cols_pi(const bf16_t* t, int c, int tile) const {
    bf16x8 a;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const wa_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          WA_LDS_S16X4((const char*)t + (tr[hf] ^ (tile << 6)) + c * (16 * D * 2)));
      const bf16x4 b = __builtin_bit_cast(bf16x4, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * hf + e] = b[e];
    }
    return a;
  }
};
__device__ __forceinline__ int pi32(int x) { return (x & 0x13) | ((x & 4) << 1) | ((x & 8) >> 1); }

// TileStream (tile.h) over one segment, with the descriptor cut to the chunk's rows: any distance between the
// segment's first and last token, D (so that the cut falls between rows) to kMaxTokenStride elements between two.
constexpr int64_t kMaxTokenStride = (int64_t)1 << 23;
template <int D, int NW>
struct ChunkStream {
  static constexpr int NI = TileStream<D, NW>::NI, RPI = TileStream<D, NW>::RPI;
  static_assert(NW * RPI % 16 == 0, "the swizzle repeats every 16 rows, so one lane offset serves all instructions");
  const bf16_t* base;
  int64_t st;
  int off;
  __device__ __forceinline__ void init(const View& x, int b, int h, int64_t first, int w, int lane) {
    base = (const bf16_t*)x.p + (int64_t)b * x.sb + (int64_t)h * x.sh + first * x.st;
    st = x.st;
    const int row = w * RPI + lane / (D / 8), pos = lane % (D / 8);
    off = (row * (int)st + (pos ^ dual_swizzle<D>(row)) * 8) * 2;
  }
  // rows row0 .. row0 + rows - 1 (at most 64) into `lds`, zeros behind them
  __device__ __forceinline__ void issue(bf16_t* lds, int row0, int rows, int w) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int skip = i * NW * RPI;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(base + (int64_t)(row0 + skip) * st), (short)0, rows > skip ? ((rows - skip - 1) * (int)st + D) * 2 : 0, WA_BUF_DWORD3);
      lds_dma16(rs, lds + (i * NW + w) * RPI * D, off);
    }
  }
};

__device__ __forceinline__ bf16x8 pack8(const f32x16& a, int h) {
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (bf16_t)a[8 * h + e];
  return v;
}

// x = hi + mid + lo exactly: three bf16 values cut off a float's 24 bits.
__device__ __forceinline__ void cut3(const float (&x)[8], bf16x8& hi, bf16x8& mid, bf16x8& lo) {
  u32x4 h, m, l;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t hb[2], mb[2], lb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float v = x[2 * q + i];
      hb[i] = __float_as_uint(v);
      const float r = v - __uint_as_float(hb[i] & 0xffff0000u);
      mb[i] = __float_as_uint(r);
      lb[i] = __float_as_uint(r - __uint_as_float(mb[i] & 0xffff0000u));
    }
    h[q] = __builtin_amdgcn_perm(hb[1], hb[0], 0x07060302);   // the high halves of two floats side by side
    m[q] = __builtin_amdgcn_perm(mb[1], mb[0], 0x07060302);
    l[q] = __builtin_amdgcn_perm(lb[1], lb[0], 0x07060302);
  }
  hi = __builtin_bit_cast(bf16x8, h);
  mid = __builtin_bit_cast(bf16x8, m);
  lo = __builtin_bit_cast(bf16x8, l);
}

// The 8 weights of a fragment's tokens (accumulator order).
__device__ __forceinline__ void load_weights(const float* wt, int c, int g, float (&w)[8]) {
  const f32x4 a = *(const f32x4*)(wt + 16 * c + 4 * g), b = *(const f32x4*)(wt + 16 * c + 8 + 4 * g);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = a[e];
    w[e + 4] = b[e];
  }
}

// A segment's own state. Wave (ch, half) of D / 16 waves: columns 32 ch .. + 31 over all rows, from half of each
// chunk's tokens (the two halves meet in LDS at the end): every weighted operand is then cut once a workgroup.
// It enters in three parts, so the state carries no rounding but its fp32 sums'. The state decays once in two
// chunks, whose tokens' weights run to the end of the two. 32,760 tokens of 12 x 128: 51 us in 21 segments, 41 of
// them what its 200 MB take at a copy's rate; with derivatives in 64 segments 100, and 112-117 in the backward pass,
// which multiplies them with the forward's. A wave a half of the rows, cutting twice, decaying every chunk: 99
// without derivatives.
constexpr int kSpan = 2 * kChunk;

template <int D, bool DERIV>
__global__ void __launch_bounds__(64 * (D / 16)) segment_state_bf16_kernel(StateParams p) {
  constexpr int NW = D / 16, CT = D / 32, STAGES = 3, NI = ChunkStream<D, NW>::NI;
  __shared__ __attribute__((aligned(1024))) bf16_t tiles[2 * STAGES * kChunk * D];
  __shared__ __attribute__((aligned(16))) float wt[2][kSpan];
  __shared__ double red[NW];
  static_assert(sizeof(float) * D * D <= sizeof(tiles), "one half's state passes through the stages");
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  const int ch = w % CT, half = w / CT;
  const int n = tokens_of(p.s, b, seg), chunks = (n + kChunk - 1) / kChunk, spans = (n + kSpan - 1) / kSpan;
  const int tail = n - (spans - 1) * kSpan;   // tokens of the span cut off at the end
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  ChunkStream<D, NW> sb, sc;
  sb.init(p.b, b, h, first, w, lane);
  sc.init(p.c, b, h, first, w, lane);
  auto stage_b = [&](int it) { return tiles + (it % STAGES) * 2 * kChunk * D; };
  auto stage_c = [&](int it) { return tiles + (it % STAGES) * 2 * kChunk * D + kChunk * D; };
  // step `it` takes chunk `it`, backwards the spans from the last one with their chunks in order
  auto chunk_of = [&](int it) {
    if (!p.rev) return it;
    const int of_last = chunks - 2 * (spans - 1);
    return it < of_last ? 2 * (spans - 1) + it : 2 * (spans - 2 - (it - of_last) / 2) + (it - of_last) % 2;
  };
  auto issue = [&](int it) {
    const int row0 = chunk_of(it) * kChunk, rows = min(kChunk, n - row0);
    sb.issue(stage_b(it), row0, rows, w);
    sc.issue(stage_c(it), row0, rows, w);
  };
  TileReads<D> rd;
  rd.init(lane);
  f32x16 acc[CT], dacc[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) acc[i] = dacc[i] = f32x16{};
  if (tid < kSpan) {   // weights of whole spans' tokens, and of the one cut off
    wt[0][tid] = p.w_scale * power(g2, p.rev ? tid + 1 : kSpan - 1 - tid);
    wt[1][tid] = p.w_scale * power(g2, p.rev ? tid + 1 : max(0, tail - 1 - tid));
  }
  if (chunks > 0) issue(0);
  if (chunks > 1) issue(1);
  for (int it = 0; it < chunks; ++it) {
    // tile it has landed (it + 1 may stream) and every wave is past tile it - 1, whose stage is refilled
    if (it + 1 < chunks) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NI) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (it + 2 < chunks) issue(it + 2);
    const int c = chunk_of(it), at = c % 2 * kChunk;   // the chunk's place in its span
    const bool cut = c / 2 == spans - 1;
    const int m = cut ? tail : kSpan;
    if (c % 2 == 0) {
      const float keep = power(g2, m);
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (DERIV) dacc[i][r] = keep * (dacc[i][r] + (float)m * acc[i][r]);
          acc[i][r] *= keep;
        }
    }
    const bf16_t* B = stage_b(it);
    const bf16_t* C = stage_c(it);
    rd.renew_cols();
    bf16x8 cv[2], bv[2][CT];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      cv[x] = rd.cols_pi(C, 2 * half + x, ch);
#pragma unroll
      for (int i = 0; i < CT; ++i) bv[x][i] = rd.cols_pi(B, 2 * half + x, i);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float wv[8];
      load_weights(wt[cut ? 1 : 0] + at, 2 * half + x, g, wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] *= (float)cv[x][e];
      bf16x8 hi, mid, lo;
      cut3(wv, hi, mid, lo);
#pragma unroll
      for (int i = 0; i < CT; ++i) acc[i] = wa_mfma32(bv[x][i], lo, acc[i]);
#pragma unroll
      for (int i = 0; i < CT; ++i) acc[i] = wa_mfma32(bv[x][i], mid, acc[i]);
#pragma unroll
      for (int i = 0; i < CT; ++i) acc[i] = wa_mfma32(bv[x][i], hi, acc[i]);
      if (DERIV) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = at + 16 * (2 * half + x) + 4 * g + 8 * (e >> 2) + (e & 3);
          wv[e] *= (float)(p.rev ? j + 1 : max(0, m - 1 - j));
        }
        cut3(wv, hi, mid, lo);
#pragma unroll
        for (int i = 0; i < CT; ++i) dacc[i] = wa_mfma32(bv[x][i], lo, dacc[i]);
#pragma unroll
        for (int i = 0; i < CT; ++i) dacc[i] = wa_mfma32(bv[x][i], mid, dacc[i]);
#pragma unroll
        for (int i = 0; i < CT; ++i) dacc[i] = wa_mfma32(bv[x][i], hi, dacc[i]);
      }
    }
  }
  // The halves meet: the first takes the states, the second the derivatives.
  float* meet = (float*)tiles;
  auto join = [&](f32x16 (&x)[CT], int to) {
    __syncthreads();
    if (half != to) {
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) meet[((ch * CT + i) * 16 + r) * 64 + lane] = x[i][r];
    }
    __syncthreads();
    if (half == to) {
#pragma unroll
      for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] += meet[((ch * CT + i) * 16 + r) * 64 + lane];
    }
  };
  join(acc, 0);
  if (DERIV) join(dacc, 1);
  const int64_t at = ((int64_t)bh * p.s.n_seg + seg) * D * D, dat = ((int64_t)bh * (p.s.n_seg + 1) + seg) * D * D;
  double sum = 0.0;
  auto element = [&](int i, int r) { return (32 * i + 16 * (r >> 3) + 8 * g + (r & 7)) * D + 32 * ch + pi32(l32); };
  auto write = [&](const f32x16 (&x)[CT], float* out) {
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[element(i, r)] = x[i][r];
  };
  auto dot = [&](const f32x16 (&x)[CT], const float* other) {
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      float o[16], part = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) o[r] = other[element(i, r)];
#pragma unroll
      for (int r = 0; r < 16; ++r) part += o[r] * x[i][r];
      sum += (double)part;
    }
  };
  if (half == 0) {
    write(acc, p.states + at);
    if (DERIV && p.rev) dot(acc, p.T + dat);
  } else if (DERIV) {
    if (p.rev) dot(dacc, p.S + at);
    else write(dacc, p.derivs + dat);
  }
  if (DERIV && p.rev) {
    sum = workgroup_sum<NW>(sum, red);
    if (tid == 0) p.part[(int64_t)bh * p.n_part + seg] = sum;
  }
}

// Rows, in units of 32 tokens a wave (256 for D = 128, 128 for D = 64). A wave holds one 32-row tile of the
// unit and, for the running state, two (one) of its D x D tiles. Per unit, with P^T = B A^T decayed and masked,
//   Y^T = s_inter lambda^.. X^T A^T + s_intra C^T P^T,    X = lambda^m X + (weighted B)^T C:
// X^T is read from LDS (two parts, written once a unit), P^T's accumulators are the next product's operand in
// place, and the keys and values of the unit stream through a ring of two 64-token stages that serve the rows
// behind them and the state at once. Work a unit, not a chunk, pays for the state: with a state read and
// rewritten every 64 tokens (two waves a tile, no LDS copy) the vector instructions were 2,600 a wave and unit
// and the launch took 235 us at 32,760 tokens of 12 x 128; it takes 127-131, the three gradients in one launch
// 370-387. Bound by its instructions: the ring and X^T fill a CU's LDS, so one workgroup runs at a time.
template <int D>
__global__ void __launch_bounds__(64 * (D / 16)) rows_bf16_kernel(RowsParams p) {
  constexpr int NW = D / 16, CT = D / 32, KS = D / 16, STAGES = 2, UNIT = 32 * NW;
  constexpr int XT = CT * CT / NW;          // state tiles of a wave: row tile w % CT, columns from (w / CT) XT on
  __shared__ __attribute__((aligned(1024))) bf16_t tb[STAGES][kChunk * D];
  __shared__ __attribute__((aligned(1024))) bf16_t tc[STAGES][kChunk * D];
  __shared__ __attribute__((aligned(1024))) bf16_t xh[D * D], xl[D * D];   // X^T: row e, column d
  __shared__ __attribute__((aligned(16))) float wt[UNIT], edge[32];
  int seg, bh, job;
  place_of(p, seg, bh, job);
  const Job& jb = p.job[job];
  const int b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  const int xd = w % CT, xe = w / CT * XT;
  const int rt = w < NW / 2 ? w : 3 * NW / 2 - 1 - w;   // row tile: the two waves of a SIMD share the causal work evenly
  const bool rev = jb.rev;
  const int n = tokens_of(p.s, b, seg);
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  bf16_t* yb = (bf16_t*)jb.y + (int64_t)b * jb.y_sb + (int64_t)h * jb.y_sh + first * jb.y_st;

  // tokens past the sequence's end
  const int rows = (int)min((int64_t)p.s.seg, p.s.L - first);
  for (int u = tid; u < (rows - n) * (D / 8); u += 64 * NW)
    *(u32x4*)(yb + (int64_t)(n + u / (D / 8)) * jb.y_st + (u % (D / 8)) * 8) = u32x4{0, 0, 0, 0};
  if (n == 0) return;

  const int units = (n + UNIT - 1) / UNIT, chunks = (n + kChunk - 1) / kChunk;
  constexpr int CPU = UNIT / kChunk;        // chunks of a whole unit
  ChunkStream<D, NW> sb, sc;
  sb.init(jb.b, b, h, first, w, lane);
  sc.init(jb.c, b, h, first, w, lane);
  // chunk `c` of the segment into the stage of the step that takes it
  auto issue = [&](int c, int step) {
    const int m = min(kChunk, n - c * kChunk);
    sb.issue(tb[step % STAGES], c * kChunk, m, w);
    sc.issue(tc[step % STAGES], c * kChunk, m, w);
  };
  issue(rev ? (units - 1) * CPU : 0, 0);

  // X[d][e] of lane (l32, g): e = 32 (xe + i) + pi(l32), register 8 hf + x: d = 32 xd + 16 hf + 8 g + x
  f32x16 X[XT];
  const float* x0 = jb.x + ((int64_t)bh * p.s.n_seg + seg) * D * D;
#pragma unroll
  for (int i = 0; i < XT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * xd + 16 * (r >> 3) + 8 * g + (r & 7), e = 32 * (xe + i) + pi32(l32);
      X[i][r] = jb.x_trans ? x0[e * D + d] : x0[d * D + e];
    }
  auto put_state = [&](int row, int half) {   // the lane's pi(l32) and g
#pragma unroll
    for (int i = 0; i < XT; ++i)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        bf16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = X[i][8 * hf + e];
          hi[e] = (bf16_t)x;
          lo[e] = (bf16_t)(x - (float)hi[e]);
        }
        tile_put8<D>(xh, 32 * (xe + i) + row, 4 * xd + 2 * hf + half, hi);
        tile_put8<D>(xl, 32 * (xe + i) + row, 4 * xd + 2 * hf + half, lo);
      }
  };
  put_state(pi32(l32), g);
  // weights of a unit's tokens in the state after it (backwards, before it): whole units
  if (tid < UNIT) wt[tid] = jb.w_scale * power(g2, rev ? tid + 1 : UNIT - 1 - tid);
  // decay between the tokens of a tile and its edge on the rows' side
  if (tid < 32) edge[tid] = jb.in_unit * power(g2, rev ? tid : 31 - tid);

  float in_log2 = jb.in_log2;     // a register: read where it is used, it would come from memory there
  asm volatile("" : "+s"(in_log2));
  // One step a chunk: the unit's first one starts its rows, its last one stores them and passes the state on.
  bf16x8 a[KS];
  auto load_rows = [&](int t, int half) {     // the operands of row t of the segment
    const bf16_t* ap = (const bf16_t*)jb.a.p + (int64_t)b * jb.a.sb + (int64_t)h * jb.a.sh + (first + t) * jb.a.st + 8 * half;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      a[k] = bf16x8{};
      if (t < n) a[k] = *(const bf16x8*)(ap + 16 * k);
    }
  };
  int u0 = rev ? (units - 1) * UNIT : 0, c = 0;   // the unit's first token, the chunk in it
  load_rows(u0 + 32 * rt + l32, g);
  f32x16 y[CT];
  TileReads<D> rd;
  rd.init(lane);
  for (int step = 0; step < chunks; ++step) {
    // this step's tiles have landed and every wave is past the step before, whose stage is refilled
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // the rows' operands have landed with them: named here, so that no wait for them follows the loads below
#pragma unroll
    for (int k = 0; k < KS; ++k) asm volatile("" : "+v"(a[k]));
    const int m = min(UNIT, n - u0), next_u0 = rev ? u0 - UNIT : u0 + UNIT;
    const bool last = (c + 1) * kChunk >= m, more = rev ? u0 > 0 : u0 + UNIT < n;   // of the unit; units behind it
    if (!last) issue(u0 / kChunk + c + 1, step + 1);
    else if (more) issue(next_u0 / kChunk, step + 1);
    const bf16_t* B = tb[step % STAGES];
    const bf16_t* C = tc[step % STAGES];
    if (c == 0) {
#pragma unroll
      for (int et = 0; et < CT; ++et) y[et] = f32x16{};
    }
    const bool any = 32 * rt < m;
    // tiles of the chunk that the rows see: [lo, hi) of 0, 1 (the diagonal one among them)
    const int at = rt - 2 * c, lo = rev ? max(0, at) : 0, hi = rev ? 2 : min(2, at + 1);
    const bool sees = any && lo < hi;
    constexpr int Q = 4;      // operands are read four at a time, while the four products before them run
    bf16x8 f[2][Q];
    rd.renew();
    int ln = lane;     // renewed likewise, for what is derived from it
    asm volatile("" : "+v"(ln));
    const int lg = ln >> 5, lr = ln & 31;
    if (c == 0) {
      // the carried state's part
      const float fs = jb.x_in_unit * power(g2, rev ? max(0, m - 1 - (32 * rt + lr)) : 32 * rt + lr + 1);
      if (any) {
#pragma unroll
        for (int x = 0; x < Q; ++x) f[0][x] = rd.rows_pi(xl, 0, x);
        constexpr int PER = 2 * KS / Q;       // groups of an output tile: the low parts, then the high ones
        f32x16 s;
#pragma unroll
        for (int q = 0; q < CT * PER; ++q) {
          if (q + 1 < CT * PER) {
            const int nq = q + 1, k0 = nq % PER * Q;
#pragma unroll
            for (int x = 0; x < Q; ++x)
              f[nq % 2][x] = rd.rows_pi(k0 < KS ? xl : xh, nq / PER, (k0 + x) % KS);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (q % PER == 0) s = f32x16{};
#pragma unroll
          for (int x = 0; x < Q; ++x) s = wa_mfma32(f[q % 2][x], a[(q % PER * Q + x) % KS], s);
          if (q % PER == PER - 1) {
#pragma unroll
            for (int r = 0; r < 16; ++r) y[q / PER][r] += s[r] * fs;
          }
        }
      }
    }
    // decayed products with the chunk's two tiles of tokens, zero where the rows do not see them
    bf16x8 pr[4];
    if (sees) {
      f32x16 s[2] = {};
#pragma unroll
      for (int x = 0; x < Q; ++x) f[0][x] = rd.rows(B, 0, x);
#pragma unroll
      for (int q = 0; q < 2 * KS / Q; ++q) {
        if (q + 1 < 2 * KS / Q) {
#pragma unroll
          for (int x = 0; x < Q; ++x)
            f[(q + 1) % 2][x] = rd.rows(B, (q + 1) * Q / KS, (Q * (q + 1) + x) % KS);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < Q; ++x) s[q * Q / KS] = wa_mfma32(f[q % 2][x], a[(Q * q + x) % KS], s[q * Q / KS]);
      }
#pragma unroll
      for (int jh = 0; jh < 2; ++jh) {
        if (jh == at) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int steps = rev ? acc_row(r, lg) - lr : lr - acc_row(r, lg);
            s[jh][r] = steps >= 0 ? s[jh][r] * __builtin_amdgcn_exp2f(__builtin_fmaf(g2, (float)steps, in_log2)) : 0.f;
          }
        } else if (jh >= lo && jh < hi) {
          const float fj = power(g2, rev ? 32 * (jh - at) - lr : 32 * (at - jh) + lr - 31);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 e = *(const f32x4*)(edge + 8 * r + 4 * lg);
#pragma unroll
            for (int x = 0; x < 4; ++x) s[jh][4 * r + x] *= e[x] * fj;
          }
        } else {
          s[jh] = f32x16{};
        }
        pr[2 * jh] = pack8(s[jh], 0);
        pr[2 * jh + 1] = pack8(s[jh], 1);
      }
    }
    // weighted keys of this wave's state rows (past the last unit the state is not used again)
    if (c == 0) {
      const float keep = power(g2, m);
#pragma unroll
      for (int i = 0; i < XT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) X[i][r] *= keep;
    }
    bf16x8 bw[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) bw[q] = rd.cols_pi(B, q, xd);
#pragma unroll
    for (int q = 0; q < Q; ++q) f[0][q] = rd.cols_pi(C, q, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float wv[8];
      load_weights(wt + c * kChunk, q, lg, wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) bw[q][e] = (bf16_t)(wv[e] * (float)bw[q][e]);
    }
#pragma unroll
    for (int et = 0; et < CT; ++et) {
      if (et + 1 < CT) {
#pragma unroll
        for (int q = 0; q < Q; ++q) f[(et + 1) % 2][q] = rd.cols_pi(C, q, et + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (sees) {
#pragma unroll
        for (int q = 0; q < 4; ++q) y[et] = wa_mfma32(f[et % 2][q], pr[q], y[et]);
      }
      if (et / XT == xe / XT) {
#pragma unroll
        for (int q = 0; q < 4; ++q) X[et % XT] = wa_mfma32(bw[q], f[et % 2][q], X[et % XT]);
      }
    }
    ++c;
    if (!last) continue;
    const int lp = pi32(lr);
    const int t = u0 + 32 * rt + lr;
    if (t < n) {
      bf16_t* at = yb + (int64_t)t * jb.y_st + 8 * lg;
#pragma unroll
      for (int et = 0; et < CT; ++et)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          bf16x8 o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = (bf16_t)(jb.unit * y[et][8 * hf + e]);
          *(bf16x8*)(at + 32 * et + 16 * hf) = o;
        }
    }
    if (more) {
      if (c == 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // every wave has read the old state
      put_state(lp, lg);
      u0 = next_u0;
      c = 0;
      load_rows(u0 + 32 * rt + lr, lg);
    }
  }
}

// Pairs: a workgroup takes 256 rows i of a segment, its four waves two 32-row tiles each (w and 7 - w, which
// share the causal work evenly), whose queries and output gradients stay in registers as operands; the
// segment's keys and values up to the rows pass through a ring of two LDS stages, each operand read
// serving both tiles. 32,760 tokens of 12 x 128 in 64 segments: 111-117 us, 0.45 PFLOP/s of the products' causal
// half; bound by the instructions that decay, mask and multiply the two score tiles. Tiles before the diagonal
// separate: with e the tile's last token, (i - j) lambda^(i - j) = lambda^(i - e) [(i - e) + (e - j)] lambda^(e - j),
// no power above 1.
constexpr int kPairRows = 256;

template <int D>
__global__ void __launch_bounds__(256, 2) pairs_bf16_kernel(PairsParams p) {
  constexpr int NW = 4, KS = D / 16, STAGES = 2, Q = 2, PER = KS / Q;
  __shared__ __attribute__((aligned(1024))) bf16_t tk[STAGES][kChunk * D];
  __shared__ __attribute__((aligned(1024))) bf16_t tv[STAGES][kChunk * D];
  __shared__ __attribute__((aligned(16))) float edge[2][32];   // lambda^(e - j) of a tile's tokens, and (e - j) times it
  __shared__ double red[NW];
  const int groups = (p.s.seg + kPairRows - 1) / kPairRows;
  // the groups with the most keys first, so that the short ones fill the end of the launch
  const int seg = blockIdx.x / groups, ig = groups - 1 - (int)blockIdx.x % groups, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  const int n = tokens_of(p.s, b, seg), i0 = ig * kPairRows;
  double* out = p.part + (int64_t)bh * p.n_part + p.part_at + blockIdx.x;
  if (i0 >= n) {
    if (tid == 0) *out = 0.0;
    return;
  }
  const int row0[2] = {i0 + 32 * w, i0 + 32 * (7 - w)};
  const int chunks = (min(n, i0 + kPairRows) + kChunk - 1) / kChunk;
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  ChunkStream<D, NW> sk, sv;
  sk.init(p.k, b, h, first, w, lane);
  sv.init(p.v, b, h, first, w, lane);
  auto issue = [&](int it) {
    sk.issue(tk[it % STAGES], it * kChunk, min(kChunk, n - it * kChunk), w);
    sv.issue(tv[it % STAGES], it * kChunk, min(kChunk, n - it * kChunk), w);
  };
  TileReads<D> rd;
  rd.init(lane);
  // The rows' operands come through the stages too (the four hold 256 rows), in whole lines: read straight
  // into registers, 32 bytes of 32 rows at a time, they took 14 us of a workgroup's 60 (260 us against 231 in 21
  // segments of the size above).
  bf16x8 q[2][KS], d[2][KS];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    ChunkStream<D, NW> sr;
    sr.init(x ? p.d : p.q, b, h, first, w, lane);
#pragma unroll
    for (int y = 0; y < 4; ++y) sr.issue(y < 2 ? tk[y] : tv[y - 2], i0 + kChunk * y, min(kChunk, n - (i0 + kChunk * y)), w);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int rt = y ? 7 - w : w;
      const bf16_t* T = rt < 4 ? tk[rt / 2] : tv[rt / 2 - 2];
#pragma unroll
      for (int k = 0; k < KS; ++k) (x ? d : q)[y][k] = rd.rows(T, rt % 2, k);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
  if (tid < 32) {
    edge[0][tid] = power(g2, 31 - tid);
    edge[1][tid] = (float)(31 - tid) * edge[0][tid];
  }
  issue(0);
  double sum = 0.0;
  // One tile of 32 tokens from jt on against both row tiles (the upper one may not see it).
  auto tile = [&](const bf16_t* K, const bf16_t* V, int jh, int jt) {
    bf16x8 f[2][Q];
    f32x16 s[2] = {}, t[2] = {};
#pragma unroll
    for (int x = 0; x < Q; ++x) f[0][x] = rd.rows(K, jh, x);
#pragma unroll
    for (int u = 0; u < 2 * PER; ++u) {   // keys, then values: two operands read behind the products before them
      if (u + 1 < 2 * PER) {
#pragma unroll
        for (int x = 0; x < Q; ++x) f[(u + 1) % 2][x] = rd.rows((u + 1) / PER ? V : K, jh, (u + 1) % PER * Q + x);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < Q; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (u / PER) t[y] = wa_mfma32(f[u % 2][x], d[y][u % PER * Q + x], t[y]);
          else s[y] = wa_mfma32(f[u % 2][x], q[y][u % PER * Q + x], s[y]);
        }
    }
    int ln = lane;     // the lane renewed, so that the powers below are not kept in registers
    asm volatile("" : "+v"(ln));
    const int lg = ln >> 5, lr = ln & 31;
    float u[2] = {0.f, 0.f}, v[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const f32x4 e0 = *(const f32x4*)(edge[0] + 8 * r + 4 * lg), e1 = *(const f32x4*)(edge[1] + 8 * r + 4 * lg);
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float x = s[y][4 * r + z] * t[y][4 * r + z];
          u[y] += e0[z] * x;
          v[y] += e1[z] * x;
        }
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      if (jt < row0[y]) {
        const int steps = row0[y] + lr - jt - 31;
        sum += (double)(power(g2, steps) * ((float)steps * u[y] + v[y]));
      } else if (jt == row0[y]) {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int steps = lr - acc_row(r, lg);
          x += steps > 0 ? (float)steps * power(g2, steps) * (s[y][r] * t[y][r]) : 0.f;
        }
        sum += (double)x;
      }
    }
  };
  for (int it = 0; it < chunks; ++it) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (it + 1 < chunks) issue(it + 1);
#pragma unroll 1
    for (int jh = 0; jh < 2; ++jh) {
      const int jt = it * kChunk + 32 * jh;
      if (jt > row0[1] || jt >= n) break;
      rd.renew_rows();
      tile(tk[it % STAGES], tv[it % STAGES], jh, jt);
    }
  }
  sum = workgroup_sum<NW>(sum * (double)p.scale, red);
  if (tid == 0) *out = sum;
}

// ---------------------------------------------------------------------------------------------
// In place: each segment's own state becomes the state carried into it, and the last one leaves; forwards the
// derivatives with them, backwards the sequence's end of the decay's gradient, <T, dS>.
// ---------------------------------------------------------------------------------------------
struct CarryParams {
  Shape s;
  float* states;
  float* derivs;        // forwards, or null: [B, H, n_seg + 1, D, D], the last one the sequence's
  const float* first;   // [B, H, D, D] or null
  float* last;          // or null
  const float* T;       // backwards, or null: the derivatives
  double* part;
  int n_part, part_at;
  int rev, dd;
};

// One element a thread: only the multiply-adds are sequential, so the loads of eight segments go out together.
__global__ void __launch_bounds__(kThreads) carry_kernel(CarryParams p) {
  constexpr int AHEAD = 8;
  __shared__ double red[kThreads / 64];
  const int e = blockIdx.x * kThreads + threadIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const float g2 = log2_decay(p.s, h);
  const int64_t own = (int64_t)bh * p.dd + e;
  float x = p.first ? p.first[own] : 0.f, dx = 0.f;
  float* st = p.states + (int64_t)bh * p.s.n_seg * p.dd + e;
  float* dt = p.derivs ? p.derivs + (int64_t)bh * (p.s.n_seg + 1) * p.dd + e : nullptr;
  if (p.T) {
    const double sum = workgroup_sum<kThreads / 64>((double)(x * p.T[((int64_t)bh * (p.s.n_seg + 1) + p.s.n_seg) * p.dd + e]), red);
    if (threadIdx.x == 0) p.part[(int64_t)bh * p.n_part + p.part_at + blockIdx.x] = sum;
  }
  for (int i0 = 0; i0 < p.s.n_seg; i0 += AHEAD) {
    float local[AHEAD], dlocal[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int c = p.rev ? p.s.n_seg - 1 - (i0 + i) : i0 + i;
      if (i0 + i < p.s.n_seg) local[i] = st[(int64_t)c * p.dd];
      if (i0 + i < p.s.n_seg && dt) dlocal[i] = dt[(int64_t)c * p.dd];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int c = p.rev ? p.s.n_seg - 1 - (i0 + i) : i0 + i;
      if (i0 + i < p.s.n_seg) {
        const int n = tokens_of(p.s, b, c);
        const float keep = power(g2, n);
        st[(int64_t)c * p.dd] = x;
        if (dt) {
          dt[(int64_t)c * p.dd] = dx;
          dx = keep * (dx + (float)n * x) + dlocal[i];
        }
        x = x * keep + local[i];
      }
    }
  }
  if (p.last) p.last[own] = x;
  if (dt) dt[(int64_t)p.s.n_seg * p.dd] = dx;
}

// The decay's gradient of one head: all parts of its rows, in a fixed order.
__global__ void __launch_bounds__(kThreads) decay_grad_kernel(const double* part, int B, int H, int n_part, float* out) {
  __shared__ double red[kThreads / 64];
  const int h = blockIdx.x;
  double s = 0.0;
  for (int i = threadIdx.x; i < B * n_part; i += kThreads) s += part[((int64_t)(i / n_part) * H + h) * n_part + i % n_part];
  s = workgroup_sum<kThreads / 64>(s, red);
  if (threadIdx.x == 0) out[h] = (float)s;
}

// ---------------------------------------------------------------------------------------------
// Single tokens. A workgroup holds a slice of the value channels of one state: thread (row, column
// group) takes rows row, row + R, ... of VEC columns. Bound by reading and writing the state once: 64
// sequences x 16 heads of 128 x 128, 134 MB, 23 us (5.8 TB/s); one sequence of 12 heads 4.5 us.
// ---------------------------------------------------------------------------------------------
struct StepParams {
  View q, k, v;
  void* o; int64_t o_sb, o_st, o_sh;
  int L, H, D, Dv, dtype;
  const float* log_decay;
  float* state; int64_t st_sb, st_sh;
  float scale;
};

constexpr int kStepMax = 256;   // head dim

template <int VEC, int COLS>
__global__ void __launch_bounds__(kThreads) step_kernel(StepParams p) {
  constexpr int CT = COLS / VEC, R = kThreads / CT;   // threads along the columns, rows at a time
  __shared__ float sq[kStepMax], sk[kStepMax];
  __shared__ float red[R][COLS + 1];
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, ct = tid % CT, row0 = tid / CT;
  const int col = blockIdx.x * COLS + ct * VEC;
  const float g = p.log_decay[h], lam = expf(g < -1e30f ? -1e30f : g);
  float* st = p.state + (int64_t)b * p.st_sb + (int64_t)h * p.st_sh;
  for (int t = 0; t < p.L; ++t) {
    const int64_t qo = (int64_t)b * p.q.sb + (int64_t)t * p.q.st + (int64_t)h * p.q.sh;
    const int64_t ko = (int64_t)b * p.k.sb + (int64_t)t * p.k.st + (int64_t)h * p.k.sh;
    const int64_t vo = (int64_t)b * p.v.sb + (int64_t)t * p.v.st + (int64_t)h * p.v.sh;
    for (int i = tid; i < p.D; i += kThreads) {
      sq[i] = wa_load_f(p.q.p, qo + i, p.dtype);
      sk[i] = wa_load_f(p.k.p, ko + i, p.dtype);
    }
    float v[VEC], o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[e] = col + e < p.Dv ? wa_load_f(p.v.p, vo + col + e, p.dtype) : 0.f;
      o[e] = 0.f;
    }
    __syncthreads();
    if (col < p.Dv) {
#pragma unroll 4
      for (int d = row0; d < p.D; d += R) {
        float* at = st + (int64_t)d * p.Dv + col;
        if constexpr (VEC == 4) {
          f32x4 s = *(f32x4*)at;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[e] = s[e] * lam + sk[d] * v[e];
            o[e] += sq[d] * s[e];
          }
          *(f32x4*)at = s;
        } else {
          const float s = *at * lam + sk[d] * v[0];
          o[0] += sq[d] * s;
          *at = s;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[row0][ct * VEC + e] = o[e];
    __syncthreads();
    if (tid < COLS && blockIdx.x * COLS + tid < p.Dv) {
      float s = 0.f;
      for (int r = 0; r < R; ++r) s += red[r][tid];
      wa_store_f(p.o, (int64_t)b * p.o_sb + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + blockIdx.x * COLS + tid, s * p.scale, p.dtype);
    }
    __syncthreads();
  }
}

// Segments. The rows kernel's LDS ring takes most of a CU, so its workgroups run in rounds of 256, as long as a
// segment; each segment costs its states' writing, carrying and reading; with derivatives (training) the pairs
// inside a segment grow with its length. Weights in us, fitted at 32,760 tokens of 12 x 128: 0.08 a token of a
// round and rows launch (5 launches' worth in training, 1.4 with the state pass alone), 0.05 (0.2 with
// derivatives) a segment, 2.8e-7 a token and token of segment. That call takes 21 segments of 1,600 tokens for its
// output alone and 64 of 512 in training (the call 823 us; in 32 segments 888, 43 871, 86 923). The weights and the
// 256 are bf16's with D = 128, used for all: with D = 64 two workgroups fit a CU and half of a round stays empty (111
// us for the same tokens and heads, 367 in training), and fp32's rows take longer than a weight says (4 heads of 8,190
// tokens of 128: 80 us, 335 in training). Sequences count as full, whatever their lengths. "Training" is a call that
// asks for the decays' gradient; with fixed decays the segments are the output's (590 us for the call above).
int64_t segment_length(int64_t B, int64_t L, int64_t H, bool derivs) {
  const double rows = (double)(B * H);
  int64_t best = 0;
  double best_cost = 0.0;
  for (int64_t k = 1; k <= std::min<int64_t>(512, (L + 127) / 128); ++k) {
    const int64_t seg = std::max<int64_t>(128, ((L + k - 1) / k + kChunk - 1) / kChunk * kChunk);
    const int64_t n = (L + seg - 1) / seg, rounds = (B * H * n + 255) / 256;
    const double cost = (derivs ? 0.4 : 0.11) * (double)(rounds * seg) + rows * ((derivs ? 0.2 : 0.05) * (double)n +
                        (derivs ? 2.8e-7 * (double)L * (double)seg : 0.0));
    if (best == 0 || cost < best_cost) {
      best_cost = cost;
      best = seg;
    }
  }
  return best;
}

// Rows that the kernels read or write: 16-byte aligned, at most kMaxTokenStride elements apart and at least `apart`.
bool rows16(const void* p, int64_t sb, int64_t st, int64_t sh, int dtype, int64_t apart) {
  const int v = dtype == WA_BF16 ? 8 : 4;
  return wa_aligned16(p) && st >= apart && st <= kMaxTokenStride && sb % v == 0 && st % v == 0 && sh % v == 0;
}
// Outputs are written once, and ChunkStream cuts rows off by a byte range, which holds parts of them all where they
// overlap: there each row must lie behind the one before it.
int64_t apart_written(int64_t L, int64_t D) { return L > 1 ? D : 0; }
int64_t apart_read(int dtype, int64_t L, int64_t D) { return dtype == WA_BF16 ? apart_written(L, D) : 0; }

int check_shape(const char* what, int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  WA_CHECK_ARG(dtype == WA_F32 || dtype == WA_BF16, "%s: unsupported dtype %d", what, dtype);
  WA_CHECK_ARG(D == 64 || D == 128, "%s: head dim must be 64 or 128, got %lld", what, (long long)D);
  WA_CHECK_ARG(B >= 0 && L >= 0 && H >= 0 && L <= INT32_MAX / 2 && B * H <= 65535, "%s: bad sizes B %lld L %lld H %lld", what,
               (long long)B, (long long)L, (long long)H);
  return WA_OK;
}

Shape shape_of(int64_t B, int64_t L, int64_t H, bool derivs, const float* g, const int32_t* lengths) {
  const int64_t seg = segment_length(B, L, H, derivs);
  return Shape{(int)B, (int)L, (int)H, (int)seg, (int)((L + seg - 1) / seg), g, lengths};
}

// Workgroups of the pairs kernel along a head: one per segment in fp32, one per 256 rows in bf16.
int64_t pair_groups(int dtype, const Shape& s) {
  return dtype == WA_F32 ? s.n_seg : (int64_t)s.n_seg * ((s.seg + kPairRows - 1) / kPairRows);
}

template <int D, bool DERIV>
void segment_states(int dtype, const StateParams& p, hipStream_t st) {
  const dim3 grid(p.s.n_seg, p.s.B * p.s.H);
  if (dtype == WA_BF16) hipLaunchKernelGGL((segment_state_bf16_kernel<D, DERIV>), grid, dim3(64 * (D / 16)), 0, st, p);
  else hipLaunchKernelGGL((segment_state_f32_kernel<D, DERIV>), grid, dim3(kThreads), 0, st, p);
}

template <int D>
void all_rows(int dtype, const RowsParams& p, int jobs, hipStream_t st) {
  const dim3 grid(p.s.n_seg * jobs, p.s.B * p.s.H);
  if (dtype == WA_BF16) hipLaunchKernelGGL((rows_bf16_kernel<D>), grid, dim3(64 * (D / 16)), 0, st, p);
  else hipLaunchKernelGGL((rows_f32_kernel<D>), grid, dim3(kThreads), 0, st, p);
}

template <int D>
int run_fwd(const wa_decay_fwd_args* a, hipStream_t st) {
  const Shape s = shape_of(a->B, a->L, a->H, a->derivs != nullptr, a->log_decay, a->lengths);
  const View q{a->q, a->q_sb, a->q_st, a->q_sh}, k{a->k, a->k_sb, a->k_st, a->k_sh}, v{a->v, a->v_sb, a->v_st, a->v_sh};
  StateParams sp{};
  sp.s = s; sp.b = k; sp.c = v; sp.states = a->states; sp.derivs = a->derivs; sp.w_scale = 1.f;
  if (a->derivs) segment_states<D, true>(a->dtype, sp, st);
  else segment_states<D, false>(a->dtype, sp, st);
  CarryParams cp{};
  cp.s = s; cp.states = a->states; cp.derivs = a->derivs; cp.first = a->initial; cp.last = a->final_state; cp.dd = D * D;
  hipLaunchKernelGGL(carry_kernel, dim3(D * D / kThreads, s.B * s.H), dim3(kThreads), 0, st, cp);
  RowsParams p{};
  p.s = s;
  p.job[0] = rows_job(q, k, v, a->o, a->o_sb, a->o_st, a->o_sh, a->states, false, false, a->scale);
  all_rows<D>(a->dtype, p, 1, st);
  return wa_launch_status("decay_fwd");
}

template <int D>
int run_bwd(const wa_decay_bwd_args* a, hipStream_t st) {
  const Shape s = shape_of(a->B, a->L, a->H, a->derivs != nullptr, a->log_decay, a->lengths);
  const View q{a->q, a->q_sb, a->q_st, a->q_sh}, k{a->k, a->k_sb, a->k_st, a->k_sh}, v{a->v, a->v_sb, a->v_st, a->v_sh};
  const View d{a->dout, a->d_sb, a->d_st, a->d_sh};
  float* Y = (float*)a->workspace;
  double* part = (double*)(Y + (int64_t)s.B * s.H * s.n_seg * D * D);
  const int pairs = (int)pair_groups(a->dtype, s), n_part = s.n_seg + D * D / kThreads + pairs;
  StateParams sp{};
  sp.s = s; sp.b = q; sp.c = d; sp.states = Y; sp.S = a->states; sp.T = a->derivs; sp.part = part; sp.n_part = n_part;
  sp.rev = 1; sp.w_scale = a->scale;
  if (a->dlog_decay) segment_states<D, true>(a->dtype, sp, st);
  else segment_states<D, false>(a->dtype, sp, st);
  CarryParams cp{};
  cp.s = s; cp.states = Y; cp.first = a->dfinal; cp.last = a->dinitial; cp.rev = 1; cp.dd = D * D;
  if (a->dlog_decay) {
    cp.T = a->derivs; cp.part = part; cp.n_part = n_part; cp.part_at = s.n_seg;
  }
  hipLaunchKernelGGL(carry_kernel, dim3(D * D / kThreads, s.B * s.H), dim3(kThreads), 0, st, cp);
  RowsParams p{};
  p.s = s;
  p.job[0] = rows_job(d, v, k, a->dq, a->dq_sb, a->dq_st, a->dq_sh, a->states, true, false, a->scale);
  p.job[1] = rows_job(k, q, d, a->dv, a->dv_sb, a->dv_st, a->dv_sh, Y, false, true, a->scale);
  p.job[2] = rows_job(v, d, q, a->dk, a->dk_sb, a->dk_st, a->dk_sh, Y, true, true, a->scale);
  all_rows<D>(a->dtype, p, 3, st);
  if (a->dlog_decay) {
    const PairsParams pp{s, q, k, v, d, part, n_part, s.n_seg + D * D / kThreads, a->scale};
    const dim3 grid((unsigned)pairs, s.B * s.H);
    if (a->dtype == WA_BF16) hipLaunchKernelGGL((pairs_bf16_kernel<D>), grid, dim3(256), 0, st, pp);
    else hipLaunchKernelGGL((pairs_f32_kernel<D>), grid, dim3(kThreads), 0, st, pp);
    hipLaunchKernelGGL(decay_grad_kernel, dim3(s.H), dim3(kThreads), 0, st, (const double*)part, s.B, s.H, n_part, a->dlog_decay);
  }
  return wa_launch_status("decay_bwd");
}

}  // namespace

extern "C" int64_t wa_decay_segments(int64_t B, int64_t L, int64_t H, int32_t derivs) {
  if (B <= 0 || L <= 0 || H <= 0) return 0;
  return shape_of(B, L, H, derivs != 0, nullptr, nullptr).n_seg;
}

extern "C" int64_t wa_decay_bwd_workspace_bytes(int64_t B, int64_t L, int64_t H, int64_t D, int32_t derivs) {
  if (B <= 0 || L <= 0 || H <= 0) return 0;
  const Shape s = shape_of(B, L, H, derivs != 0, nullptr, nullptr);
  const int64_t parts = s.n_seg + D * D / kThreads + std::max(pair_groups(WA_F32, s), pair_groups(WA_BF16, s));
  return B * H * (s.n_seg * D * D * 4 + parts * 8);
}

extern "C" int wa_decay_fwd(const wa_decay_fwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "decay_fwd: null args");
  const int rc = check_shape("decay_fwd", a->dtype, a->B, a->L, a->H, a->D);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->B > 0 && a->L > 0 && a->H > 0, "decay_fwd: nothing to compute");
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->log_decay && a->states, "decay_fwd: null tensor");
  const int64_t wr = apart_written(a->L, a->D), rd = apart_read(a->dtype, a->L, a->D);
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh, a->dtype, rd) && rows16(a->k, a->k_sb, a->k_st, a->k_sh, a->dtype, rd) &&
               rows16(a->v, a->v_sb, a->v_st, a->v_sh, a->dtype, rd) && rows16(a->o, a->o_sb, a->o_st, a->o_sh, a->dtype, wr),
               "decay_fwd: rows must be 16-byte aligned, tokens at most 2^23 elements apart and, written or in bf16, not overlapping");
  hipStream_t s = (hipStream_t)stream;
  return a->D == 128 ? run_fwd<128>(a, s) : run_fwd<64>(a, s);
}

extern "C" int wa_decay_bwd(const wa_decay_bwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "decay_bwd: null args");
  const int rc = check_shape("decay_bwd", a->dtype, a->B, a->L, a->H, a->D);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->B > 0 && a->L > 0 && a->H > 0, "decay_bwd: nothing to compute");
  WA_CHECK_ARG(a->q && a->k && a->v && a->dout && a->dq && a->dk && a->dv && a->log_decay && a->states && a->workspace,
               "decay_bwd: null tensor");
  WA_CHECK_ARG(!a->dlog_decay == !a->derivs, "decay_bwd: dlog_decay goes with the forward's derivs");
  const int64_t wr = apart_written(a->L, a->D), rd = apart_read(a->dtype, a->L, a->D);
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh, a->dtype, rd) && rows16(a->k, a->k_sb, a->k_st, a->k_sh, a->dtype, rd) &&
               rows16(a->v, a->v_sb, a->v_st, a->v_sh, a->dtype, rd) && rows16(a->dout, a->d_sb, a->d_st, a->d_sh, a->dtype, rd) &&
               rows16(a->dq, a->dq_sb, a->dq_st, a->dq_sh, a->dtype, wr) && rows16(a->dk, a->dk_sb, a->dk_st, a->dk_sh, a->dtype, wr) &&
               rows16(a->dv, a->dv_sb, a->dv_st, a->dv_sh, a->dtype, wr) &&
               wa_aligned16(a->workspace), "decay_bwd: rows and workspace must be 16-byte aligned, tokens at most 2^23 elements apart and, written or in bf16, not overlapping");
  hipStream_t s = (hipStream_t)stream;
  return a->D == 128 ? run_bwd<128>(a, s) : run_bwd<64>(a, s);
}

extern "C" int wa_decay_step(const wa_decay_step_args* a, void* stream) {
  WA_CHECK_ARG(a, "decay_step: null args");
  WA_CHECK_ARG(a->dtype == WA_F32 || a->dtype == WA_BF16, "decay_step: unsupported dtype %d", (int)a->dtype);
  WA_CHECK_ARG(a->D >= 1 && a->D <= kStepMax && a->Dv >= 1 && a->Dv <= kStepMax, "decay_step: head dims must be 1 .. %d, got %lld and %lld",
               kStepMax, (long long)a->D, (long long)a->Dv);
  WA_CHECK_ARG(a->B >= 0 && a->L >= 0 && a->H >= 0 && a->B <= 65535 && a->H <= 65535 && a->L <= INT32_MAX, "decay_step: bad sizes B %lld L %lld H %lld",
               (long long)a->B, (long long)a->L, (long long)a->H);
  if (a->B == 0 || a->L == 0 || a->H == 0) return WA_OK;
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->log_decay && a->state, "decay_step: null tensor");
  WA_CHECK_ARG((a->B == 1 || a->st_sb != 0) && (a->H == 1 || a->st_sh != 0) && (a->B == 1 || a->H == 1 || a->st_sb != a->st_sh),
               "decay_step: states must not share memory");
  const StepParams p{View{a->q, a->q_sb, a->q_st, a->q_sh}, View{a->k, a->k_sb, a->k_st, a->k_sh}, View{a->v, a->v_sb, a->v_st, a->v_sh},
                     a->o, a->o_sb, a->o_st, a->o_sh, (int)a->L, (int)a->H, (int)a->D, (int)a->Dv, (int)a->dtype,
                     a->log_decay, a->state, a->st_sb, a->st_sh, a->scale};
  hipStream_t s = (hipStream_t)stream;
  const bool wide = wa_aligned16(a->state) && a->Dv % 4 == 0 && a->st_sb % 4 == 0 && a->st_sh % 4 == 0;
  if (wide) hipLaunchKernelGGL((step_kernel<4, 32>), dim3((unsigned)((a->Dv + 31) / 32), (unsigned)a->H, (unsigned)a->B), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((step_kernel<1, 32>), dim3((unsigned)((a->Dv + 31) / 32), (unsigned)a->H, (unsigned)a->B), dim3(kThreads), 0, s, p);
  return wa_launch_status("decay_step");
}
