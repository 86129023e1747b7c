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
// Y = lambda^n Y' + scale sum_j lambda^(n - j) q_j dO_j^T, which ends as the initial state's gradient.
//
// Three launches: every segment's own state (segment_state_kernel), the carried states (carry_kernel,
// in place), the rows (rows_kernel, 64-token chunks in sequence with the running state on chip). The
// states are fp32 everywhere; what enters a matrix product of bf16 tensors is rounded to bf16 except
// where an fp32 result leaves the kernel (segment states, the decay's gradient): there the rounded
// operand is split in two bf16 parts (2^-17 relative), so that a state is as exact as its sum.
#include <algorithm>

#include "tile.h"

namespace {

constexpr int kChunk = 64;      // tokens a step of the running state takes
constexpr int kThreads = 256;

typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Frag;
template <> struct Frag<bf16_t> { typedef bf16x8 type; };
template <> struct Frag<float> { typedef f32x8 type; };

// 32 x 32 += (32 x 16) (16 x 32): lane (l32, g) holds 8 values of the contraction, 8 g .. 8 g + 7, of
// operand row / column l32. fp32 runs as 8 products of depth 2 over the same slots.
__device__ __forceinline__ f32x16 mma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return wa_mfma32(a, b, c); }
__device__ __forceinline__ f32x16 mma(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// Accumulator register r of lane (l32, g) is row 8 (r / 4) + 4 g + r % 4, column l32.
__device__ __forceinline__ int acc_row(int r, int g) { return 8 * (r >> 2) + 4 * g + (r & 3); }

// Row-major LDS tiles of W columns: bf16 swizzled (tile.h), fp32 padded by one 16-byte slot.
template <typename T, int W> struct Tile;
template <int W> struct Tile<bf16_t, W> {
  static constexpr int kRow = W;
  static __device__ __forceinline__ bf16x8 row8(const bf16_t* t, int row, int chunk) { return tile_row8<W>(t, row, chunk); }
  static __device__ __forceinline__ bf16x8 col8(const bf16_t* t, int c, int col0, int lane) { return tile_tr8n<W>(t, c, col0, lane); }
  static __device__ __forceinline__ void put8(bf16_t* t, int row, int chunk, const bf16x8& v) { tile_put8<W>(t, row, chunk, v); }
  static __device__ __forceinline__ void put(bf16_t* t, int row, int col, float v) {
    t[row * W + (((col >> 3) ^ dual_swizzle<W>(row)) * 8) + (col & 7)] = (bf16_t)v;
  }
};
template <int W> struct Tile<float, W> {
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

__device__ __forceinline__ bf16x8 load8(const bf16_t* p) { return *(const bf16x8*)p; }
__device__ __forceinline__ f32x8 load8(const float* p) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
  return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

struct View {
  const void* p; int64_t sb, st, sh;
};

// Geometry shared by all kernels. Segment c holds n = clamp(length - c seg, 0, seg) tokens; token i of
// it, in the direction of time taken, is token seg c + i or (backwards) seg c + n - 1 - i.
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
__device__ __forceinline__ float power(float g2, int steps) { return exp2f(g2 * (float)steps); }

// Rows [c0, c0 + 64) of a segment into a tile; rows from n on are zeros.
template <typename T, int D>
__device__ __forceinline__ void stage_rows(T* tile, const T* base, int64_t st, int c0, int n, bool rev) {
  constexpr int CPR = D / 8;
#pragma unroll
  for (int i = 0; i < kChunk * CPR / kThreads; ++i) {
    const int u = threadIdx.x + i * kThreads, row = u / CPR, ch = u % CPR, t = c0 + row;
    typename Frag<T>::type v{};
    if (t < n) v = load8(base + (int64_t)(rev ? n - 1 - t : t) * st + ch * 8);
    Tile<T, D>::put8(tile, row, ch, v);
  }
}

// The state's operand of 16 tokens with its weights lambda^(last - token), in one part or two.
__device__ __forceinline__ void weigh(const bf16x8& b, const float (&w)[8], bf16x8& hi, bf16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = (float)b[e] * w[e];
    hi[e] = (bf16_t)x;
    lo[e] = (bf16_t)(x - (float)hi[e]);
  }
}
__device__ __forceinline__ void weigh(const f32x8& b, const float (&w)[8], f32x8& hi, f32x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = b[e] * w[e];
    lo[e] = 0.f;
  }
}

// acc (this wave's tiles of the state) = lambda^m acc + sum_j w_scale lambda^(m - 1 - j + ahead) b_j c_j^T over
// the chunk's m tokens. D = 128: wave w holds state rows 32 w .. + 31 in four column tiles; D = 64: tile
// (w / 2, w % 2). `split`: the weighted operand in two parts.
template <typename T, int D, bool SPLIT>
__device__ __forceinline__ void state_update(f32x16 (&acc)[D / 32 * D / 32 / 4], const T* tb, const T* tc, int m, float g2,
                                             int ahead, float w_scale, int w, int lane) {
  constexpr int TPW = D / 32 * D / 32 / 4;
  const int g = lane >> 5, dt = D == 128 ? w : w >> 1;
  const float keep = power(g2, m);
#pragma unroll
  for (int i = 0; i < TPW; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] *= keep;
#pragma unroll
  for (int jc = 0; jc < kChunk / 16; ++jc) {
    float wt[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[e] = w_scale * power(g2, max(0, m - 1 - (16 * jc + 8 * g + e) + ahead));
    typename Frag<T>::type hi, lo;
    weigh(Tile<T, D>::col8(tb, jc, 32 * dt, lane), wt, hi, lo);
#pragma unroll
    for (int i = 0; i < TPW; ++i) {
      const int et = D == 128 ? i : w & 1;
      const auto c = Tile<T, D>::col8(tc, jc, 32 * et, lane);
      if (SPLIT && sizeof(T) == 2) acc[i] = mma(lo, c, acc[i]);
      acc[i] = mma(hi, c, acc[i]);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Each segment's own state (or gradient state, backwards with lag 0).
// ---------------------------------------------------------------------------------------------
struct StateParams {
  Shape s;
  View b, c;
  float* states;   // [B, H, n_seg, D, D]
  int rev;
  float w_scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) segment_state_kernel(StateParams p) {
  constexpr int TPW = D / 32 * D / 32 / 4;
  __shared__ __attribute__((aligned(1024))) T tb[kChunk * Tile<T, D>::kRow];
  __shared__ __attribute__((aligned(1024))) T tc[kChunk * Tile<T, D>::kRow];
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 5, l32 = lane & 31;
  const int n = tokens_of(p.s, b, seg);
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  const T* bb = (const T*)p.b.p + (int64_t)b * p.b.sb + (int64_t)h * p.b.sh + first * p.b.st;
  const T* cb = (const T*)p.c.p + (int64_t)b * p.c.sb + (int64_t)h * p.c.sh + first * p.c.st;
  f32x16 acc[TPW];
#pragma unroll
  for (int i = 0; i < TPW; ++i) acc[i] = f32x16{};
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    stage_rows<T, D>(tb, bb, p.b.st, c0, n, p.rev);
    stage_rows<T, D>(tc, cb, p.c.st, c0, n, p.rev);
    __syncthreads();
    state_update<T, D, true>(acc, tb, tc, min(kChunk, n - c0), g2, p.rev, p.w_scale, w, lane);
    __syncthreads();
  }
  float* out = p.states + ((int64_t)bh * p.s.n_seg + seg) * D * D;
  const int dt = D == 128 ? w : w >> 1;
#pragma unroll
  for (int i = 0; i < TPW; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) out[(32 * dt + acc_row(r, g)) * D + 32 * (D == 128 ? i : w & 1) + l32] = acc[i][r];
}

// ---------------------------------------------------------------------------------------------
// In place: each segment's own state becomes the state carried into it, and the last one leaves.
// ---------------------------------------------------------------------------------------------
struct CarryParams {
  Shape s;
  float* states;
  const float* first;   // [B, H, D, D] or null
  float* last;          // or null
  int rev, dd;
};

__global__ void __launch_bounds__(kThreads) carry_kernel(CarryParams p) {
  const int e = (blockIdx.x * kThreads + threadIdx.x) * 4, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  if (e >= p.dd) return;
  const float g2 = log2_decay(p.s, h);
  const int64_t own = (int64_t)bh * p.dd + e;
  f32x4 x = p.first ? *(const f32x4*)(p.first + own) : f32x4{0.f, 0.f, 0.f, 0.f};
  float* st = p.states + (int64_t)bh * p.s.n_seg * p.dd + e;
  for (int i = 0; i < p.s.n_seg; ++i) {
    const int c = p.rev ? p.s.n_seg - 1 - i : i;
    float* at = st + (int64_t)c * p.dd;
    const f32x4 local = *(const f32x4*)at;
    *(f32x4*)at = x;
    const float keep = power(g2, tokens_of(p.s, b, c));
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = x[q] * keep + local[q];
  }
  if (p.last) *(f32x4*)(p.last + own) = x;
}

// ---------------------------------------------------------------------------------------------
// Rows: one workgroup per (segment, batch and head, job).
// ---------------------------------------------------------------------------------------------
struct Job {
  View a, b, c;
  void* y; int64_t y_sb, y_st, y_sh;
  const float* x;     // carried states
  int x_trans, rev;
  float s_intra, s_inter;
};
struct RowsParams {
  Shape s;
  Job job[3];
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowsParams p) {
  constexpr int TPW = D / 32 * D / 32 / 4;  // state tiles of a wave
  constexpr int YT = D / 64;                // output tiles of a wave: 32 rows x D / 2 columns
  typedef typename Frag<T>::type F;
  __shared__ __attribute__((aligned(1024))) T tb[kChunk * Tile<T, D>::kRow];
  __shared__ __attribute__((aligned(1024))) T tc[kChunk * Tile<T, D>::kRow];
  __shared__ __attribute__((aligned(1024))) T tp[kChunk * Tile<T, kChunk>::kRow];
  __shared__ __attribute__((aligned(1024))) T tx[D * Tile<T, D>::kRow];
  const Job& jb = p.job[blockIdx.z];
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, l32 = lane & 31;
  const int rh = w >> 1, ch = w & 1, dt = D == 128 ? w : w >> 1;
  const int n = tokens_of(p.s, b, seg), lag = jb.rev ? 0 : 1;
  const float g2 = log2_decay(p.s, h), w_scale = jb.s_intra / jb.s_inter;
  const int64_t first = (int64_t)seg * p.s.seg;
  const T* ab = (const T*)jb.a.p + (int64_t)b * jb.a.sb + (int64_t)h * jb.a.sh + first * jb.a.st;
  const T* bb = (const T*)jb.b.p + (int64_t)b * jb.b.sb + (int64_t)h * jb.b.sh + first * jb.b.st;
  const T* cb = (const T*)jb.c.p + (int64_t)b * jb.c.sb + (int64_t)h * jb.c.sh + first * jb.c.st;
  T* yb = (T*)jb.y + (int64_t)b * jb.y_sb + (int64_t)h * jb.y_sh + first * jb.y_st;

  // tokens past the sequence's end
  const int rows = (int)min((int64_t)p.s.seg, p.s.L - first);
  for (int u = tid; u < (rows - n) * (D / 8); u += kThreads) {
    T* at = yb + (int64_t)(n + u / (D / 8)) * jb.y_st + (u % (D / 8)) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) at[e] = (T)0.f;
  }
  if (n == 0) return;

  const float* x0 = jb.x + ((int64_t)bh * p.s.n_seg + seg) * D * D;
  f32x16 acc[TPW];
#pragma unroll
  for (int i = 0; i < TPW; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * dt + acc_row(r, g), col = 32 * (D == 128 ? i : w & 1) + l32;
      acc[i][r] = jb.x_trans ? x0[col * D + row] : x0[row * D + col];
    }

  for (int c0 = 0; c0 < n; c0 += kChunk) {
    const int m = min(kChunk, n - c0);
    stage_rows<T, D>(tb, bb, jb.b.st, c0, n, jb.rev);
    stage_rows<T, D>(tc, cb, jb.c.st, c0, n, jb.rev);
#pragma unroll
    for (int i = 0; i < TPW; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        Tile<T, D>::put(tx, 32 * dt + acc_row(r, g), 32 * (D == 128 ? i : w & 1) + l32, acc[i][r]);
    F a[D / 16];
    const int ta = c0 + 32 * rh + l32;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      a[k] = F{};
      if (ta < n) a[k] = load8(ab + (int64_t)(jb.rev ? n - 1 - ta : ta) * jb.a.st + 16 * k + 8 * g);
    }
    __syncthreads();
    // decayed products of this wave's 32 x 32 rows and columns of the chunk
    f32x16 s{};
    if (ch <= rh) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) s = mma(a[k], Tile<T, D>::row8(tb, 32 * ch + l32, 2 * k + g), s);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = 32 * rh + acc_row(r, g), j = 32 * ch + l32;
      Tile<T, kChunk>::put(tp, i, j, j <= i ? s[r] * power(g2, i - j) : 0.f);
    }
    __syncthreads();
#pragma unroll
    for (int yt = 0; yt < YT; ++yt) {
      const int col0 = ch * (D / 2) + 32 * yt;
      f32x16 intra{}, inter{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) inter = mma(a[k], Tile<T, D>::col8(tx, k, col0, lane), inter);
#pragma unroll
      for (int jc = 0; jc < kChunk / 16; ++jc)
        intra = mma(Tile<T, kChunk>::row8(tp, 32 * rh + l32, 2 * jc + g), Tile<T, D>::col8(tc, jc, col0, lane), intra);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = 32 * rh + acc_row(r, g), t = c0 + i;
        if (t < n)
          yb[(int64_t)(jb.rev ? n - 1 - t : t) * jb.y_st + col0 + l32] =
              (T)(jb.s_intra * intra[r] + jb.s_inter * power(g2, i + lag) * inter[r]);
      }
    }
    // the running state enters products of bf16 tensors rounded to bf16, so one part does here
    state_update<T, D, false>(acc, tb, tc, m, g2, 1 - lag, w_scale, w, lane);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// The decay's gradient, d/d log(lambda). A path from token j to token i counts its i - j steps; those
// inside a segment of n tokens are, with S the state before it and Y the gradient state after it,
//   scale sum_{j < i} (i - j) lambda^(i - j) (q_i . k_j)(dO_i . v_j)          both ends inside
// + scale sum_i (i + 1) lambda^(i + 1) q_i S dO_i                             only the end
// + sum_j (n - 1 - j) lambda^(n - 1 - j) k_j Y v_j                            only the beginning
// + n lambda^n <S, Y>                                                         neither.
// All of it from unrounded products (fp32 accumulators; S and Y in two parts), summed in fp64.
// ---------------------------------------------------------------------------------------------
struct GammaParams {
  Shape s;
  View q, k, v, d;
  const float* S; const float* Y;
  double* part;   // [B, H, n_seg]
  float scale;
};

// sum_i weight(i) x_i M z_i over a segment's rows, M fp32 [D, D] in global memory
template <typename T, int D, typename W>
__device__ double bilinear(const float* M, const T* xb, int64_t x_st, const T* zb, int64_t z_st, int n, T* mhi, T* mlo,
                           const W& weight) {
  typedef typename Frag<T>::type F;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, l32 = lane & 31, rh = w >> 1, ch = w & 1;
  __syncthreads();
  for (int u = tid; u < D * D; u += kThreads) {
    const float x = M[u];
    const T hi = (T)x;
    Tile<T, D>::put(mhi, u / D, u % D, (float)hi);
    if (sizeof(T) == 2) Tile<T, D>::put(mlo, u / D, u % D, x - (float)hi);
  }
  __syncthreads();
  double sum = 0.0;
  for (int c0 = 0; c0 < n; c0 += kChunk) {
    F a[D / 16];
    const int ta = c0 + 32 * rh + l32;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      a[k] = F{};
      if (ta < n) a[k] = load8(xb + (int64_t)ta * x_st + 16 * k + 8 * g);
    }
#pragma unroll
    for (int yt = 0; yt < D / 64; ++yt) {
      const int col0 = ch * (D / 2) + 32 * yt;
      f32x16 s{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        if (sizeof(T) == 2) s = mma(a[k], Tile<T, D>::col8(mlo, k, col0, lane), s);
        s = mma(a[k], Tile<T, D>::col8(mhi, k, col0, lane), s);
      }
      float part = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int t = c0 + 32 * rh + acc_row(r, g);
        if (t < n) part += weight(t) * s[r] * (float)zb[(int64_t)t * z_st + col0 + l32];
      }
      sum += (double)part;
    }
  }
  return sum;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) gamma_kernel(GammaParams p) {
  typedef typename Frag<T>::type F;
  __shared__ __attribute__((aligned(1024))) T t0[D * Tile<T, D>::kRow];   // keys and values of a chunk, or a state
  __shared__ __attribute__((aligned(1024))) T t1[sizeof(T) == 2 ? D * Tile<T, D>::kRow : kChunk * Tile<T, D>::kRow];
  __shared__ double red[4];
  const int seg = blockIdx.x, bh = blockIdx.y, b = bh / p.s.H, h = bh % p.s.H;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, l32 = lane & 31, rh = w >> 1, ch = w & 1;
  const int n = tokens_of(p.s, b, seg);
  const float g2 = log2_decay(p.s, h);
  const int64_t first = (int64_t)seg * p.s.seg;
  const T* qb = (const T*)p.q.p + (int64_t)b * p.q.sb + (int64_t)h * p.q.sh + first * p.q.st;
  const T* kb = (const T*)p.k.p + (int64_t)b * p.k.sb + (int64_t)h * p.k.sh + first * p.k.st;
  const T* vb = (const T*)p.v.p + (int64_t)b * p.v.sb + (int64_t)h * p.v.sh + first * p.v.st;
  const T* db = (const T*)p.d.p + (int64_t)b * p.d.sb + (int64_t)h * p.d.sh + first * p.d.st;
  T* tk = t0;
  T* tv = t1;
  double sum = 0.0;
  for (int i0 = 0; i0 < n; i0 += kChunk) {
    F aq[D / 16], ad[D / 16];
    const int ta = i0 + 32 * rh + l32;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      aq[k] = F{};
      ad[k] = F{};
      if (ta < n) {
        aq[k] = load8(qb + (int64_t)ta * p.q.st + 16 * k + 8 * g);
        ad[k] = load8(db + (int64_t)ta * p.d.st + 16 * k + 8 * g);
      }
    }
    for (int j0 = 0; j0 <= i0; j0 += kChunk) {
      __syncthreads();
      stage_rows<T, D>(tk, kb, p.k.st, j0, n, false);
      stage_rows<T, D>(tv, vb, p.v.st, j0, n, false);
      __syncthreads();
      f32x16 a{}, e{};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        a = mma(aq[k], Tile<T, D>::row8(tk, 32 * ch + l32, 2 * k + g), a);
        e = mma(ad[k], Tile<T, D>::row8(tv, 32 * ch + l32, 2 * k + g), e);
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
  sum *= (double)p.scale;
  if (n > 0) {
    const float* S = p.S + ((int64_t)bh * p.s.n_seg + seg) * D * D;
    const float* Y = p.Y + ((int64_t)bh * p.s.n_seg + seg) * D * D;
    sum += (double)p.scale * bilinear<T, D>(S, qb, p.q.st, db, p.d.st, n, t0, t1,
                                            [&](int i) { return (float)(i + 1) * power(g2, i + 1); });
    sum += bilinear<T, D>(Y, kb, p.k.st, vb, p.v.st, n, t0, t1,
                          [&](int j) { return (float)(n - 1 - j) * power(g2, n - 1 - j); });
    double dot = 0.0;
    for (int u = tid; u < D * D; u += kThreads) dot += (double)(S[u] * Y[u]);
    sum += dot * (double)((float)n * power(g2, n));
  }
  sum = wa_wave_sum_d(sum);
  if (lane == 0) red[w] = sum;
  __syncthreads();
  if (tid == 0) p.part[(int64_t)bh * p.s.n_seg + seg] = (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ void __launch_bounds__(64) gamma_sum_kernel(const double* part, int B, int H, int n_seg, float* out) {
  const int h = blockIdx.x, lane = threadIdx.x;
  double s = 0.0;
  for (int i = lane; i < B * n_seg; i += 64) s += part[((int64_t)(i / n_seg) * H + h) * n_seg + i % n_seg];
  s = wa_wave_sum_d(s);
  if (lane == 0) out[h] = (float)s;
}

// ---------------------------------------------------------------------------------------------
// Single tokens. A workgroup holds a slice of the value channels of one state: thread (row, column
// group) takes rows row, row + R, ... of VEC columns. Bound by reading and writing the state once.
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

// Segments: enough workgroups for two on each of 256 CUs, a segment not below 128 tokens (its fp32 state,
// read and written, then costs no more than its tokens) and a multiple of the chunk.
int64_t segment_length(int64_t B, int64_t L, int64_t H) {
  const int64_t want = (L * B * H + 511) / 512;
  return std::max<int64_t>(128, (want + kChunk - 1) / kChunk * kChunk);
}

bool rows16(const void* p, int64_t sb, int64_t st, int64_t sh, int dtype) {
  const int v = dtype == WA_BF16 ? 8 : 4;
  return wa_aligned16(p) && sb % v == 0 && st % v == 0 && sh % v == 0;
}

int check_shape(const char* what, int dtype, int64_t B, int64_t L, int64_t H, int64_t D) {
  WA_CHECK_ARG(dtype == WA_F32 || dtype == WA_BF16, "%s: unsupported dtype %d", what, dtype);
  WA_CHECK_ARG(D == 64 || D == 128, "%s: head dim must be 64 or 128, got %lld", what, (long long)D);
  WA_CHECK_ARG(B >= 0 && L >= 0 && H >= 0 && L <= INT32_MAX / 2 && B * H <= 65535, "%s: bad sizes B %lld L %lld H %lld", what,
               (long long)B, (long long)L, (long long)H);
  return WA_OK;
}

Shape shape_of(int64_t B, int64_t L, int64_t H, const float* g, const int32_t* lengths) {
  return Shape{(int)B, (int)L, (int)H, (int)segment_length(B, L, H), (int)wa_decay_segments(B, L, H), g, lengths};
}

template <typename T, int D>
void launch_states(const Shape& s, const View& b, const View& c, float* states, const float* first, float* last, bool rev,
                   float w_scale, hipStream_t st) {
  hipLaunchKernelGGL((segment_state_kernel<T, D>), dim3(s.n_seg, s.B * s.H), dim3(kThreads), 0, st,
                     StateParams{s, b, c, states, rev, w_scale});
  hipLaunchKernelGGL(carry_kernel, dim3(D * D / 4 / kThreads, s.B * s.H), dim3(kThreads), 0, st,
                     CarryParams{s, states, first, last, rev, D * D});
}

template <typename T, int D>
int run_fwd(const wa_decay_fwd_args* a, hipStream_t st) {
  const Shape s = shape_of(a->B, a->L, a->H, a->log_decay, a->lengths);
  const View q{a->q, a->q_sb, a->q_st, a->q_sh}, k{a->k, a->k_sb, a->k_st, a->k_sh}, v{a->v, a->v_sb, a->v_st, a->v_sh};
  launch_states<T, D>(s, k, v, a->states, a->initial, a->final_state, false, 1.f, st);
  RowsParams p{};
  p.s = s;
  p.job[0] = Job{q, k, v, a->o, a->o_sb, a->o_st, a->o_sh, a->states, 0, 0, a->scale, a->scale};
  hipLaunchKernelGGL((rows_kernel<T, D>), dim3(s.n_seg, s.B * s.H, 1), dim3(kThreads), 0, st, p);
  return wa_launch_status("decay_fwd");
}

template <typename T, int D>
int run_bwd(const wa_decay_bwd_args* a, hipStream_t st) {
  const Shape s = shape_of(a->B, a->L, a->H, a->log_decay, a->lengths);
  const View q{a->q, a->q_sb, a->q_st, a->q_sh}, k{a->k, a->k_sb, a->k_st, a->k_sh}, v{a->v, a->v_sb, a->v_st, a->v_sh};
  const View d{a->dout, a->d_sb, a->d_st, a->d_sh};
  float* Y = (float*)a->workspace;
  double* part = (double*)(Y + (int64_t)s.B * s.H * s.n_seg * D * D);
  launch_states<T, D>(s, q, d, Y, a->dfinal, a->dinitial, true, a->scale, st);
  RowsParams p{};
  p.s = s;
  p.job[0] = Job{d, v, k, a->dq, a->dq_sb, a->dq_st, a->dq_sh, a->states, 1, 0, a->scale, a->scale};
  p.job[1] = Job{k, q, d, a->dv, a->dv_sb, a->dv_st, a->dv_sh, Y, 0, 1, a->scale, 1.f};
  p.job[2] = Job{v, d, q, a->dk, a->dk_sb, a->dk_st, a->dk_sh, Y, 1, 1, a->scale, 1.f};
  hipLaunchKernelGGL((rows_kernel<T, D>), dim3(s.n_seg, s.B * s.H, 3), dim3(kThreads), 0, st, p);
  if (a->dlog_decay) {
    hipLaunchKernelGGL((gamma_kernel<T, D>), dim3(s.n_seg, s.B * s.H), dim3(kThreads), 0, st,
                       GammaParams{s, q, k, v, d, a->states, Y, part, a->scale});
    hipLaunchKernelGGL(gamma_sum_kernel, dim3(s.H), dim3(64), 0, st, (const double*)part, s.B, s.H, s.n_seg, a->dlog_decay);
  }
  return wa_launch_status("decay_bwd");
}

}  // namespace

extern "C" int64_t wa_decay_segments(int64_t B, int64_t L, int64_t H) {
  if (B <= 0 || L <= 0 || H <= 0) return 0;
  const int64_t seg = segment_length(B, L, H);
  return (L + seg - 1) / seg;
}

extern "C" int64_t wa_decay_bwd_workspace_bytes(int64_t B, int64_t L, int64_t H, int64_t D) {
  return B * H * wa_decay_segments(B, L, H) * (D * D * 4 + 8);
}

extern "C" int wa_decay_fwd(const wa_decay_fwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "decay_fwd: null args");
  const int rc = check_shape("decay_fwd", a->dtype, a->B, a->L, a->H, a->D);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->B > 0 && a->L > 0 && a->H > 0, "decay_fwd: nothing to compute");
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->log_decay && a->states, "decay_fwd: null tensor");
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh, a->dtype) && rows16(a->k, a->k_sb, a->k_st, a->k_sh, a->dtype) &&
               rows16(a->v, a->v_sb, a->v_st, a->v_sh, a->dtype) && wa_aligned16(a->states) && wa_aligned16(a->initial) &&
               wa_aligned16(a->final_state), "decay_fwd: rows and states must be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == WA_BF16) return a->D == 128 ? run_fwd<bf16_t, 128>(a, s) : run_fwd<bf16_t, 64>(a, s);
  return a->D == 128 ? run_fwd<float, 128>(a, s) : run_fwd<float, 64>(a, s);
}

extern "C" int wa_decay_bwd(const wa_decay_bwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "decay_bwd: null args");
  const int rc = check_shape("decay_bwd", a->dtype, a->B, a->L, a->H, a->D);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->B > 0 && a->L > 0 && a->H > 0, "decay_bwd: nothing to compute");
  WA_CHECK_ARG(a->q && a->k && a->v && a->dout && a->dq && a->dk && a->dv && a->log_decay && a->states && a->workspace,
               "decay_bwd: null tensor");
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh, a->dtype) && rows16(a->k, a->k_sb, a->k_st, a->k_sh, a->dtype) &&
               rows16(a->v, a->v_sb, a->v_st, a->v_sh, a->dtype) && rows16(a->dout, a->d_sb, a->d_st, a->d_sh, a->dtype) &&
               wa_aligned16(a->states) && wa_aligned16(a->workspace) && wa_aligned16(a->dfinal) && wa_aligned16(a->dinitial),
               "decay_bwd: rows, states and workspace must be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == WA_BF16) return a->D == 128 ? run_bwd<bf16_t, 128>(a, s) : run_bwd<bf16_t, 64>(a, s);
  return a->D == 128 ? run_bwd<float, 128>(a, s) : run_bwd<float, 64>(a, s);
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
  const StepParams p{View{a->q, a->q_sb, a->q_st, a->q_sh}, View{a->k, a->k_sb, a->k_st, a->k_sh}, View{a->v, a->v_sb, a->v_st, a->v_sh},
                     a->o, a->o_sb, a->o_st, a->o_sh, (int)a->L, (int)a->H, (int)a->D, (int)a->Dv, (int)a->dtype,
                     a->log_decay, a->state, a->st_sb, a->st_sh, a->scale};
  hipStream_t s = (hipStream_t)stream;
  const bool wide = wa_aligned16(a->state) && a->Dv % 4 == 0 && a->st_sb % 4 == 0 && a->st_sh % 4 == 0;
  if (wide) hipLaunchKernelGGL((step_kernel<4, 32>), dim3((unsigned)((a->Dv + 31) / 32), (unsigned)a->H, (unsigned)a->B), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((step_kernel<1, 32>), dim3((unsigned)((a->Dv + 31) / 32), (unsigned)a->H, (unsigned)a->B), dim3(kThreads), 0, s, p);
  return wa_launch_status("decay_step");
}
