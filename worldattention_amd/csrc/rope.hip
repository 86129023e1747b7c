// Rotary positions with several axes (time, height, width, ...) for queries and keys, forward and
// gradient (the rotation by the negative angle). No reference counterpart beyond the fixed 3-D table
// of the QKV epilogue (cache.hip): positions are given per token and axis, so text, action and image
// tokens mix freely and lie as far out as an integer reaches.
//
// Angle: position * inv_freq in revolutions, reduced from a product of two doubles that keeps the bits of
// its fraction: off by less than 2^-40 of a revolution at any 64-bit position and frequencies up to 1 (at
// position 10^6 and frequency 1 an fp32 angle is off by 0.03 rad; an fp64 one is at 2^40 by 10^-4). Then one
// fp32 sine and cosine of the reduced angle. A workgroup forms them once per (token, pair) in LDS and
// uses them for its heads, so the fp64 part is 1 / heads of the work.
#include <algorithm>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 2048;    // units (a 16-byte chunk, or the two of a half-split pair run) per workgroup
constexpr int kTurns = 1024;    // (token, pair) sines and cosines a workgroup holds in LDS

struct RopeTensor {
  const void* x; int64_t sb, st, sh;
  void* y; int64_t y_sb, y_st, y_sh;
};

struct RopeAxesParams {
  RopeTensor q, k;
  const void* pos; int64_t p_sb, p_st, p_sa; int pos64;
  const double* inv_freq;
  int sec_end[WA_ROPE_MAX_AXES];
  int L, Hq, H, D, P;           // H: query heads, then key heads
  int TT, HW, t_groups, h_groups, units;  // tokens and heads of a workgroup; units of a head row
  uint32_t row_magic, head_magic;         // div_by's constants of HW * units and of units
  int inverse;
};

// u / n by n's constant floor(2^32 / n) + 1 (0 for n = 1), exact for u n < 2^32.
__device__ __forceinline__ uint32_t div_by(uint32_t u, uint32_t magic) { return magic ? __umulhi(u, magic) : u; }

// The fraction, -1/2 to 1/2, of position * freq / (2 pi). 1 / (2 pi) and the revolutions of a step (freq / (2 pi)) are
// sums of two doubles, 2^-105 relative; the position is cut into 53 bits, a double, and the 11 behind them.
__device__ __forceinline__ double revolutions(int64_t position, double freq) {
#pragma clang fp contract(off)   // a product fused into the difference below would count its rounding twice
  constexpr double kInv = 0.15915494309189535, kInvLow = -9.839338337591243e-18;
  const double step = freq * kInv, low = fma(freq, kInv, -step) + freq * kInvLow;
  const int64_t tail = position & 2047;
  const double head = (double)(position - tail), whole = head * step;
  // the difference is exact, and the first fma what the product rounded off; all but it stays below 2^12
  const double x = (whole - rint(whole)) + (fma(head, step, -whole) + fma(head, low, (double)tail * step));
  return x - rint(x);
}

template <typename T, int VEC>
struct Chunk {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T* p) {
  Chunk<T, VEC> c;
  if constexpr (VEC * sizeof(T) == 16) {
    const u32x4 w = *(const u32x4*)p;
    __builtin_memcpy(&c, &w, 16);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) c.v[e] = p[e];
  }
  return c;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T, VEC>& c) {
  if constexpr (VEC * sizeof(T) == 16) {
    u32x4 w;
    __builtin_memcpy(&w, &c, 16);
    *(u32x4*)p = w;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p[e] = c.v[e];
  }
}

// A unit is the work of one thread at a time. Interleaved: VEC consecutive channels (the last unit of
// an odd D holds one). Half-split: VEC pairs (p, p + P), or past the pairs VEC copied channels.
// Bound by reading and writing every channel once: 40 heads x 32,760 tokens x 128 bf16 244 us (5.5 TB/s), one
// token each of 16 sequences of 32 + 8 heads 3.7 us.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(RopeAxesParams p) {
  __shared__ float2 turn[kTurns];
  const int tid = threadIdx.x;
  int g = blockIdx.x;
  const int hg = g % p.h_groups;
  g /= p.h_groups;
  const int tg = g % p.t_groups, b = g / p.t_groups;
  const int t0 = tg * p.TT, rows = min(p.TT, p.L - t0), h0 = hg * p.HW, heads = min(p.HW, p.H - h0);

  for (int i = tid; i < rows * p.P; i += kThreads) {
    const int r = i / p.P, pr = i - r * p.P;
    int axis = 0;
#pragma unroll
    for (int a = 0; a < WA_ROPE_MAX_AXES - 1; ++a) axis += pr >= p.sec_end[a];
    const int64_t at = (int64_t)b * p.p_sb + (int64_t)(t0 + r) * p.p_st + (int64_t)axis * p.p_sa;
    const int64_t pos = p.pos64 ? ((const int64_t*)p.pos)[at] : (int64_t)((const int32_t*)p.pos)[at];
    float s, c;
    sincospif(2.f * (float)revolutions(pos, p.inv_freq[pr]), &s, &c);
    turn[i] = float2{c, p.inverse ? -s : s};
  }
  __syncthreads();

  const int total = rows * p.HW * p.units;
  for (int u = tid; u < total; u += kThreads) {
    const int r = (int)div_by(u, p.row_magic), ru = u - r * p.HW * p.units;
    const int hl = (int)div_by(ru, p.head_magic), c = ru - hl * p.units;
    if (hl >= heads) continue;
    const int h = h0 + hl;
    const RopeTensor& x = h < p.Hq ? p.q : p.k;
    const int hh = h < p.Hq ? h : h - p.Hq;
    const T* src = (const T*)x.x + (int64_t)b * x.sb + (int64_t)(t0 + r) * x.st + (int64_t)hh * x.sh;
    T* dst = (T*)x.y + (int64_t)b * x.y_sb + (int64_t)(t0 + r) * x.y_st + (int64_t)hh * x.y_sh;
    const float2* tr = turn + r * p.P;
    if constexpr (INTER) {
      const int d = c * VEC;
      if (VEC == 2 && d + 1 >= p.D) {  // the single channel at the end of an odd D
        dst[d] = src[d];
        continue;
      }
      Chunk<T, VEC> v = load_chunk<T, VEC>(src + d);
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const int pr = (d + e) / 2;
        if (pr < p.P) {
          const float2 w = tr[pr];
          const float re = (float)v.v[e], im = (float)v.v[e + 1];
          v.v[e] = (T)(re * w.x - im * w.y);
          v.v[e + 1] = (T)(re * w.y + im * w.x);
        }
      }
      store_chunk<T, VEC>(dst + d, v);
    } else {
      const int d = c * VEC;
      if (d >= p.P) {
        const int at = d + p.P;
        store_chunk<T, VEC>(dst + at, load_chunk<T, VEC>(src + at));
        continue;
      }
      Chunk<T, VEC> v = load_chunk<T, VEC>(src + d), w = load_chunk<T, VEC>(src + d + p.P);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 cs = tr[d + e];
        const float re = (float)v.v[e], im = (float)w.v[e];
        v.v[e] = (T)(re * cs.x - im * cs.y);
        w.v[e] = (T)(re * cs.y + im * cs.x);
      }
      store_chunk<T, VEC>(dst + d, v);
      store_chunk<T, VEC>(dst + d + p.P, w);
    }
  }
}

uint32_t div_magic(uint32_t n) { return n == 1 ? 0u : (uint32_t)((1ull << 32) / n) + 1u; }

bool wide_tensor(const RopeTensor& x, int vec) {
  return wa_aligned16(x.x) && wa_aligned16(x.y) && x.sb % vec == 0 && x.st % vec == 0 && x.sh % vec == 0 &&
         x.y_sb % vec == 0 && x.y_st % vec == 0 && x.y_sh % vec == 0;
}

template <typename T, int VEC>
void rope_launch(const RopeAxesParams& p, bool inter, int64_t grid, hipStream_t s) {
  if (inter) hipLaunchKernelGGL((rope_axes_kernel<T, VEC == 1 ? 2 : VEC, true>), dim3((unsigned)grid), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((rope_axes_kernel<T, VEC, false>), dim3((unsigned)grid), dim3(kThreads), 0, s, p);
}

}  // namespace

extern "C" int wa_rope_axes(const wa_rope_axes_args* a, void* stream) {
  WA_CHECK_ARG(a, "rope_axes: null args");
  WA_CHECK_ARG(a->dtype == WA_F32 || a->dtype == WA_BF16, "rope_axes: unsupported dtype %d", (int)a->dtype);
  WA_CHECK_ARG(a->B >= 0 && a->L >= 0 && a->Hq >= 0 && a->Hk >= 0 && a->D >= 1 && a->D <= WA_ROPE_MAX_DIM,
               "rope_axes: bad sizes B %lld L %lld heads %lld / %lld D %lld", (long long)a->B, (long long)a->L,
               (long long)a->Hq, (long long)a->Hk, (long long)a->D);
  WA_CHECK_ARG(a->n_axes >= 1 && a->n_axes <= WA_ROPE_MAX_AXES, "rope_axes: 1 to %d axes, got %lld", WA_ROPE_MAX_AXES,
               (long long)a->n_axes);
  int64_t pairs = 0;
  RopeAxesParams p{};
  for (int i = 0; i < WA_ROPE_MAX_AXES; ++i) {
    if (i < a->n_axes) {
      WA_CHECK_ARG(a->sections[i] >= 0 && a->sections[i] <= a->D, "rope_axes: bad section %lld", (long long)a->sections[i]);
      pairs += a->sections[i];
    }
    // pairs past the last axis do not exist, so its end is never passed
    p.sec_end[i] = i < a->n_axes - 1 ? (int)pairs : INT32_MAX;
  }
  WA_CHECK_ARG(pairs >= 1 && 2 * pairs <= a->D, "rope_axes: %lld pairs do not fit head dim %lld", (long long)pairs,
               (long long)a->D);
  const int64_t heads = a->Hq + (a->k ? a->Hk : 0);
  if (a->B == 0 || a->L == 0 || heads == 0) return WA_OK;
  WA_CHECK_ARG((a->q || a->Hq == 0) && (a->q_out || a->Hq == 0) && (!a->k || a->k_out || a->Hk == 0) && a->positions && a->inv_freq,
               "rope_axes: null tensor");
  WA_CHECK_ARG(a->L <= INT32_MAX && heads <= 65536, "rope_axes: too many tokens or heads");
  p.q = RopeTensor{a->q, a->q_sb, a->q_st, a->q_sh, a->q_out, a->qo_sb, a->qo_st, a->qo_sh};
  p.k = RopeTensor{a->k, a->k_sb, a->k_st, a->k_sh, a->k_out, a->ko_sb, a->ko_st, a->ko_sh};
  p.pos = a->positions; p.p_sb = a->p_sb; p.p_st = a->p_st; p.p_sa = a->p_sa; p.pos64 = a->pos_int64;
  p.inv_freq = a->inv_freq;
  p.L = (int)a->L; p.Hq = (int)a->Hq; p.H = (int)heads; p.D = (int)a->D; p.P = (int)pairs;
  p.inverse = a->inverse != 0;
  const bool inter = a->interleaved != 0;
  int vec = a->dtype == WA_BF16 ? 8 : 4;
  // 16-byte chunks where every row starts on one and no chunk crosses from pairs to partners
  const bool wide = a->D % vec == 0 && (inter || pairs % vec == 0) && wide_tensor(p.q, vec) && (!a->k || wide_tensor(p.k, vec));
  if (!wide) vec = inter ? 2 : 1;
  p.units = inter ? (p.D + vec - 1) / vec : (p.D - p.P) / vec;
  // A workgroup takes whole tokens (their sines serve all heads) up to kUnits units; short inputs are
  // cut finer, down to one unit a thread, until they fill the GPU.
  int64_t per = kUnits;
  const int64_t all = a->B * a->L * heads * p.units;
  while (per > kThreads && all / per < 1024) per /= 2;
  p.HW = (int)std::min<int64_t>(heads, std::max<int64_t>(1, per / p.units));
  p.TT = (int)std::max<int64_t>(1, std::min<int64_t>({a->L, per / ((int64_t)p.HW * p.units), kTurns / pairs}));
  p.h_groups = (int)((heads + p.HW - 1) / p.HW);
  p.t_groups = (int)((a->L + p.TT - 1) / p.TT);
  p.row_magic = div_magic((uint32_t)(p.HW * p.units));
  p.head_magic = div_magic((uint32_t)p.units);
  const int64_t grid = a->B * p.t_groups * (int64_t)p.h_groups;
  WA_CHECK_ARG(a->B <= INT32_MAX && grid <= INT32_MAX, "rope_axes: too many tokens");
  hipStream_t s = (hipStream_t)stream;
  if (a->dtype == WA_BF16) {
    if (wide) rope_launch<bf16_t, 8>(p, inter, grid, s);
    else rope_launch<bf16_t, 1>(p, inter, grid, s);
  } else {
    if (wide) rope_launch<float, 4>(p, inter, grid, s);
    else rope_launch<float, 1>(p, inter, grid, s);
  }
  return wa_launch_status("rope_axes");
}
