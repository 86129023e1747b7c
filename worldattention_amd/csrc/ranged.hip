// Attention whose rows see up to two runs of keys (documents, prefixes, windows with sinks, frames), with capped scores and a
// bias by distance: the ranges themselves and the forward pass. No reference counterpart; the backward pass is ranged_bwd.hip.
#include <algorithm>
#include <type_traits>

#include "pipe.h"
#include "ranges.h"

namespace {

// ---------------------------------------------------------------------------------------------
// Ranges: one wave per 64 rows, a row a lane; the summary is a wave's reductions. Made once for a batch.
// ---------------------------------------------------------------------------------------------
struct RulesParams {
  const int32_t* kv_len; int64_t kv_len_all;
  const int32_t* given;
  int causal; int64_t chunk, window, sink;
  const int32_t* prefix; int64_t prefix_all;
  const int32_t* docs; int64_t docs_sb, n_docs;   // borders
  int32_t* rows; int32_t* tiles;
  int B, Lq, Lk, n_tiles;
};

// Disjoint runs, the lower one second: runs that touch become one.
__device__ int4 ordered(int64_t a0, int64_t a1, int64_t b0, int64_t b1, int Lk) {
  auto in = [&](int64_t x) { return (int)min(max(x, (int64_t)0), (int64_t)Lk); };
  int4 r = {in(a0), in(a1), in(b0), in(b1)};
  if (r.y <= r.x) r.x = r.y = 0;
  if (r.w <= r.z) r.z = r.w = 0;
  if (r.y == 0) {          // the only run is the upper one
    r = int4{r.z, r.w, 0, 0};
  } else if (r.w > 0) {
    if (r.z > r.x) r = int4{r.z, r.w, r.x, r.y};
    if (r.w >= r.x) r = int4{r.z, max(r.y, r.w), 0, 0};
  }
  return r;
}

__device__ __forceinline__ int64_t held_tokens(const RulesParams& p, int b) {
  return min(max(p.kv_len ? (int64_t)p.kv_len[b] : p.kv_len_all, (int64_t)0), (int64_t)p.Lk);
}

__device__ int4 by_rules(const RulesParams& p, int b, int i) {
  const int64_t len = held_tokens(p, b);
  const int64_t t = len - p.Lq + i;
  if (t < 0) return int4{0, 0, 0, 0};
  int64_t first = 0, end = len;
  if (p.docs) {
    const int32_t* d = p.docs + b * p.docs_sb;
    int lo = 0, hi = (int)p.n_docs;   // borders up to t
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (d[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    if (lo == 0 || lo == p.n_docs) return int4{0, 0, 0, 0};
    first = (int64_t)d[lo - 1];   // before the first token, too: its chunks, sinks and prefix count from there
    end = min((int64_t)d[lo], len);
  }
  const int64_t reach = p.causal ? min(end, first + ((t - first) / p.chunk + 1) * p.chunk) : end;
  int64_t a0 = first, a1 = reach;
  if (p.window > 0) {
    a0 = max(first, t - p.window + 1);
    if (!p.causal) a1 = min(reach, t + p.window);
  }
  const int64_t prefix = p.prefix ? (int64_t)p.prefix[b] : p.prefix_all;
  return ordered(a0, a1, first, max(min(first + p.sink, reach), min(first + prefix, end)), p.Lk);
}

template <typename Op>
__device__ __forceinline__ int over_wave(int x, const Op& op) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x = op(x, __shfl_xor(x, m, 64));
  return x;
}

__global__ void __launch_bounds__(256) ranges_kernel(RulesParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= (int64_t)p.B * p.n_tiles) return;
  const int b = (int)(tile / p.n_tiles), row0 = (int)(tile % p.n_tiles) * kRangeRows, i = row0 + lane;
  const bool mine = i < p.Lq;
  int4 r = {0, 0, 0, 0};
  if (mine) {
    const int64_t at = ((int64_t)b * p.Lq + i) * 4;
    if (p.given) r = ordered(p.given[at], p.given[at + 1], p.given[at + 2], p.given[at + 3], p.Lk);
    else r = by_rules(p, b, i);
    *(int4*)(p.rows + at) = r;
  }
  auto lowest = [](int x, int y) { return min(x, y); };
  auto highest = [](int x, int y) { return max(x, y); };
  int v[WA_RANGE_TILE_INTS];
#pragma unroll
  for (int run = 0; run < 2; ++run) {
    const int s = run ? r.z : r.x, e = run ? r.w : r.y;
    const bool has = e > s;
    v[2 * run + 1] = over_wave(has ? e : 0, highest);
    v[2 * run] = v[2 * run + 1] > 0 ? over_wave(has ? s : INT32_MAX, lowest) : 0;
    v[4 + 2 * run] = over_wave(!mine ? 0 : has ? s : INT32_MAX, highest);
    v[5 + 2 * run] = over_wave(!mine ? INT32_MAX : has ? e : 0, lowest);
  }
  v[kRowEnd] = over_wave(r.y > 0 || r.w > 0 ? i + 1 : 0, highest);
  v[9] = v[10] = v[11] = 0;
  if (lane == 0) {
#pragma unroll
    for (int x = 0; x < WA_RANGE_TILE_INTS; ++x) p.tiles[tile * WA_RANGE_TILE_INTS + x] = v[x];
  }
}

// The order in which tiles of 128 rows, and of 128 keys, are worked on: those with the most steps first, so that what is left for the end is short
// (8,190 tokens in 7 uneven documents, 16 heads: forward 115 us, 143 in row order; dK and dV 233, 287). One workgroup for the rows and one for the keys
// of a set; a tile's place is the number of tiles before it, in ascending order where there are too many to count against each other. Once for a batch, it
// costs 75 us at 32,760 causal rows, 1.3 ms at 131,072 and 22 ms at 524,288 (kOrderMax), about half that or less under windows and documents; it gains each call of uneven
// documents its last tiles (32,760 rows, 4 heads of 64: 36 us of a forward's 302, 270 of a training call's 1,344; 131,072 rows: 140 of 2,408, 260 of 13,078;
// 524,288 rows, one head: 0.9 ms of a forward's 9.8), causal masks and windows nothing.
constexpr int kOrderMax = 4096;

__global__ void __launch_bounds__(1024) order_kernel(Ranges p, RulesParams rules, int32_t* order, int sorted) {
  __shared__ int s_steps[kOrderMax], s_place[kOrderMax];
  const int set = blockIdx.x >> 1, keys = blockIdx.x & 1, tid = threadIdx.x, n = keys ? p.key_tiles() : p.row_tiles();
  int32_t* out = order + (int64_t)set * (p.row_tiles() + p.key_tiles() + 1) + (keys ? p.row_tiles() : 0);
  if (keys && tid == 0) out[n] = (int)(held_tokens(rules, set) - p.Lq);
  if (n > kOrderMax || !sorted) {   // right for a causal mask: the last rows, the first keys
    for (int i = tid; i < n; i += 1024) out[i] = keys ? i : n - 1 - i;
    return;
  }
  for (int i = tid; i < n; i += 1024) {
    s_steps[i] = s_place[i] = 0;
    if (!keys) {
      Steps st;
      st.of(p, set, 2 * i, 2);
      s_steps[i] = st.total;
    }
  }
  __syncthreads();
  if (keys) {
    for (int t = tid; t < p.n_tiles; t += 1024) {   // a row tile counts for the keys of its two hulls, once where they meet
      const int32_t* r = p.tile(set, t);
      int lo[2], hi[2];
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        const int x = max(r[2 * run], 0), y = min(r[2 * run + 1], p.Lk);
        lo[run] = y > x ? x / 128 : 0;
        hi[run] = y > x ? (y + 127) / 128 : 0;
      }
      for (int i = lo[0]; i < hi[0]; ++i) atomicAdd(&s_steps[i], 1);
      for (int i = lo[1]; i < hi[1]; ++i)
        if (i < lo[0] || i >= hi[0]) atomicAdd(&s_steps[i], 1);
    }
    __syncthreads();
  }
  for (int x = tid; x < n * n; x += 1024) {
    const int i = x / n, j = x % n, mine = s_steps[i], its = s_steps[j];
    if (its > mine || (its == mine && (keys ? j < i : j > i))) atomicAdd(&s_place[i], 1);
  }
  __syncthreads();
  for (int i = tid; i < n; i += 1024) out[s_place[i]] = i;
}

// ---------------------------------------------------------------------------------------------
// Forward. One workgroup of four waves per 128 rows of a head, one pass over the 64-key steps that its rows see, each with the
// running maximum and sum of its softmax; the step loop is pipe.h's: while a half-step's products run, the exponentials of the one before
// it do. A step that every row sees whole needs no mask; the others compare each key with the row's two runs, a row a lane.
// A run's first step starts at its first key and its last one ends with it: keys that no row of the workgroup sees are not read.
// ---------------------------------------------------------------------------------------------
struct FwdParams {
  const bf16_t* q; int64_t q_sb, q_st, q_sh;
  const bf16_t* k; int64_t k_sb, k_st, k_sh;
  const bf16_t* v; int64_t v_sb, v_st, v_sh;
  bf16_t* o; int64_t o_sb, o_st, o_sh;
  float* lse;
  Ranges ranges;
  const float* slopes;
  int B, H, Hk;
  Bend bend;
  int splits;       // parts of a workgroup's steps
  float* part_o;    // [splits][B, H, Lq, D] sums of parts' weighted values
  float* part_ml;   // [splits][B, H, Lq][2] their maxima and sums
};

// Running maximum before the first key: below every score, and finite, so that no difference of it is NaN where a row sees nothing yet.
constexpr float kNoMax = -3.4028234e38f;

template <int D, Bends BENT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) ranged_fwd_kernel(FwdParams p) {
  constexpr int NW = 4, QT = 1, BM = 32 * NW * QT, DC = D / 16, DT = D / 32, TILE = 64 * D;
  using NT = NextTile<D, NW>;
  __shared__ __attribute__((aligned(1024))) bf16_t ks0[TILE];
  __shared__ __attribute__((aligned(1024))) bf16_t ks1[TILE];
  __shared__ __attribute__((aligned(1024))) bf16_t vs0[TILE];
  __shared__ __attribute__((aligned(1024))) bf16_t vs1[TILE];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  // Sequences and key heads fastest, then the heads of a group, then the parts, then the rows: the longest workgroups start first, and the heads that
  // share keys run on one XCD.
  static_assert(BM == 128, "the order is of 128-row tiles");
  const int per = p.H / p.Hk, nbh = p.B * p.Hk;
  int u = (int)blockIdx.x;
  const int bh = u % nbh;
  u /= nbh;
  const int h = (bh % p.Hk) * per + u % per, b = bh / p.Hk;
  u /= per;
  const int split = u % p.splits, qt0 = p.ranges.row_tile(b, u / p.splits);
  Steps st;
  st.init(p.ranges, b, qt0 * (BM / kRangeRows), BM / kRangeRows);
  st.cut(split, p.splits);

  int qi[QT];
  bool q_ok[QT];
  int4 runs[QT];
  bf16x8 qf[QT][DC];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    qi[qt] = qt0 * BM + (w * QT + qt) * 32 + l32;
    q_ok[qt] = qi[qt] < p.ranges.Lq;
    const int row = q_ok[qt] ? qi[qt] : 0;
    runs[qt] = p.ranges.row(b, row);
    if (!q_ok[qt]) runs[qt] = int4{0, 0, 0, 0};
    const bf16_t* qr = p.q + (int64_t)b * p.q_sb + (int64_t)h * p.q_sh + (int64_t)row * p.q_st;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const bf16x8 t = *(const bf16x8*)(qr + c * 16 + g * 8);
      qf[qt][c] = q_ok[qt] ? t : bf16x8{};
    }
  }
  Bend bend = p.bend;
  int pos0 = 0;
  if (BENT && p.slopes) {
    bend.slope2 = p.slopes[h] * WA_LOG2E;
    pos0 = p.ranges.position(b);
  }

  const bf16_t* kb = p.k + (int64_t)b * p.k_sb + (int64_t)(bh % p.Hk) * p.k_sh;
  const bf16_t* vb = p.v + (int64_t)b * p.v_sb + (int64_t)(bh % p.Hk) * p.v_sh;
  int k_off[NT::NI], v_off[NT::NI];
#pragma unroll
  for (int i = 0; i < NT::NI; ++i) {
    const int row = (i * NW + w) * NT::RPI + lane / NT::CPR, pos = lane % NT::CPR;
    k_off[i] = (int)(row * p.k_st + (pos ^ k_swizzle<D>(row)) * 8) * 2;
    v_off[i] = (int)(row * p.v_st + (pos ^ v_swizzle(row)) * 8) * 2;
  }
  // Step s's tile: a descriptor from its first row to the run's end, empty behind the last step.
  auto tile_rs = [&](int s, bool is_k) {
    const bool ok = s < st.total;
    const int key = ok ? st.key(s) : 0, rows = ok ? min(64, st.end(s) - key) : 0;
    const int64_t stride = is_k ? p.k_st : p.v_st;
    return __builtin_amdgcn_make_buffer_rsrc((void*)((is_k ? kb : vb) + key * stride), (short)0,
                                             rows > 0 ? (int)((rows - 1) * stride + D) * 2 : 0, WA_BUF_DWORD3);
  };
  auto load_tile = [&](int s, bool is_k, bf16_t* lds) {
    const __amdgpu_buffer_rsrc_t rs = tile_rs(s, is_k);
#pragma unroll
    for (int i = 0; i < NT::NI; ++i) pipe_dma16(rs, lds + (i * NW + w) * NT::RPI * D, is_k ? k_off[i] : v_off[i]);
  };
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
    for (int c = 0; c < DC; ++c) asm volatile("" : "+v"(qf[qt][c]));
    asm volatile("" : "+v"(runs[qt].x), "+v"(runs[qt].y), "+v"(runs[qt].z), "+v"(runs[qt].w));
  }
  int k_rd[DC];
#pragma unroll
  for (int c = 0; c < DC; ++c) k_rd[c] = l32 * D + ((2 * c + g) ^ k_swizzle<D>(l32)) * 8;
  const int G = lane >> 4, tr_r = (lane & 15) >> 2, tr_q = lane & 3;
  int v_rd[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
    v_rd[t] = (4 * (G >> 1) + tr_r) * D + (((4 * t + 2 * (G & 1) + (tr_q >> 1)) ^ (2 * tr_r)) * 8) + 4 * (tr_q & 1);

  f32x16 oacc[QT][DT];
  float m_i[QT], l_i[QT], neg_m[QT], rs[QT];
  f32x16 S[2][QT];
  bf16x8 P[4][QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
    for (int t = 0; t < DT; ++t) oacc[qt][t] = f32x16{};
    m_i[qt] = kNoMax;
    l_i[qt] = 0.f;
    S[0][qt] = S[1][qt] = f32x16{};
#pragma unroll
    for (int c = 0; c < 4; ++c) P[c][qt] = bf16x8{};
  }
  // Scores are scaled in the exponential's multiply-add: its product is not rounded and the running maximum is, which the weights of a row
  // share while that rounding is small. From a maximum of 2^20 on (a rounding of 2^-4 of a power) the wave forms each half's weights again,
  // from scores that are rounded as the maximum is.
  constexpr float kLarge = 0x1p20f;
  const float sl2 = BENT ? 1.f : p.bend.scale2;
  float most_sum = 65536.f;   // of a row's weights in a half; behind it, the half's weights are formed again
  // Before a half's exponentials: its scores bent, and those of keys that the row does not see at -inf (lane (l32, g) holds keys
  // 32 KH + 8 (r / 4) + 4 g + r % 4 of step s).
  auto ready = [&](auto half, int s) {
    constexpr int KH = decltype(half)::value;
    const int key = st.key(s), end = st.end(s), key0 = key + 32 * KH + 4 * g;
    if constexpr (BENT) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const float far = (float)(key0 - pos0 - qi[qt]);
        f32x16 x = S[KH][qt];   // a copy: an array that the forms' branches reach into goes to memory
        auto bend_all = [&](auto form) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float unused;
            x[r] = bend.bent<decltype(form)::value>(x[r], far + (float)(8 * (r >> 2) + (r & 3)), unused);
          }
        };
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[r]));
        by_form<BENT>(bend, most, bend_all);
        S[KH][qt] = x;
      }
    }
    if (!st.whole(key, end)) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const RowRuns mine(runs[qt], end);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!mine.sees(key0 + 8 * (r >> 2) + (r & 3))) S[KH][qt][r] = -INFINITY;
      }
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) neg_m[qt] = -m_i[qt];
  };
  auto accept = [&](auto half) {
    constexpr int KH = decltype(half)::value;
    bool again = false;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) again |= !(rs[qt] <= most_sum);
    if (__any(again)) {
      if constexpr (BENT) {
        pipe_rescale<D, QT, KH>(S[KH], P, oacc, m_i, l_i, rs, sl2);
      } else {
        float most = kNoMax;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, S[KH][qt][r]);
        const bool large = most_sum < 0.f || __any(most != kNoMax && fabsf(most) * sl2 > kLarge);
        if (large) most_sum = -1.f;
        const float before = large ? sl2 : 1.f;
        f32x16 x[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) x[qt] = S[KH][qt] * before;
        pipe_rescale<D, QT, KH>(x, P, oacc, m_i, l_i, rs, large ? 1.f : sl2);
      }
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) l_i[qt] += rs[qt];
  };
  using H0 = std::integral_constant<int, 0>;
  using H1 = std::integral_constant<int, 1>;
  const PipeLoad no_load{};
  const int T = st.total;
  if (T > 0) {
    load_tile(0, true, ks0);
    load_tile(1, true, ks1);
    load_tile(0, false, vs0);
    pipe_sync<2 * NT::NI>();
    pipe_slot<D, NW, QT, 1, false, true, false, false>(S, P, oacc, qf, ks0, vs0, k_rd, v_rd, neg_m, sl2, no_load, k_off, no_load,
                                                      v_off, w, rs);
    ready(H0{}, 0);
    pipe_slot<D, NW, QT, 0, true, true, false, false>(S, P, oacc, qf, ks0, vs0, k_rd, v_rd, neg_m, sl2, no_load, k_off, no_load,
                                                     v_off, w, rs);
    accept(H0{});
    auto block = [&](auto par, int s) {
      constexpr int PAR = decltype(par)::value;
      bf16_t* const kcur = PAR ? ks1 : ks0;
      bf16_t* const knext = PAR ? ks0 : ks1;
      bf16_t* const vprev = PAR ? vs0 : vs1;
      bf16_t* const vcur = PAR ? vs1 : vs0;
      pipe_sync<0>();
      ready(H1{}, s - 1);
      const PipeLoad ldk{tile_rs(s + 1, true), knext}, ldv{tile_rs(s, false), vcur};
      pipe_slot<D, NW, QT, 1, true, true, true, true>(S, P, oacc, qf, kcur, vprev, k_rd, v_rd, neg_m, sl2, ldk, k_off, ldv, v_off, w, rs);
      accept(H1{});
      ready(H0{}, s);
      pipe_slot<D, NW, QT, 0, true, true, true, false>(S, P, oacc, qf, kcur, vprev, k_rd, v_rd, neg_m, sl2, no_load, k_off, no_load,
                                                      v_off, w, rs);
      accept(H0{});
    };
    int s = 1;
    for (; s + 1 < T; s += 2) {
      block(H1{}, s);
      block(H0{}, s + 1);
    }
    if (s < T) block(H1{}, s);
    auto last = [&](auto par) {
      constexpr int PAR = decltype(par)::value;   // (T - 1) % 2: the stage of V(T - 1)
      bf16_t* const vprev = PAR ? vs1 : vs0;
      pipe_sync<0>();
      ready(H1{}, T - 1);
      pipe_slot<D, NW, QT, 1, true, false, true, false>(S, P, oacc, qf, ks0, vprev, k_rd, v_rd, neg_m, sl2, no_load, k_off, no_load,
                                                       v_off, w, rs);
      accept(H1{});
      pipe_slot<D, NW, QT, 0, false, false, true, false>(S, P, oacc, qf, ks0, vprev, k_rd, v_rd, neg_m, sl2, no_load, k_off, no_load,
                                                        v_off, w, rs);
    };
    if ((T - 1) & 1) last(H1{});
    else last(H0{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // The weights were rounded to bf16 for their product with the values (2^-9 each on average, independent); the sum that divides them, and
  // the log-sum-exp, are of the unrounded ones. Channel 32 t + 8 (r / 4) + 4 g + r % 4 of row l32 is register r of accumulator t.
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float l = l_i[qt] + __shfl_xor(l_i[qt], 32, 64);
    if (!q_ok[qt]) continue;
    const int64_t row = ((int64_t)b * p.H + h) * p.ranges.Lq + qi[qt];
    if (p.splits > 1) {
      const int64_t at = split * ((int64_t)p.B * p.H * p.ranges.Lq) + row;
#pragma unroll
      for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          *(f32x4*)(p.part_o + at * D + 32 * t + 8 * rq + 4 * g) =
              f32x4{oacc[qt][t][4 * rq], oacc[qt][t][4 * rq + 1], oacc[qt][t][4 * rq + 2], oacc[qt][t][4 * rq + 3]};
      }
      if (g == 0) {
        p.part_ml[2 * at] = m_i[qt];
        p.part_ml[2 * at + 1] = l;
      }
      continue;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bf16_t* at = p.o + (int64_t)b * p.o_sb + (int64_t)qi[qt] * p.o_st + (int64_t)h * p.o_sh + 4 * g;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        bf16x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (bf16_t)(oacc[qt][t][4 * rq + i] * inv);
        *(bf16x4*)(at + 32 * t + 8 * rq) = x;
      }
    }
    if (g == 0) p.lse[row] = l == 0.f ? -INFINITY : (m_i[qt] + log2f(l)) * WA_LN2;
  }
}

// The parts of a split launch, in their order: D / 8 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(FwdParams p, int64_t n_rows) {
  constexpr int TPR = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int c0 = threadIdx.x % TPR * 8;
  if (row >= n_rows) return;
  float top = kNoMax;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[2 * (s * n_rows + row)]);
  float l = 0.f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const int64_t at = s * n_rows + row;
    const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * at] - top);
    l += p.part_ml[2 * at + 1] * f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const f32x4 x = *(const f32x4*)(p.part_o + at * D + c0 + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[4 * c + e] += x[e] * f;
    }
  }
  const int i = (int)(row % p.ranges.Lq), h = (int)(row / p.ranges.Lq % p.H), b = (int)(row / p.ranges.Lq / p.H);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf16x8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (bf16_t)(o[e] * inv);
  *(bf16x8*)(p.o + (int64_t)b * p.o_sb + (int64_t)i * p.o_st + (int64_t)h * p.o_sh + c0) = x;
  if (c0 == 0) p.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * WA_LN2;
}

// Parts of a workgroup's steps: while the rows alone leave a CU without its two workgroups, but none below 16 steps (a part's sums are written and
// read once more, and a second launch joins them). 1,024 rows of 32 heads over up to 8,256 keys, capped: two parts 276 us and 9 to join, uncut 354.
int fwd_splits(int64_t B, int64_t H, int64_t Lq, int64_t Lk) {
  const int64_t groups = B * H * ((Lq + 127) / 128);
  return (int)std::max<int64_t>(1, std::min<int64_t>(512 / groups, (Lk + 63) / 64 / 16));
}

template <int D>
void launch_fwd(const FwdParams& p, Bends bends, hipStream_t s) {
  const int64_t grid = (int64_t)p.B * p.H * ((p.ranges.Lq + 127) / 128) * p.splits;
  if (bends == kPlain) hipLaunchKernelGGL((ranged_fwd_kernel<D, kPlain>), dim3((unsigned)grid), dim3(256), 0, s, p);
  else if (bends == kUsual) hipLaunchKernelGGL((ranged_fwd_kernel<D, kUsual>), dim3((unsigned)grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((ranged_fwd_kernel<D, kOther>), dim3((unsigned)grid), dim3(256), 0, s, p);
  if (p.splits > 1) {
    const int64_t n_rows = (int64_t)p.B * p.H * p.ranges.Lq, per = 2048 / D;
    hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)((n_rows + per - 1) / per)), dim3(256), 0, s, p, n_rows);
  }
}

}  // namespace

extern "C" int wa_key_ranges(const wa_key_ranges_args* a, void* stream) {
  WA_CHECK_ARG(a, "key_ranges: null args");
  WA_CHECK_ARG(a->B >= 1 && a->Lq >= 1 && a->Lk >= 0 && a->Lq <= 1 << 30 && a->Lk <= 1 << 30, "key_ranges: bad sizes B %lld Lq %lld Lk %lld",
               (long long)a->B, (long long)a->Lq, (long long)a->Lk);
  WA_CHECK_ARG(a->rows && a->tiles && a->order && wa_aligned16(a->rows), "key_ranges: null or misaligned output");
  WA_CHECK_ARG(a->given || (a->chunk >= 1 && a->window >= 0 && a->sink >= 0 && (a->prefix || a->prefix_all >= 0)),
               "key_ranges: chunk must be at least 1, window, sink and prefix at least 0");
  WA_CHECK_ARG(!a->documents || a->n_borders >= 2, "key_ranges: documents need two borders at least, got %lld", (long long)a->n_borders);
  RulesParams p{};
  p.kv_len = a->kv_len; p.kv_len_all = a->kv_len_all; p.given = a->given; p.causal = a->causal;
  // a rule beyond any sequence is that of the longest one
  const int64_t far = (int64_t)1 << 31;
  p.chunk = std::min(a->chunk, far); p.window = std::min(a->window, far); p.sink = std::min(a->sink, far);
  p.prefix = a->prefix; p.prefix_all = std::min(a->prefix_all, far);
  p.docs = a->documents; p.docs_sb = a->documents_sb; p.n_docs = a->n_borders;
  p.rows = a->rows; p.tiles = a->tiles;
  p.B = (int)a->B; p.Lq = (int)a->Lq; p.Lk = (int)a->Lk; p.n_tiles = (int)((a->Lq + kRangeRows - 1) / kRangeRows);
  const int64_t grid = (a->B * p.n_tiles + 3) / 4;
  WA_CHECK_ARG(a->B <= 1 << 30 && grid <= INT32_MAX, "key_ranges: too many rows");
  hipLaunchKernelGGL(ranges_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, p);
  const Ranges made{a->rows, a->tiles, 1, p.Lq, p.Lk, p.n_tiles, nullptr};
  hipLaunchKernelGGL(order_kernel, dim3((unsigned)(2 * a->B)), dim3(1024), 0, (hipStream_t)stream, made, p, a->order, a->in_order ? 0 : 1);
  return wa_launch_status("key_ranges");
}

extern "C" int64_t wa_ranged_fwd_workspace_bytes(int64_t B, int64_t H, int64_t, int64_t Lq, int64_t Lk, int64_t D) {
  if (B < 1 || H < 1 || Lq < 1 || Lk < 1) return 0;
  const int splits = fwd_splits(B, H, Lq, Lk);
  return splits > 1 ? splits * B * H * Lq * (D + 2) * 4 : 0;
}

extern "C" int wa_ranged_fwd(const wa_ranged_fwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "ranged_fwd: null args");
  WA_CHECK_ARG(a->D == 64 || a->D == 128, "ranged_fwd: head dim must be 64 or 128, got %lld", (long long)a->D);
  WA_CHECK_ARG(a->B >= 1 && a->Lq >= 1 && a->Lk >= 1 && a->Lq <= 1 << 30 && a->Lk <= 1 << 30 && a->Hk >= 1 && a->H >= a->Hk && a->H % a->Hk == 0 &&
               a->B <= INT32_MAX / a->H,
               "ranged_fwd: bad sizes B %lld Lq %lld Lk %lld heads %lld / %lld", (long long)a->B, (long long)a->Lq, (long long)a->Lk,
               (long long)a->H, (long long)a->Hk);
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->lse && a->rows && a->tiles && a->order && wa_aligned16(a->rows), "ranged_fwd: null tensor");
  auto rows16 = [](const void* x, int64_t sb, int64_t st, int64_t sh) {
    return wa_aligned16(x) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
  };
  auto near = [](int64_t st) { return st >= 0 && st <= (int64_t)1 << 23; };   // a tile at 32-bit offsets from its first row
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh) && rows16(a->k, a->k_sb, a->k_st, a->k_sh) && rows16(a->v, a->v_sb, a->v_st, a->v_sh) &&
               rows16(a->o, a->o_sb, a->o_st, a->o_sh) && near(a->k_st) && near(a->v_st),
               "ranged_fwd: rows must be 16-byte aligned, keys and values at most 2^23 elements apart");
  WA_CHECK_ARG(a->scale >= 0.f && a->scale < INFINITY && (a->cap == 0.f || (a->cap >= 1e-6f && a->cap <= 1e6f && a->scale <= 1e30f)),
               "ranged_fwd: scale must be finite and not below 0, cap 0 or 1e-6 .. 1e6 (with a scale of at most 1e30)");
  FwdParams p{};
  p.q = (const bf16_t*)a->q; p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.k = (const bf16_t*)a->k; p.k_sb = a->k_sb; p.k_st = a->k_st; p.k_sh = a->k_sh;
  p.v = (const bf16_t*)a->v; p.v_sb = a->v_sb; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.o = (bf16_t*)a->o; p.o_sb = a->o_sb; p.o_st = a->o_st; p.o_sh = a->o_sh;
  p.lse = a->lse;
  p.ranges = {a->rows, a->tiles, a->ranges_sb ? 1 : 0, (int)a->Lq, (int)a->Lk, (int)((a->Lq + kRangeRows - 1) / kRangeRows), a->order};
  p.slopes = a->slopes;
  p.B = (int)a->B; p.H = (int)a->H; p.Hk = (int)a->Hk;
  const float scale = a->scale == 0.f ? 1.f / sqrtf((float)a->D) : a->scale;
  p.bend = bend_of(scale, a->cap);
  WA_CHECK_ARG(a->B * a->H * ((a->Lq + 127) / 128) <= INT32_MAX, "ranged_fwd: too many rows");
  p.splits = fwd_splits(a->B, a->H, a->Lq, a->Lk);
  WA_CHECK_ARG(p.splits == 1 || (a->workspace && wa_aligned16(a->workspace)), "ranged_fwd: a launch in %d parts needs a workspace", p.splits);
  p.part_o = (float*)a->workspace;
  p.part_ml = p.part_o + p.splits * a->B * a->H * a->Lq * a->D;
  const Bends bends = bends_of(scale, a->cap, a->slopes);
  if (a->D == 128) launch_fwd<128>(p, bends, (hipStream_t)stream);
  else launch_fwd<64>(p, bends, (hipStream_t)stream);
  return wa_launch_status("ranged_fwd");
}
