// Attention of single queries over key blocks that a score selects from a KV cache: the selection from
// the cached key block sums (route.hip keeps its own for whole query blocks) and the attention over the
// chosen blocks, for a decoding step, a few drafted tokens or a prompt chunk. No reference counterpart.
#include <algorithm>

#include "tile.h"

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

// Tokens query i of n sees: those up to its own, token length - n + i.
__device__ __forceinline__ int64_t seen_tokens(const int32_t* kv_len, int64_t kv_len_all, int64_t cap, int n, int b, int i) {
  const int64_t len = kv_len ? (int64_t)kv_len[b] : kv_len_all;
  const int64_t in = len < 0 ? 0 : (len > cap ? cap : len);
  const int64_t s = in - n + i + 1;
  return s < 0 ? 0 : s;
}

// =============================================================================================
// Scores: (sum of a group's queries) . (block's key sum) in fp64, 16 queries x 16 blocks at a time
// (v_mfma_f64_16x16x4). D products and their sum are off by at most D 2^-52 of the sum of the products'
// magnitudes, so only scores as close as that depend on the order of the products, of which there are two (a
// single query's below); blocks of equal key sums take the same steps and tie in either. The sums are read
// once; a decoding step fills one row of 16, which the fp64 matrix rate still hides behind the read.
// =============================================================================================
struct SelectParams {
  const bf16_t* q; int64_t q_sb, q_st, q_sh;
  const float* sums;
  const int32_t* kv_len; int64_t kv_len_all, cap;
  int n, H, Hk, nb, bs, topk, sink, local;
  int q_tiles, b_tiles, per;   // 16-query tiles; groups of `per` 16-block tiles
  int64_t rows;
  double* scores;              // [B, n, Hk, n_blocks]
  int32_t* index; int32_t* num;
};

// The group's queries of token qi, in contraction order: slot (step 4 i + j, lane group kg) is channel
// 16 i + 4 kg + j on both sides.
template <int D>
__device__ __forceinline__ void group_queries(const SelectParams& p, int b, int hk, int qi, int kg, double (&a)[D / 4]) {
  const int G = p.H / p.Hk;
#pragma unroll
  for (int i = 0; i < D / 4; ++i) a[i] = 0.0;
  if (qi >= p.n) return;
  const bf16_t* src = p.q + (int64_t)b * p.q_sb + (int64_t)qi * p.q_st + (int64_t)hk * G * p.q_sh + 4 * kg;
  for (int g = 0; g < G; ++g) {
    bf16x4 x[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) x[i] = *(const bf16x4*)(src + (int64_t)g * p.q_sh + 16 * i);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) a[4 * i + j] += (double)(float)x[i][j];
  }
}

template <int D>
__device__ __forceinline__ void load_sums(const SelectParams& p, int64_t bh, int b0, int lane, f32x4 (&x)[D / 16]) {
  const float* src = p.sums + (bh * p.nb + min(b0 + (lane & 15), p.nb - 1)) * D + 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) x[i] = *(const f32x4*)(src + 16 * i);
}

// Accumulator register r of lane (column block, kg) is query row kg + 4 r. Two chains, so that a product need
// not wait for the one before it.
template <int D>
__device__ __forceinline__ f64x4 score_tile(const double (&a)[D / 4], const f32x4 (&x)[D / 16]) {
  f64x4 acc[2] = {{0.0, 0.0, 0.0, 0.0}, {0.0, 0.0, 0.0, 0.0}};
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[4 * i + j], (double)x[i][j], acc[j & 1], 0, 0, 0);
  return acc[0] + acc[1];
}

// Blocks that query i scores end here: from the first local one on they are chosen anyway.
__device__ __forceinline__ int score_end(const SelectParams& p, int b, int i) {
  return (int)((seen_tokens(p.kv_len, p.kv_len_all, p.cap, p.n, b, i) + p.bs - 1) / p.bs) - p.local;
}

template <int D>
__global__ void __launch_bounds__(64) score_kernel(SelectParams p) {
  const int lane = threadIdx.x, row = lane & 15, kg = lane >> 4;
  int u = blockIdx.x;
  const int bt = u % p.b_tiles;
  u /= p.b_tiles;
  const int qt = u % p.q_tiles, bh = u / p.q_tiles, b = bh / p.Hk, hk = bh % p.Hk;
  const int end = score_end(p, b, min(p.n, 16 * qt + 16) - 1), begin = bt * p.per * 16;
  if (begin >= end) return;
  double a[D / 4];
  f32x4 x[2][D / 16];
  load_sums<D>(p, bh, begin, lane, x[0]);    // first: 1,024 queries x 8 heads x 256 blocks 24.6 us, after the queries 28
  group_queries<D>(p, b, hk, 16 * qt + row, kg, a);
  auto tile = [&](int b0, const f32x4 (&now)[D / 16], f32x4 (&next)[D / 16]) {
    if (b0 + 16 < end) load_sums<D>(p, bh, b0 + 16, lane, next);
    const f64x4 acc = score_tile<D>(a, now);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * qt + kg + 4 * r;
      if (i < p.n && b0 + row < p.nb) p.scores[(((int64_t)b * p.n + i) * p.Hk + hk) * p.nb + b0 + row] = acc[r];
    }
  };
  for (int t = 0; t < p.per && begin + 16 * t < end; t += 2) {
    tile(begin + 16 * t, x[0], x[1]);
    if (t + 1 < p.per && begin + 16 * (t + 1) < end) tile(begin + 16 * (t + 1), x[1], x[0]);
  }
}

// =============================================================================================
// Choice: W waves hold a row's scores as order-preserving 64-bit keys, KPT a lane, and find the m-th
// largest by bisection over the key's bits (counts by ballots), then write the chosen ids in
// ascending order by prefix counts.
// =============================================================================================
// Larger score, larger key; NaN above all, -0 as 0. Never 0, which stands for "not scored".
__device__ __forceinline__ uint64_t score_key(double x) {
  if (x != x) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// One row (query i of sequence b, key head hk) by waves 0 .. W - 1 of a workgroup, all of which call it; this is
// wave w. score(j): the row's score of block j.
template <int W, int KPT, typename Score>
__device__ __forceinline__ void choose_row(const SelectParams& p, int b, int i, int hk, int w, int lane, int (*counts)[W], const Score& score) {
  const int64_t row = ((int64_t)b * p.n + i) * p.Hk + hk;
  const int64_t seen = seen_tokens(p.kv_len, p.kv_len_all, p.cap, p.n, b, i);
  const int vis = (int)((seen + p.bs - 1) / p.bs), take = min(vis, p.topk);
  const int lo = min(p.sink, vis), hi = max(lo, vis - p.local);   // scored: [lo, hi)
  const int m = take - (vis - (hi - lo));                         // of them chosen
  const bool all = take == vis;
  const int first = w * 64 * KPT + lane;                          // this lane's blocks: first + 64 e
  uint64_t key[KPT];
#pragma unroll
  for (int e = 0; e < KPT; ++e) {
    const int j = first + 64 * e;
    key[e] = 0;
    if (!all && j >= lo && j < hi) key[e] = score_key(score(j));
  }
  int flip = 0;
  auto total = [&](int mine) {   // over the row's waves; mine is uniform in a wave
    if (W == 1) return mine;
    if (lane == 0) counts[flip][w] = mine;
    __syncthreads();
    int s = 0;
    for (int x = 0; x < W; ++x) s += counts[flip][x];
    flip ^= 1;                   // the next count's writes leave this one's slots alone until the barrier after it
    return s;
  };
  // the m-th largest key: the largest T that at least m keys reach
  uint64_t T = 0;
  bool exact = false;            // exactly m keys reach T
  if (!all && m > 0) {
    for (int bit = 63; bit >= 0 && !exact; --bit) {
      const uint64_t cand = T | (1ull << bit);
      int c = 0;
#pragma unroll
      for (int e = 0; e < KPT; ++e) c += __popcll(__ballot(key[e] >= cand));
      c = total(c);
      if (c >= m) T = cand;
      exact = c == m;
    }
  }
  int ties = 0;                  // keys equal to T that are chosen, lowest ids first
  if (!all && m > 0 && !exact) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < KPT; ++e) c += __popcll(__ballot(key[e] > T));
    ties = m - total(c);
  }
  const uint64_t below = (1ull << lane) - 1;
  int tied = 0;                  // ties in the waves before this one
  if (W > 1 && ties > 0) {
    int c = 0;
#pragma unroll
    for (int e = 0; e < KPT; ++e) c += __popcll(__ballot(key[e] == T));
    if (lane == 0) counts[flip][w] = c;
    __syncthreads();
    for (int x = 0; x < w; ++x) tied += counts[flip][x];
    flip ^= 1;
  }
  // bit e of `mine`: this lane's block first + 64 e is chosen
  uint32_t mine = 0;
  int chosen = 0;
#pragma unroll
  for (int e = 0; e < KPT; ++e) {
    const int j = first + 64 * e;
    bool take_j = j < vis && (all || j < lo || j >= hi);
    if (!all && m > 0 && j >= lo && j < hi) take_j = exact ? key[e] >= T : key[e] > T;
    if (ties > 0) {
      const bool tie = key[e] == T && j >= lo && j < hi;
      const uint64_t t = __ballot(tie);
      if (tie && tied + __popcll(t & below) < ties) take_j = true;
      tied += __popcll(t);
    }
    chosen += __popcll(__ballot(take_j));
    mine |= (uint32_t)take_j << e;
  }
  int at = 0;
  if (W > 1) {
    if (lane == 0) counts[flip][w] = chosen;
    __syncthreads();
    for (int x = 0; x < w; ++x) at += counts[flip][x];
  }
  int32_t* out = p.index + row * p.topk;
#pragma unroll
  for (int e = 0; e < KPT; ++e) {
    const bool mine_e = (mine >> e) & 1;
    const uint64_t t = __ballot(mine_e);
    if (mine_e) out[at + __popcll(t & below)] = first + 64 * e;
    at += __popcll(t);
  }
  const int tid = 64 * w + lane;
  for (int s = take + tid; s < p.topk; s += 64 * W) out[s] = -1;
  if (tid == 0) p.num[row] = take;
}

// W = 1: four rows a workgroup and no barrier.
template <int W, int KPT>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) choose_kernel(SelectParams p) {
  __shared__ int counts[2][W];
  const int lane = threadIdx.x & 63;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (row >= p.rows) return;   // whole waves (W = 1), never a part of a workgroup with barriers
  const int hk = (int)(row % p.Hk), i = (int)(row / p.Hk % p.n), b = (int)(row / p.Hk / p.n);
  choose_row<W, KPT>(p, b, i, hk, W == 1 ? 0 : threadIdx.x >> 6, lane, counts, [&](int j) { return p.scores[row * p.nb + j]; });
}

// Scores and choice of a few queries over a short cache in one launch: a workgroup per sequence and key head,
// the scores in LDS. One launch and 8 bytes a score less; its CU reads the sums alone, so at most kFusedBlocks
// blocks. A single query multiplies on the vector units: of a matrix product it would fill one row of 16, at a
// sixteenth of the rate a CU then has alone (23 us against 16 below). 32 sequences of up to 512 blocks x 8 key heads:
// 16 us against 19.8 + 13.6 in two launches; one sequence of 64 blocks: 6.3 against 5.8 + 4.4, and a launch less
// for the host. The time of few workgroups is a wave's, so eight share the blocks; two where workgroups wait for
// CUs (8 key heads, 8 waves against 2: 32 sequences 15.9 us against 20.4, 64 of 128 blocks 10.2 against 11.6, 128 of
// them 17.3 against 14.5, 512 of 32 blocks 47 against 19).
constexpr int kFusedBlocks = 1024, kFusedScores = 8000;   // the scores within 64 KiB
constexpr int64_t kManyHeads = 1024;

template <int D, int W, bool SINGLE>
__global__ void __launch_bounds__(64 * W) select_few_kernel(SelectParams p) {
  extern __shared__ double sc[];   // [n, n_blocks]
  __shared__ int counts[2][W], one[2][1];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = lane & 15, kg = lane >> 4;
  const int bh = blockIdx.x, b = bh / p.Hk, hk = bh % p.Hk;
  const int end = score_end(p, b, p.n - 1);
  constexpr int STEP = 16 * W;
  if (p.nb > p.topk && 16 * w < end) {
    if constexpr (SINGLE) {
      // eight lanes a block, two blocks a lane: channels 32 i + 4 c + j of block b0 + 8 x + r
      const int r = lane >> 3, c = lane & 7;
      double a[D / 8];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) a[i] = 0.0;
      const bf16_t* q = p.q + (int64_t)b * p.q_sb + (int64_t)hk * (p.H / p.Hk) * p.q_sh + 4 * c;
      for (int g = 0; g < p.H / p.Hk; ++g)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const bf16x4 v = *(const bf16x4*)(q + (int64_t)g * p.q_sh + 32 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[4 * i + j] += (double)(float)v[j];
        }
      f32x4 x[2][2][D / 32];
      auto load = [&](int b0, f32x4 (&to)[2][D / 32]) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            to[y][i] = *(const f32x4*)(p.sums + ((int64_t)bh * p.nb + min(b0 + 8 * y + r, p.nb - 1)) * D + 32 * i + 4 * c);
      };
      auto tile = [&](int b0, const f32x4 (&now)[2][D / 32], f32x4 (&next)[2][D / 32]) {
        if (b0 + STEP < end) load(b0 + STEP, next);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          double s[2] = {0.0, 0.0};
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j & 1] += a[4 * i + j] * (double)now[y][i][j];
          double sum = s[0] + s[1];
#pragma unroll
          for (int m = 1; m < 8; m *= 2) sum += __shfl_xor(sum, m);
          if (c == 0 && b0 + 8 * y + r < p.nb) sc[b0 + 8 * y + r] = sum;
        }
      };
      load(16 * w, x[0]);
      for (int b0 = 16 * w; b0 < end; b0 += 2 * STEP) {
        tile(b0, x[0], x[1]);
        if (b0 + STEP < end) tile(b0 + STEP, x[1], x[0]);
      }
    } else {
      double a[D / 4];
      f32x4 x[2][D / 16];
      load_sums<D>(p, bh, 16 * w, lane, x[0]);
      group_queries<D>(p, b, hk, row, kg, a);
      auto tile = [&](int b0, const f32x4 (&now)[D / 16], f32x4 (&next)[D / 16]) {
        if (b0 + STEP < end) load_sums<D>(p, bh, b0 + STEP, lane, next);
        const f64x4 acc = score_tile<D>(a, now);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (kg + 4 * r < p.n && b0 + row < p.nb) sc[(kg + 4 * r) * p.nb + b0 + row] = acc[r];
      };
      for (int b0 = 16 * w; b0 < end; b0 += 2 * STEP) {
        tile(b0, x[0], x[1]);
        if (b0 + STEP < end) tile(b0 + STEP, x[1], x[0]);
      }
    }
  }
  __syncthreads();
  // A wave a query; a single query with many blocks takes all waves.
  if (SINGLE && p.nb > 256) {
    choose_row<W, kFusedBlocks / (64 * W)>(p, b, 0, hk, w, lane, counts, [&](int j) { return sc[j]; });
  } else {
    for (int i = w; i < p.n; i += W) {
      if (p.nb <= 256) choose_row<1, 4>(p, b, i, hk, 0, lane, one, [&](int j) { return sc[i * p.nb + j]; });
      else choose_row<1, kFusedBlocks / 64>(p, b, i, hk, 0, lane, one, [&](int j) { return sc[i * p.nb + j]; });
    }
  }
}

// =============================================================================================
// Attention. WPR waves take up to 16 query heads of one (sequence, query, key head) over a part of its block
// list, 32-key tiles in turn. Transposed products keep every operand where it was loaded or computed:
//   S^T (32 keys x 16 heads) = K Q^T: a lane holds 16 bytes of a key row;
//   O^T (D x 16 heads) += V^T P^T: the accumulator's keys are the next product's contraction slots
//   (lane group kg, element e: key 16 (e / 4) + 4 kg + e % 4), and lane m's 16 bytes of those eight value
//   rows, regrouped by channel, are rows d = D / 16 m + j of V^T for product j.
// Values go straight into registers, whole rows at a time; keys pass through 8 KiB of LDS of the wave's own
// by direct loads, whole rows too (loaded as operands, 64 bytes of 16 rows at a time, they took more than
// twice the values' time: 1,024 queries x 8 key heads of 16 blocks 322 us against 245, both with WPR 4). A
// tile's registers are not doubled: with a second tile loaded ahead a SIMD holds fewer waves, and less is in
// flight (503 us). Bound by reading the chosen keys and values: from HBM for a decoding step (32 ragged
// sequences x 32 blocks 42 us), from the L2s for a prompt, whose queries share blocks (190 us with WPR 1: 4.3 GB,
// 22 TB/s; a fourth wave a SIMD makes it 208).
// =============================================================================================
struct AttnParams {
  const bf16_t* q; int64_t q_sb, q_st, q_sh;
  const bf16_t* k; int64_t k_sb, k_st, k_sh;
  const bf16_t* v; int64_t v_sb, v_st, v_sh;
  bf16_t* o; int64_t o_sb, o_st, o_sh;
  float* lse;
  const int32_t* index; const int32_t* num;
  const int32_t* kv_len; int64_t kv_len_all, cap;
  int n, H, Hk, topk, bs, g_tiles, splits;
  float scale2;      // scale / ln 2
  float* part;       // [rows][g_tiles][splits][16][D + 2] fp32 of split rows
};

__device__ __forceinline__ f32x4 mma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

constexpr float kLowest = -3.4028234e38f;   // running maximum before the first key: below every score, and no difference of it is NaN

constexpr float kSlack = 8.f;       // log2 of the growth that the running maximum lets pass

// A lane's value combined over the four 16-lane groups (lanes of equal number in their group).
template <typename Op>
__device__ __forceinline__ float over_groups(float x, const Op& op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ uint32_t half_word(const bf16x8& v, int i) { return __builtin_bit_cast(u32x4, v)[i]; }
__device__ __forceinline__ uint32_t half_word(const bf16x4& v, int i) { return __builtin_bit_cast(u32x2, v)[i]; }

template <int N> struct RowPart;     // N bf16 values of a value row
template <> struct RowPart<8> { typedef bf16x8 type; };
template <> struct RowPart<4> { typedef bf16x4 type; };

// Two waves a SIMD promised keep the outputs out of the accumulation registers, whose moves cost 1,024 rows 38 us
// against 34; one-wave rows, bound by the caches, do not gain.
template <int D, int WPR>
__global__ void __launch_bounds__(WPR == 8 ? 512 : 256, WPR == 1 ? 1 : 2) attend_kernel(AttnParams p) {
  constexpr int NW = WPR == 8 ? 8 : 4, ROWS = NW / WPR;   // waves and query rows of a workgroup
  constexpr int KC = D / 32, VC = D / 16;   // 32-channel steps of a key row; channels of a value row a lane holds
  constexpr int CPR = D / 8, RPI = 64 / CPR, KI = 32 / RPI;   // 16-byte chunks of a row; rows and direct loads of a tile
  constexpr int KBYTES = NW * 32 * D * 2, OBYTES = WPR == 1 ? 0 : NW * 16 * (D + 4) * 4;
  typedef typename RowPart<VC>::type VRow;
  __shared__ __attribute__((aligned(1024))) char lds[KBYTES > OBYTES ? KBYTES : OBYTES];   // keys, then the waves' outputs
  __shared__ float sm[NW][16], sl[NW][16];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, kg = lane >> 4;
  const int wr = w % WPR;                   // the wave's number in its row
  int64_t u = blockIdx.x;
  const int split = (int)(u % p.splits);
  u /= p.splits;
  const int gt = (int)(u % p.g_tiles);
  u /= p.g_tiles;
  // neighbouring workgroups take the key heads in turn: with eight of them each XCD's L2 sees one head's cache
  const int hk = (int)(u % p.Hk), groups = (p.n + ROWS - 1) / ROWS;
  u /= p.Hk;
  const int i = (int)(u % groups) * ROWS + w / WPR, b = (int)(u / groups), G = p.H / p.Hk;
  if (i >= p.n) return;                     // a whole wave, where waves share nothing
  const int64_t row = ((int64_t)b * p.n + i) * p.Hk + hk;
  const int heads = min(16, G - 16 * gt);
  const int64_t seen = seen_tokens(p.kv_len, p.kv_len_all, p.cap, p.n, b, i);
  const int shift = p.bs == 64 ? 1 : 2;     // log2 of a block's tiles
  const int tiles = max(0, min(p.num[row], p.topk)) << shift;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  const int32_t* list = p.index + row * p.topk;

  bf16x8 q[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    q[c] = bf16x8{};
    if (l16 < heads)
      q[c] = *(const bf16x8*)(p.q + (int64_t)b * p.q_sb + (int64_t)i * p.q_st + (int64_t)(hk * G + 16 * gt + l16) * p.q_sh + 32 * c + 8 * kg);
  }
  const bf16_t* kb = p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh;
  const bf16_t* vb = p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh;
  float m = kLowest, l = 0.f;
  f32x4 o[VC];
#pragma unroll
  for (int j = 0; j < VC; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // The ids of this wave's next 64 tiles sit in its lanes; a tile without seen tokens is passed over before its
  // loads.
  int ids = 0, ids_at = t1;     // first tile whose id is held
  auto key_of = [&](int t) -> int64_t {   // the tile's first key, -1 if none of its tokens is seen
    if (t >= ids_at + 64 * WPR || t < ids_at) {
      ids_at = t;
      const int mine = t + lane * WPR;
      ids = mine < t1 ? list[mine >> shift] : -1;
    }
    const int id = __builtin_amdgcn_readlane(ids, (t - ids_at) / WPR);
    const int64_t key0 = ((int64_t)id << (shift + 5)) + (t & ((1 << shift) - 1)) * 32;
    return id < 0 || key0 >= seen ? -1 : key0;
  };
  // Keys in LDS: 16-byte chunk c of row r in slot c ^ swizzle(r), so that 16 rows' chunks fall in all banks.
  bf16_t* kt = (bf16_t*)lds + w * 32 * D;
  auto swizzle = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  int k_off[D == 128 ? 4 : 2];  // the lane's row and chunk in direct load i: the swizzle repeats every 16 rows
#pragma unroll
  for (int x = 0; x < (D == 128 ? 4 : 2); ++x) {
    const int r = lane / CPR;
    k_off[x] = (r * (int)p.k_st + ((lane % CPR) ^ swizzle(x * RPI + r)) * 8) * 2;
  }
  const uint32_t v_off = (uint32_t)(4 * kg * (int)p.v_st + VC * l16) * 2;

  for (int t = t0 + wr; t < t1; t += WPR) {
    const int64_t key0 = key_of(t);
    if (key0 < 0) continue;
    const int live = (int)min((int64_t)32, seen - key0);   // keys of the tile that are seen
    VRow v[8];
    const bf16_t* kr = kb + key0 * p.k_st;
    const bf16_t* vr = vb + key0 * p.v_st;
#pragma unroll
    for (int x = 0; x < KI; ++x) {
      const int r0 = x * RPI;   // rows from `live` on read as zeros
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(kr + (int64_t)r0 * p.k_st), (short)0, live > r0 ? ((live - r0 - 1) * (int)p.k_st + D) * 2 : 0, WA_BUF_DWORD3);
      lds_dma16(rs, kt + r0 * D, k_off[x % (D == 128 ? 4 : 2)]);
    }
    if (live == 32) {           // rows at scalar addresses plus one lane offset
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *(const VRow*)((const char*)(vr + (16 * (e >> 2) + (e & 3)) * p.v_st) + v_off);
    } else {                    // past the last seen token its row again
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = *(const VRow*)(vr + min(16 * (e >> 2) + 4 * kg + (e & 3), live - 1) * p.v_st + VC * l16);
    }
    // the keys have landed (only the eight value loads were issued after theirs)
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    float s[8];
    {
      bf16x8 ka[2][KC];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < KC; ++c) ka[h][c] = *(const bf16x8*)(kt + (16 * h + l16) * D + ((4 * c + kg) ^ swizzle(l16)) * 8);
      f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[h] = mma16(ka[h][c], q[c], acc[h]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * h + r] = acc[h][r] * p.scale2;
    }
    if (live < 32) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (16 * (e >> 2) + 4 * kg + (e & 3) >= live) {
          s[e] = -INFINITY;
          v[e] = VRow{};    // a weight of 0 does not silence an infinity
        }
    }
    const float top = over_groups(fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))),
                                  [](float a, float b) { return fmaxf(a, b); });
    // the running maximum follows only when a score is 2^kSlack above it: weights of up to 2^kSlack are as exact
    if (__any(top > m + kSlack)) {
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= f;
#pragma unroll
      for (int j = 0; j < VC; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[j][r] *= f;
    }
    // weights round to bf16 for their product with the values (2^-8 each, independent, so the sum over
    // the keys gains from averaging); the sum that they are divided by, and that leaves as the log-sum-exp,
    // is of the unrounded ones
    bf16x8 pr;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __builtin_amdgcn_exp2f(s[e] - m);
      pr[e] = (bf16_t)x;
      l += x;
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      u32x4 vt;     // channel j of the eight rows: halves of two rows side by side
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vt[e] = __builtin_amdgcn_perm(half_word(v[2 * e + 1], j / 2), half_word(v[2 * e], j / 2), j % 2 ? 0x07060302 : 0x05040100);
      o[j] = mma16(__builtin_bit_cast(bf16x8, vt), pr, o[j]);
    }
  }
  l = over_groups(l, [](float a, float b) { return a + b; });

  // Channel VC (4 kg + r) + j of head l16 is register r of accumulator j.
  auto finish = [&](int g, int d, float sum, float tm, float tl) {
    const int h = hk * G + 16 * gt + g;
    if (p.splits == 1) {
      p.o[(int64_t)b * p.o_sb + (int64_t)i * p.o_st + (int64_t)h * p.o_sh + d] = (bf16_t)(tl > 0.f ? sum / tl : (tl == 0.f ? 0.f : tl));
      if (d == 0 && p.lse) p.lse[((int64_t)b * p.H + h) * p.n + i] = tl == 0.f ? -INFINITY : (tm + log2f(tl)) * WA_LN2;
    } else {
      float* at = p.part + (((row * p.g_tiles + gt) * p.splits + split) * 16 + g) * (D + 2);
      at[2 + d] = sum;
      if (d == 0) {
        at[0] = tm;
        at[1] = tl;
      }
    }
  };
  if constexpr (WPR == 1) {
    if (l16 < heads) {
      const int h = hk * G + 16 * gt + l16;
      const float inv = l > 0.f ? 1.f / l : l;   // 0 for a row without keys, NaN where the scores were
      bf16_t* at = p.o + (int64_t)b * p.o_sb + (int64_t)i * p.o_st + (int64_t)h * p.o_sh;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        VRow x;
#pragma unroll
        for (int j = 0; j < VC; ++j) x[j] = (bf16_t)(o[j][r] * inv);
        *(VRow*)(at + VC * (4 * kg + r)) = x;
      }
      if (kg == 0 && p.lse) p.lse[((int64_t)b * p.H + h) * p.n + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * WA_LN2;
    }
  } else {
    // the waves' parts: each to the common maximum, then summed in wave order
    float(*so)[16][D + 4] = (float(*)[16][D + 4])lds;
    if (kg == 0) {
      sm[w][l16] = m;
      sl[w][l16] = l;
    }
    __syncthreads();
    auto highest = [&](int g) {
      float x = sm[0][g];
#pragma unroll
      for (int y = 1; y < NW; ++y) x = fmaxf(x, sm[y][g]);
      return x;
    };
    const float f = exp2f(m - highest(l16));
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[w][l16][VC * (4 * kg + r) + j] = o[j][r] * f;
    __syncthreads();
    for (int x = tid; x < heads * D; x += 64 * NW) {
      const int g = x / D, d = x % D;
      const float tm = highest(g);
      float sum = 0.f, tl = 0.f;
#pragma unroll
      for (int y = 0; y < NW; ++y) {
        sum += so[y][g][d];
        tl += sl[y][g] * exp2f(sm[y][g] - tm);
      }
      finish(g, d, sum, tm, tl);
    }
  }
}

// The parts of split rows, in split order. One wave per (row, head).
template <int D>
__global__ void __launch_bounds__(kThreads) join_kernel(AttnParams p, int64_t units) {
  const int lane = threadIdx.x & 63;
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);   // (row, query head of the group)
  if (u >= units) return;
  const int G = p.H / p.Hk, g = (int)(u % G);
  const int64_t row = u / G;
  const int hk = (int)(row % p.Hk), i = (int)(row / p.Hk % p.n), b = (int)(row / p.Hk / p.n);
  const float* at = p.part + (((row * p.g_tiles + g / 16) * p.splits) * 16 + g % 16) * (D + 2);
  constexpr int64_t kSplit = 16 * (D + 2);
  float top = kLowest;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, at[s * kSplit]);
  float l = 0.f, o[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float f = exp2f(at[s * kSplit] - top);
    l += at[s * kSplit + 1] * f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] += at[s * kSplit + 2 + lane + 64 * e] * f;
  }
  const int h = hk * G + g;
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    p.o[(int64_t)b * p.o_sb + (int64_t)i * p.o_st + (int64_t)h * p.o_sh + lane + 64 * e] = (bf16_t)(l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l));
  if (lane == 0 && p.lse) p.lse[((int64_t)b * p.H + h) * p.n + i] = l == 0.f ? -INFINITY : (top + log2f(l)) * WA_LN2;
}

// Waves of a row: one where the rows alone fill the GPU (a list's ids and a row's ends are then paid once, and no
// barrier), else four, and eight where the rows leave CUs empty. One wave against four against eight, us: 8,192 rows of
// 16 blocks 194 / 246 / 339, 2,048 98 / 70 / 92, 1,024 46 / 34 / 48; 512 of 32 108 / 87 / 88, 256 - / 43 / 43,
// 8 of 16 (with parts) - / 14.8 / 10.3. One-wave rows share a workgroup by query, so single queries take four (4,096
// rows 282 / 288).
int waves_per_row(int64_t rows, int64_t n) { return rows >= 4096 && n >= 4 ? 1 : rows >= 512 ? 4 : 8; }

// Parts of a row: while the rows alone leave CUs without a workgroup, but not below four tiles for each wave, since
// the parts cost a second launch.
int64_t attn_splits(int64_t rows, int64_t tiles) {
  const int64_t want = rows > 0 ? 256 / rows : 1;
  return std::max<int64_t>(1, std::min<int64_t>(want, tiles / (4 * 8)));
}

int check_lists(const char* what, int64_t B, int64_t n, int64_t H, int64_t Hk, int64_t D, int64_t bs, int64_t topk) {
  WA_CHECK_ARG(D == 64 || D == 128, "%s: head dim must be 64 or 128, got %lld", what, (long long)D);
  WA_CHECK_ARG(bs == 64 || bs == 128, "%s: block size must be 64 or 128, got %lld", what, (long long)bs);
  WA_CHECK_ARG(B >= 1 && n >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0, "%s: bad sizes B %lld n %lld heads %lld / %lld", what,
               (long long)B, (long long)n, (long long)H, (long long)Hk);
  WA_CHECK_ARG(topk >= 1 && topk <= WA_SELECT_MAX_BLOCKS, "%s: topk must be 1 .. %d, got %lld", what, WA_SELECT_MAX_BLOCKS, (long long)topk);
  WA_CHECK_ARG(n <= INT32_MAX && B <= INT32_MAX && H <= 65536 && B * n <= (int64_t)1 << 31, "%s: too many queries", what);
  return WA_OK;
}

// Whether one launch scores and chooses: at most 16 queries (one product tile) whose scores fit.
bool fused(int64_t n, int64_t n_blocks) { return n <= 16 && n_blocks <= kFusedBlocks && n * n_blocks <= kFusedScores; }

template <int W, int KPT>
void launch_choose(const SelectParams& p, hipStream_t s) {
  const int64_t grid = W == 1 ? (p.rows + 3) / 4 : p.rows;
  hipLaunchKernelGGL((choose_kernel<W, KPT>), dim3((unsigned)grid), dim3(W == 1 ? 256 : 64 * W), 0, s, p);
}

template <int D, int W>
void launch_few(const SelectParams& p, dim3 grid, size_t lds, hipStream_t s) {
  if (p.n == 1) hipLaunchKernelGGL((select_few_kernel<D, W, true>), grid, dim3(64 * W), lds, s, p);
  else hipLaunchKernelGGL((select_few_kernel<D, W, false>), grid, dim3(64 * W), lds, s, p);
}
template <int D>
void launch_few(const SelectParams& p, bool many, dim3 grid, size_t lds, hipStream_t s) {
  if (many) launch_few<D, 2>(p, grid, lds, s);
  else launch_few<D, 8>(p, grid, lds, s);
}

}  // namespace

extern "C" int64_t wa_select_blocks_workspace_bytes(int64_t B, int64_t n, int64_t Hk, int64_t n_blocks) {
  return fused(n, n_blocks) ? 0 : B * n * Hk * n_blocks * 8;
}

extern "C" int wa_select_blocks(const wa_select_blocks_args* a, void* stream) {
  WA_CHECK_ARG(a, "select_blocks: null args");
  const int rc = check_lists("select_blocks", a->B, a->n, a->H, a->Hk, a->D, a->block_size, a->topk);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->n_blocks >= 1 && a->n_blocks <= WA_SELECT_MAX_BLOCKS, "select_blocks: 1 .. %d blocks, got %lld", WA_SELECT_MAX_BLOCKS,
               (long long)a->n_blocks);
  WA_CHECK_ARG(a->cap >= 0 && a->cap <= a->n_blocks * a->block_size, "select_blocks: %lld blocks do not hold %lld tokens",
               (long long)a->n_blocks, (long long)a->cap);
  WA_CHECK_ARG(a->sink_blocks >= 0 && a->local_blocks >= 1 && a->sink_blocks <= a->topk && a->local_blocks <= a->topk - a->sink_blocks,
               "select_blocks: topk %lld must hold %lld sink and %lld (>= 1) local blocks", (long long)a->topk,
               (long long)a->sink_blocks, (long long)a->local_blocks);
  WA_CHECK_ARG(a->q && a->k_sums && a->index && a->num && (a->workspace || fused(a->n, a->n_blocks)), "select_blocks: null tensor");
  WA_CHECK_ARG(a->B * a->n * a->Hk <= INT32_MAX, "select_blocks: too many queries");
  WA_CHECK_ARG(wa_aligned16(a->k_sums) && wa_aligned16(a->workspace) && ((uintptr_t)a->q & 7) == 0 && a->q_sb % 4 == 0 &&
               a->q_st % 4 == 0 && a->q_sh % 4 == 0, "select_blocks: misaligned rows");
  const int64_t cap = a->cap ? a->cap : a->n_blocks * a->block_size;
  const int64_t rows = a->B * a->n * a->Hk;
  hipStream_t s = (hipStream_t)stream;
  SelectParams p{};
  p.q = (const bf16_t*)a->q; p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.sums = a->k_sums; p.kv_len = a->kv_len; p.kv_len_all = a->kv_len_all; p.cap = cap;
  p.n = (int)a->n; p.H = (int)a->H; p.Hk = (int)a->Hk; p.nb = (int)a->n_blocks; p.bs = (int)a->block_size;
  p.topk = (int)a->topk; p.sink = (int)a->sink_blocks; p.local = (int)a->local_blocks;
  p.rows = rows; p.index = a->index; p.num = a->num;
  if (fused(a->n, a->n_blocks)) {
    const dim3 grid((unsigned)(a->B * a->Hk));
    const size_t scores = (size_t)(a->n * a->n_blocks * 8);
    const bool many = a->B * a->Hk >= kManyHeads;
    if (a->D == 128) launch_few<128>(p, many, grid, scores, s);
    else launch_few<64>(p, many, grid, scores, s);
    return wa_launch_status("select_blocks");
  }
  p.scores = (double*)a->workspace;
  p.q_tiles = (int)((a->n + 15) / 16);
  // A wave keeps its queries for up to 8 block tiles where the tiles are many, and takes one while waves are few
  // (one against eight: 1,024 queries x 8 heads x 256 blocks 54 us against 28, 128 queries 10 against 18).
  const int64_t tiles = (a->n_blocks + 15) / 16, waves = a->B * a->Hk * p.q_tiles * tiles;
  p.per = (int)std::max<int64_t>(1, std::min<int64_t>({8, tiles, waves / 2048}));
  p.b_tiles = (int)((tiles + p.per - 1) / p.per);
  const int64_t grid = a->B * a->Hk * p.q_tiles * p.b_tiles;
  WA_CHECK_ARG(grid <= INT32_MAX, "select_blocks: too many queries");
  if (a->n_blocks > a->topk) {   // otherwise every seen block is chosen
    if (a->D == 128) hipLaunchKernelGGL((score_kernel<128>), dim3((unsigned)grid), dim3(64), 0, s, p);
    else hipLaunchKernelGGL((score_kernel<64>), dim3((unsigned)grid), dim3(64), 0, s, p);
  }
  if (p.nb <= 256) launch_choose<1, 4>(p, s);
  else if (p.nb <= 1024) launch_choose<1, 16>(p, s);
  else if (p.nb <= 4096) launch_choose<4, 16>(p, s);
  else if (p.nb <= 16384) launch_choose<16, 16>(p, s);
  else launch_choose<16, 32>(p, s);
  return wa_launch_status("select_blocks");
}

extern "C" int64_t wa_selected_attn_workspace_bytes(int64_t B, int64_t n, int64_t H, int64_t Hk, int64_t D, int64_t topk,
                                                    int64_t block_size) {
  if (Hk < 1 || H < Hk) return 0;
  const int64_t units = B * n * Hk * ((H / Hk + 15) / 16), splits = attn_splits(units, topk * block_size / 32);
  return splits > 1 ? units * splits * 16 * (D + 2) * 4 : 0;
}

extern "C" int wa_selected_attn(const wa_selected_attn_args* a, void* stream) {
  WA_CHECK_ARG(a, "selected_attn: null args");
  const int rc = check_lists("selected_attn", a->B, a->n, a->H, a->Hk, a->D, a->block_size, a->topk);
  if (rc != WA_OK) return rc;
  WA_CHECK_ARG(a->cap >= 1 && a->cap <= INT32_MAX, "selected_attn: bad cache of %lld tokens", (long long)a->cap);
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->index && a->num, "selected_attn: null tensor");
  auto rows16 = [](const void* x, int64_t sb, int64_t st, int64_t sh) {
    return wa_aligned16(x) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
  };
  // a tile's keys and values at 32-bit offsets from its first one
  auto near = [](int64_t st) { return st >= 0 && st <= (int64_t)1 << 24; };
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh) && rows16(a->k, a->k_sb, a->k_st, a->k_sh) && rows16(a->v, a->v_sb, a->v_st, a->v_sh) &&
               rows16(a->o, a->o_sb, a->o_st, a->o_sh) && near(a->k_st) && near(a->v_st),
               "selected_attn: rows must be 16-byte aligned, a cache's tokens at most 2^24 elements apart");
  AttnParams p{};
  p.q = (const bf16_t*)a->q; p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.k = (const bf16_t*)a->k; p.k_sb = a->k_sb; p.k_st = a->k_st; p.k_sh = a->k_sh;
  p.v = (const bf16_t*)a->v; p.v_sb = a->v_sb; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.o = (bf16_t*)a->o; p.o_sb = a->o_sb; p.o_st = a->o_st; p.o_sh = a->o_sh;
  p.lse = a->lse; p.index = a->index; p.num = a->num; p.kv_len = a->kv_len; p.kv_len_all = a->kv_len_all; p.cap = a->cap;
  p.n = (int)a->n; p.H = (int)a->H; p.Hk = (int)a->Hk; p.topk = (int)a->topk; p.bs = (int)a->block_size;
  p.g_tiles = (int)((a->H / a->Hk + 15) / 16);
  p.scale2 = (a->scale == 0.f ? 1.f / sqrtf((float)a->D) : a->scale) * WA_LOG2E;
  p.part = (float*)a->workspace;
  const int64_t units = a->B * a->n * a->Hk * p.g_tiles;
  p.splits = (int)attn_splits(units, a->topk * a->block_size / 32);
  WA_CHECK_ARG(p.splits == 1 || p.part, "selected_attn: a launch of %lld rows needs a workspace", (long long)units);
  WA_CHECK_ARG(units * p.splits <= INT32_MAX && a->B * a->n * a->H <= INT32_MAX, "selected_attn: too many queries");
  hipStream_t s = (hipStream_t)stream;
  const int wpr = waves_per_row(units, a->n), rows = wpr == 1 ? 4 : 1;   // waves of a row, rows of a workgroup
  const dim3 grid((unsigned)(a->B * ((a->n + rows - 1) / rows) * a->Hk * p.g_tiles * p.splits));
  const int64_t heads = a->B * a->n * a->H;
  if (a->D == 128) {
    if (wpr == 1) hipLaunchKernelGGL((attend_kernel<128, 1>), grid, dim3(256), 0, s, p);
    else if (wpr == 4) hipLaunchKernelGGL((attend_kernel<128, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attend_kernel<128, 8>), grid, dim3(512), 0, s, p);
  } else {
    if (wpr == 1) hipLaunchKernelGGL((attend_kernel<64, 1>), grid, dim3(256), 0, s, p);
    else if (wpr == 4) hipLaunchKernelGGL((attend_kernel<64, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((attend_kernel<64, 8>), grid, dim3(512), 0, s, p);
  }
  if (p.splits > 1) {
    if (a->D == 128) hipLaunchKernelGGL((join_kernel<128>), dim3((unsigned)((heads + 3) / 4)), dim3(kThreads), 0, s, p, heads);
    else hipLaunchKernelGGL((join_kernel<64>), dim3((unsigned)((heads + 3) / 4)), dim3(kThreads), 0, s, p, heads);
  }
  return wa_launch_status("selected_attn");
}
