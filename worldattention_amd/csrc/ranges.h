// What the rows of the ranged attention see: two runs of keys each, and what tiles of 64 rows see together
// (made by wa_key_ranges, ranged.hip).
#pragma once
#include "common.h"

namespace {

constexpr int kRangeRows = 64;   // rows of one summary

// A tile's record: the hulls of its rows' upper and lower runs (0, 0: no row has one), the keys that all its
// rows hold in their upper, and in their lower runs (start > end: some row has none), and one past its last row that sees anything.
enum { kUpLo, kUpHi, kLowLo, kLowHi, kUpIn0, kUpIn1, kLowIn0, kLowIn1, kRowEnd };

struct Ranges {
  const int32_t* rows;
  const int32_t* tiles;
  int sb, Lq, Lk, n_tiles;   // sb: 0 where the batch shares one set
  __device__ __forceinline__ const int32_t* tile(int b, int i) const {
    return tiles + ((int64_t)b * sb * n_tiles + i) * WA_RANGE_TILE_INTS;
  }
  // The row's runs (upper: x, y; lower: z, w) inside the keys, whatever the tensor holds.
  __device__ __forceinline__ int4 row(int b, int i) const {
    int4 r = *(const int4*)(rows + ((int64_t)b * sb * Lq + i) * 4);
    r.x = min(max(r.x, 0), Lk);
    r.y = min(max(r.y, r.x), Lk);
    r.z = min(max(r.z, 0), Lk);
    r.w = min(max(r.w, r.z), Lk);
    return r;
  }
};

// The 64-key steps that N consecutive tiles of rows walk: one or two runs of keys (the hulls, joined where they touch), cut into
// steps from each run's first key on. All values are wave-uniform.
struct Steps {
  int s0, e0, s1, e1, n0, total;
  int up0, up1, low0, low1;   // keys that every row holds in its upper / lower run
  __device__ __forceinline__ void init(const Ranges& p, int b, int tile, int n) {
    int v[8] = {INT32_MAX, 0, INT32_MAX, 0, 0, INT32_MAX, 0, INT32_MAX};
    for (int i = tile; i < min(tile + n, p.n_tiles); ++i) {
      const int32_t* t = p.tile(b, i);
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        const int lo = t[2 * run], hi = t[2 * run + 1];
        if (hi > lo) {
          v[2 * run] = min(v[2 * run], lo);
          v[2 * run + 1] = max(v[2 * run + 1], hi);
        }
        v[4 + 2 * run] = max(v[4 + 2 * run], t[4 + 2 * run]);
        v[5 + 2 * run] = min(v[5 + 2 * run], t[5 + 2 * run]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_readfirstlane(v[i]);
#pragma unroll
    for (int run = 0; run < 2; ++run) {
      v[2 * run] = max(v[2 * run], 0);
      v[2 * run + 1] = min(v[2 * run + 1], p.Lk);
    }
    const bool up = v[1] > v[0], low = v[3] > v[2];
    s0 = e0 = s1 = e1 = 0;
    if (up && low && v[3] < v[0]) {
      s0 = v[2]; e0 = v[3]; s1 = v[0]; e1 = v[1];
    } else if (up || low) {
      s0 = up && low ? min(v[0], v[2]) : up ? v[0] : v[2];
      e0 = up && low ? max(v[1], v[3]) : up ? v[1] : v[3];
    }
    n0 = (e0 - s0 + 63) / 64;
    total = n0 + (e1 - s1 + 63) / 64;
    up0 = v[4]; up1 = v[5]; low0 = v[6]; low1 = v[7];
  }
  // Step i's first key, and the end of the run it is in.
  __device__ __forceinline__ int key(int i) const { return i < n0 ? s0 + 64 * i : s1 + 64 * (i - n0); }
  __device__ __forceinline__ int end(int i) const { return i < n0 ? e0 : e1; }
  // Whether every row sees all 64 keys from `key` on (which lie before `end`).
  __device__ __forceinline__ bool whole(int key, int end) const {
    return key + 64 <= end && ((key >= up0 && key + 64 <= up1) || (key >= low0 && key + 64 <= low1));
  }
};

// A row's runs as what a key is compared with: start and length, cut off at `end`.
struct RowRuns {
  int up, up_n, low, low_n;
  __device__ __forceinline__ RowRuns(const int4& r, int end) : up(r.x), up_n(max(min(r.y, end) - r.x, 0)), low(r.z), low_n(max(min(r.w, end) - r.z, 0)) {}
  __device__ __forceinline__ bool sees(int key) const { return ((unsigned)(key - up) < (unsigned)up_n) | ((unsigned)(key - low) < (unsigned)low_n); }
};

// Scores beyond the plain product, in units of log2: y = cap tanh(x / cap) with, e = exp(2 x / cap) and r = 1 / (e + 1),
//   tanh = 1 - 2 r   and its derivative   1 - tanh^2 = 4 e r r,
// the first off by a few 2^-24 of the cap wherever x is (e = inf gives r = 0), the second by a few 2^-24 of itself; then the distance's bias.
struct Bend {
  float in, cap2, slope2;   // 2 scale / cap log2(e) with a cap, else scale log2(e); cap log2(e) or 0; slope log2(e)
  __device__ __forceinline__ float operator()(float s, float dist, float& turn) const {
    float y = s * in;
    turn = 1.f;
    if (cap2 > 0.f) {       // uniform over the launch
      const float e = __builtin_amdgcn_exp2f(y), r = __builtin_amdgcn_rcpf(e + 1.f);
      y = fmaf(-2.f * cap2, r, cap2);
      turn = fminf(e, 0x1p100f) * 4.f * r * r;
    }
    return fmaf(-slope2, fabsf(dist), y);
  }
};

}  // namespace
