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
  const int32_t* order;      // of each set: 128-row tiles and then 128-key tiles, those with the most steps first; the first row's position
  __device__ __forceinline__ int row_tiles() const { return (Lq + 127) / 128; }
  __device__ __forceinline__ int key_tiles() const { return (Lk + 127) / 128; }
  __device__ __forceinline__ const int32_t* of_set(int b) const { return order + (int64_t)b * sb * (row_tiles() + key_tiles() + 1); }
  __device__ __forceinline__ int row_tile(int b, int i) const { return placed(of_set(b) + i, row_tiles()); }
  __device__ __forceinline__ int key_tile(int b, int i) const { return placed(of_set(b) + row_tiles() + i, key_tiles()); }
  __device__ __forceinline__ int position(int b) const { return of_set(b)[row_tiles() + key_tiles()]; }
  __device__ __forceinline__ static int placed(const int32_t* at, int n) { return __builtin_amdgcn_readfirstlane(min(max(*at, 0), n - 1)); }
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
  int s0, e0, s1, e1, n0, first, total;
  int up0, up1, low0, low1;   // keys that every row holds in its upper / lower run
  // Any lanes' tiles.
  __device__ __forceinline__ void of(const Ranges& p, int b, int tile, int n) {
    int v[8] = {INT32_MAX, 0, INT32_MAX, 0, 0, INT32_MAX, 0, INT32_MAX};
    for (int i = tile; i < min(tile + n, p.n_tiles); ++i) {
      const int32_t* t = p.tile(b, i);
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        const int lo = t[2 * run], hi = t[2 * run + 1];
        if (hi > lo) {
          v[2 * run] = min(v[2 * run], max(lo, 0));
          v[2 * run + 1] = max(v[2 * run + 1], min(hi, p.Lk));
        }
        v[4 + 2 * run] = max(v[4 + 2 * run], t[4 + 2 * run]);
        v[5 + 2 * run] = min(v[5 + 2 * run], t[5 + 2 * run]);
      }
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
    first = 0;
    total = n0 + (e1 - s1 + 63) / 64;
    up0 = v[4]; up1 = v[5]; low0 = v[6]; low1 = v[7];
  }
  // One wave's.
  __device__ __forceinline__ void init(const Ranges& p, int b, int tile, int n) {
    of(p, b, tile, n);
    int* const all[] = {&s0, &e0, &s1, &e1, &n0, &total, &up0, &up1, &low0, &low1};
#pragma unroll
    for (int* x : all) *x = __builtin_amdgcn_readfirstlane(*x);
  }
  // The steps of part `part` of `parts` alone.
  __device__ __forceinline__ void cut(int part, int parts) {
    if (parts == 1) return;
    first = (int)((int64_t)total * part / parts);
    total = (int)((int64_t)total * (part + 1) / parts) - first;
  }
  // Step i's first key, and the end of the run it is in.
  __device__ __forceinline__ int key(int i) const { return first + i < n0 ? s0 + 64 * (first + i) : s1 + 64 * (first + i - n0); }
  __device__ __forceinline__ int end(int i) const { return first + i < n0 ? e0 : e1; }
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

// Scores beyond the plain product, in units of log2: cap tanh(x / cap), x = scale s, less the distance's bias. Which form of the tanh is right for all of
// a wave's scores is asked once for a tile:
//   kBias   no cap;
//   kClose  |x| <= 0.3 cap: tanh(z) = z P(z^2), P of degree 3 fitted to 1.3e-8 of the value (a weighted least-squares fit of tanh(z) / z on
//           [0, 0.09] with the leading 1 kept), with the scale in its coefficients: five instructions (a chunk of 1,024 rows over 8,256 keys: 256 us, 275
//           with kNear);
//   kNear   |x| <= cap / 2: the same of degree 4, on [0, 1/4] to 1.7e-8: six instructions, more exact than kFar and half its work;
//   kFar    e = exp(2 z), r = 1 / (e + 1): tanh = 1 - 2 r, off by a few 2^-24 of the cap wherever z is (e = inf gives r = 0); its derivative
//           4 e r r, off by a few 2^-24 of itself;
//   kAny    kNear's polynomial in z itself, which any scale and cap leave in fp32: seven instructions;
//   kBoth   kAny or kFar, score by score.
// The last two are of kernels of their own, for caps above kFarCap, a few 2^-24 of which (1e-4 there) show in small scores that share a tile with
// large ones, and for ratios of scale and cap whose powers leave fp32. 8,190 causal tokens, 16 heads on 4 of 128, a cap of 1,100, scores up to it
// everywhere: forward 488 us, with gradients 2,165; kFar 415 and 1,755. As further forms of one kernel they put the forward's scores in scratch and cost
// the attention over codes 4% and learnt slopes 3%, whatever the cap.
enum BendForm { kBias, kClose, kNear, kFar, kAny, kBoth };
enum Bends { kPlain, kUsual, kOther };   // kernels of no cap and no bias; of kBias to kFar; of kAny and kBoth
constexpr float kFarCap = 1024.f;
// Powers of the ratio up to the eighth, times scale2 (at most 2^23), do not pass fp32; where the last coefficient falls below it, scores are below 2^-9 and
// its term, 2^-14 of them at most, shows nowhere.
static inline bool usual_cap(float scale, float cap) {
  return !(cap > 0.f) || (cap <= kFarCap && scale >= 0x1p-15f * cap && scale <= 0x1p12f * cap);
}
static inline Bends bends_of(float scale, float cap, bool bias) { return !usual_cap(scale, cap) ? kOther : cap > 0.f || bias ? kUsual : kPlain; }
struct Bend {
  float close, near;           // largest |s| for kClose, and for kNear or kAny
  float scale2, in, in2, cap2; // scale log2(e); scale / cap; 2 scale / cap log2(e); cap log2(e) or 0
  float c[4], c3[3], icap2;    // kNear's and kClose's coefficients of s^2 (kAny's of z^2) and its powers, times scale2; 1 / cap2
  float slope2;                // slope log2(e)
  // The form for scores of at most `most`, the same in all of the wave's lanes.
  template <Bends BENDS>
  __device__ __forceinline__ BendForm form(float most) const {
    if (BENDS == kOther) return __any(most > near) ? kBoth : kAny;
    if (!(cap2 > 0.f)) return kBias;
    return !__any(most > close) ? kClose : __any(most > near) ? kFar : kNear;
  }
  // The score before the bias, and the cap's derivative there.
  template <BendForm FORM>
  __device__ __forceinline__ float capped(float s, float& turn) const {
    turn = 1.f;
    if constexpr (FORM == kBias) {
      return s * scale2;
    } else if constexpr (FORM == kBoth) {
      float turn_far;
      const float y = capped<kAny>(s, turn), far = capped<kFar>(s, turn_far);
      const bool small = fabsf(s) <= near;
      turn = small ? turn : turn_far;
      return small ? y : far;
    } else if constexpr (FORM != kFar) {
      const float z = FORM == kAny ? s * in : s, u = z * z;
      const float p = FORM == kClose ? fmaf(u, fmaf(u, fmaf(u, c3[2], c3[1]), c3[0]), scale2) : fmaf(u, fmaf(u, fmaf(u, fmaf(u, c[3], c[2]), c[1]), c[0]), scale2);
      const float y = s * p, t = y * icap2;
      turn = fmaf(-t, t, 1.f);
      return y;
    } else {
      const float e = __builtin_amdgcn_exp2f(s * in2), r = __builtin_amdgcn_rcpf(e + 1.f);
      turn = fminf(e, 0x1p100f) * 4.f * r * r;
      return fmaf(-2.f * cap2, r, cap2);
    }
  }
  template <BendForm FORM>
  __device__ __forceinline__ float bent(float s, float dist, float& turn) const {
    return fmaf(-slope2, fabsf(dist), capped<FORM>(s, turn));
  }
};
static inline Bend bend_of(float scale, float cap) {
  Bend b{};
  b.scale2 = scale * WA_LOG2E;
  b.close = b.near = -1.f;
  if (cap > 0.f) {
    const float in = scale / cap, u = usual_cap(scale, cap) ? in * in : 1.f;
    b.in = in;
    b.in2 = 2.f * in * WA_LOG2E;
    b.cap2 = cap * WA_LOG2E;
    b.icap2 = 1.f / b.cap2;
    b.close = 0.3f / in;
    b.near = fminf(0.5f / in, 3.4e38f);
    b.c3[0] = -0x1.55549ep-2f * u * b.scale2;
    b.c3[1] = 0x1.10b012p-3f * u * u * b.scale2;
    b.c3[2] = -0x1.9c99a8p-5f * u * u * u * b.scale2;
    b.c[0] = -0x1.5554d6p-2f * u * b.scale2;
    b.c[1] = 0x1.10e9fcp-3f * u * u * b.scale2;
    b.c[2] = -0x1.b28c5ep-5f * u * u * u * b.scale2;
    b.c[3] = 0x1.1a7b9cp-6f * u * u * u * u * b.scale2;
  }
  return b;
}
template <int N>
__device__ __forceinline__ float largest(const f32x16 (&s)[N]) {
  float x = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) x = fmaxf(x, fabsf(s[i][r]));
  return x;
}
template <BendForm F> struct FormTag { static constexpr BendForm value = F; };
// run(FormTag<form>) of the form for scores of at most `most`
template <Bends BENDS, typename Run>
__device__ __forceinline__ void by_form(const Bend& bend, float most, const Run& run) {
  const BendForm form = bend.form<BENDS>(most);
  if constexpr (BENDS == kOther) {
    if (form == kAny) run(FormTag<kAny>{});
    else run(FormTag<kBoth>{});
  } else {
    if (form == kBias) run(FormTag<kBias>{});
    else if (form == kClose) run(FormTag<kClose>{});
    else if (form == kNear) run(FormTag<kNear>{});
    else run(FormTag<kFar>{});
  }
}
}  // namespace
