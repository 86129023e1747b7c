// Attention of the newest tokens over an 8-bit KV cache (cache8.hip), all of it, a window with sinks, or chosen blocks. No reference counterpart.
#include <algorithm>

#include "codes.h"
#include "ranges.h"
#include "tile.h"

namespace {

// =============================================================================================
// Rows are (query, head of the group) pairs of one key head; a unit of 16 RT rows walks its tiles of 32 keys once. A part of a unit (the
// tiles that one workgroup takes) is shared by four waves, tile by tile, each with running maxima and sums of its own. A wave's codes stream through
// two LDS stages of its own by direct loads, whole rows at a time: a stage is read into registers and filled again, two tiles on, before the tile is
// used, so a CU has 128 KB on their way (one tile ahead in registers, 64 KB, and rows in halves: 283 us against 265 for 32 ragged sequences of up to
// 32,768 tokens, 8 key heads, before they shared the workgroups evenly). Codes become bf16 exactly; a block's scales are wave-uniform factors of
// the scores and of the weights (powers of two: the weights' rounding is that of the plain ones). Products are v_mfma_f32_16x16x32: S^T = K Q^T,
// O^T += V^T P^T; row a = 4 x + y of the former is key 4 y + x of its 16, which puts value rows that are read together in different banks. Bound by
// reading the codes: those 32 sequences take 204 us, 5.3 TB/s.
// =============================================================================================
struct AttendParams {
  const bf16_t* q; int64_t q_sb, q_st, q_sh;
  bf16_t* o; int64_t o_sb, o_st, o_sh;
  float* lse;
  const uint8_t* k; const uint8_t* v;
  const float* k_scale; const float* v_scale;
  const int32_t* kv_len; int64_t kv_len_all, cap;
  const int32_t* index; const int32_t* num; int topk;
  int64_t window, sink;
  const float* slopes;
  int n, H, Hk, nb, shift;        // shift: log2 of a block's tokens
  int units, parts, per;          // row units of (sequence, key head, with lists: query); parts of a unit, tiles of a part
  int even;                       // workgroups of a key head that run at once and share all sequences' tiles evenly, or 0: units are cut
  int B;
  Bend bend;
  float* part;                    // [unit][part] or, evenly, [workgroup][2], [16 RT][D + 2]: maximum, sum, outputs
};

// Tiles of a workgroup, of `all` that workgroups share of which `at_once` run at a time: at least two a wave and as many for each of the four. Beyond
// 64 they come in rounds, up to 8 of them: workgroups that start as others end even out what the memory gives each (32 sequences of 32,760 tokens, 8 key
// heads: 8 rounds of 64 tiles 392 us, two of 256 or one of 512 430; 4 sequences: one round of 64 61 us, 8 rounds of 8 85).
constexpr int64_t kRounds = 8;
// So many neighbouring workgroups take one key head's tiles, then as many the next head's: an XCD, which gets every eighth, works on all
// heads (32 ragged sequences: 204 us; with a head on each XCD 224, with turns of 8 and 64 207 and 208).
constexpr int kTurn = 16;
__host__ __device__ __forceinline__ int share(int64_t all, int64_t at_once) {
  const int64_t rounds = (all + 64 * at_once - 1) / (64 * at_once), n = at_once * (rounds < 1 ? 1 : rounds > kRounds ? kRounds : rounds);
  const int64_t each = (all + n - 1) / n;
  return each < 8 ? 8 : (int)((each + 3) & ~(int64_t)3);
}

constexpr float kLowest = -3.4028234e38f;   // running maximum before the first key: below every score, and no difference of it is NaN
constexpr float kSlack = 8.f;               // log2 of the growth that the running maximum lets pass

__device__ __forceinline__ f32x4 mma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A lane's value combined over the four 16-lane groups.
template <typename Op>
__device__ __forceinline__ float over_groups(float x, const Op& op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int D> struct ValueRow;     // a lane's part of a value row: D / 16 codes
template <> struct ValueRow<128> { typedef u32x2 type; };
template <> struct ValueRow<64> { typedef uint32_t type; };
__device__ __forceinline__ uint32_t word(const u32x2& x, int i) { return x[i]; }
__device__ __forceinline__ uint32_t word(uint32_t x, int) { return x; }

// What a unit is and which tiles its rows see, the same in the walk and in the join.
struct Unit {
  int b, hk, i0, row0, rows, tiles;   // first query (with lists), first row, rows; tiles in all
  int n0, s1;                         // without lists: the first n0 tiles, then those from s1 on
  int64_t len;
  __device__ __forceinline__ void held(const AttendParams& p) {
    const int64_t x = p.kv_len ? (int64_t)p.kv_len[b] : p.kv_len_all;
    len = min(max(x, (int64_t)0), p.cap);
  }
  // Tiles that rows at positions t0 .. t1 see.
  __device__ __forceinline__ void walk(const AttendParams& p, int64_t t0, int64_t t1) {
    const int end = (int)((t1 + 32) >> 5);          // tiles that the last row sees
    if (t1 < 0) {
      tiles = 0;
    } else if (p.window > 0 && t0 - p.window + 1 > 0) {
      n0 = (int)min((int64_t)end, (p.sink + 31) >> 5);
      s1 = max(n0, (int)((t0 - p.window + 1) >> 5));
      tiles = n0 + max(0, end - s1);
    } else {
      tiles = n0 = end;
    }
  }
  // Tiles that a whole sequence's rows see (without lists).
  __device__ __forceinline__ int of_sequence(const AttendParams& p, int sequence) {
    b = sequence;
    held(p);
    walk(p, len - p.n, len - 1);
    return tiles;
  }
  template <int RT>
  __device__ __forceinline__ void init(const AttendParams& p, unsigned u) {
    const int G = p.H / p.Hk;
    const unsigned of = p.index ? (G + 16 * RT - 1) / (16 * RT) : p.units;
    hk = (int)(u % (unsigned)p.Hk);
    u /= (unsigned)p.Hk;
    const int chunk = (int)(u % of);
    u /= of;
    i0 = p.index ? (int)(u % (unsigned)p.n) : 0;
    b = (int)(p.index ? u / (unsigned)p.n : u);
    row0 = 16 * RT * chunk;
    rows = min(16 * RT, (p.index ? G : p.n * G) - row0);
    held(p);
    n0 = s1 = 0;
    if (p.index) tiles = max(0, min(p.num[((int64_t)b * p.n + i0) * p.Hk + hk], p.topk)) << (p.shift - 5);
    else walk(p, len - p.n + row0 / G, len - p.n + (row0 + rows - 1) / G);
  }
  // Query and head (in its group) of row r of the unit.
  __device__ __forceinline__ int query(const AttendParams& p, int r) const { return p.index ? i0 : (row0 + r) / (p.H / p.Hk); }
  __device__ __forceinline__ int head(const AttendParams& p, int r) const {
    const int G = p.H / p.Hk;
    return hk * G + (p.index ? row0 + r : (row0 + r) % G);
  }
};

__device__ __forceinline__ void write_row(const AttendParams& p, int b, int i, int h, int d, float sum, float top, float l) {
  p.o[(int64_t)b * p.o_sb + (int64_t)i * p.o_st + (int64_t)h * p.o_sh + d] = (bf16_t)(l == 0.f ? 0.f : sum / l);
  if (d == 0) p.lse[((int64_t)b * p.H + h) * p.n + i] = l == 0.f ? -INFINITY : (top + log2f(l)) * WA_LN2;
}

template <typename Code, int D, int RT, Bends BENDS>
__global__ void __launch_bounds__(256, 2) attend_kernel(AttendParams p) {
  constexpr int NW = 4, KC = D / 32, VC = D / 16, KL = D / 64;   // key products of a tile half; channels of a value row a lane holds; loads of a key row
  typedef typename ValueRow<D>::type VRow;
  static_assert(NW * 4 * 32 * D >= NW * 16 * (D + 4) * 4, "the waves' outputs fit their drained rings");
  __shared__ __attribute__((aligned(1024))) char lds[NW * 4 * 32 * D];   // of each wave two stages of keys and values; then the waves' outputs
  __shared__ float sm[NW][16], sl[NW][16];
  __shared__ int s_wave[NW], s_end[256], s_seq;   // where each sequence's tiles end
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, kg = lane >> 4;
  unsigned u;
  int64_t slot;
  int t0, t1, head = 0, turn = 0, upto = 0, seq = 0;   // upto: where this workgroup's tiles end among those of all sequences
  if (p.even) {
    // Where this workgroup's tiles begin: a sequence a lane, their tiles summed over the workgroup.
    Unit x;
    const int mine = tid < p.B ? x.of_sequence(p, tid) : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int below = __shfl_up(sum, d, 64);
      if (lane >= d) sum += below;
    }
    if (lane == 63) s_wave[w] = sum;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      if (y < w) sum += s_wave[y];
      all += s_wave[y];
    }
    const int per = share(all, p.even);
    const unsigned next = blockIdx.x / kTurn;
    head = (int)(next % (unsigned)p.Hk);
    turn = (int)(next / (unsigned)p.Hk * kTurn + blockIdx.x % kTurn);
    const int64_t at = (int64_t)turn * per;
    if (at >= all) return;
    const int begin = (int)at;
    s_end[tid] = sum;
    if (begin < sum && begin >= sum - mine) s_seq = tid;
    __syncthreads();
    seq = __builtin_amdgcn_readfirstlane(s_seq);
    upto = (int)min(at + per, (int64_t)all);
    t0 = begin - (seq ? s_end[seq - 1] : 0);
  } else {
    u = blockIdx.x / p.parts;
    t0 = (int)(blockIdx.x % p.parts) * p.per;
  }
  for (bool more = true; more;) {
  Unit unit;
  bool alone;
  if (p.even) {
    u = (unsigned)seq * p.Hk + head;
    unit.init<RT>(p, u);
    unit.tiles = __builtin_amdgcn_readfirstlane(unit.tiles);
    const int before = __builtin_amdgcn_readfirstlane(seq ? s_end[seq - 1] : 0);
    t0 = __builtin_amdgcn_readfirstlane(t0);
    t1 = min(unit.tiles, upto - before);
    alone = t0 == 0 && t1 == unit.tiles;
    slot = 2 * ((int64_t)turn * p.Hk + head) + (t0 == 0);   // one sequence at most began before this workgroup's tiles, and one that begins there goes on behind
  } else {
    unit.init<RT>(p, u);
    unit.tiles = __builtin_amdgcn_readfirstlane(unit.tiles);
    t1 = min(unit.tiles, t0 + p.per);
    if (t0 >= t1 && t0 > 0) return;
    alone = unit.tiles <= p.per;
    slot = blockIdx.x;
  }
  const int b = unit.b, hk = unit.hk, window = (int)p.window, sink = (int)p.sink;

  bf16x8 q[RT][KC];
  int pos[RT], from[RT];   // the row's position: the last key that it sees; the first one of its window
  float slope2[RT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int r = 16 * x + l16;
    const bool ok = r < unit.rows;
    const int i = unit.query(p, ok ? r : 0), h = unit.head(p, ok ? r : 0);
    pos[x] = ok ? (int)(unit.len - p.n + i) : -1;
    from[x] = window > 0 ? pos[x] - window + 1 : INT32_MIN;
    slope2[x] = p.slopes ? p.slopes[h] * WA_LOG2E : 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {   // channels in the order in which the keys' come
      q[x][c] = bf16x8{};
      if (ok) q[x][c] = *(const bf16x8*)(p.q + (int64_t)b * p.q_sb + (int64_t)i * p.q_st + (int64_t)h * p.q_sh + 64 * (c >> 1) + 16 * kg + 8 * (c & 1));
    }
  }
  const int st = p.Hk * D;   // at most 2^23
  const uint8_t* kb = p.k + ((int64_t)b * p.cap * p.Hk + hk) * D;
  const uint8_t* vb = p.v + ((int64_t)b * p.cap * p.Hk + hk) * D;
  const float* ksc = p.k_scale + ((int64_t)b * p.Hk + hk) * p.nb;
  const float* vsc = p.v_scale + ((int64_t)b * p.Hk + hk) * p.nb;
  const int32_t* list = p.index ? p.index + (((int64_t)b * p.n + unit.i0) * p.Hk + hk) * p.topk : nullptr;
  const int last = p.index ? (int)(unit.len - p.n + unit.i0) : (int)(unit.len - p.n + (unit.row0 + unit.rows - 1) / (p.H / p.Hk));   // last key that any row sees
  const int lowest = p.index ? last : (int)(unit.len - p.n + unit.row0 / (p.H / p.Hk));                                              // ... that every row sees

  float m[RT], l[RT];
  f32x4 o[RT][VC];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    m[x] = kLowest;
    l[x] = 0.f;
#pragma unroll
    for (int j = 0; j < VC; ++j) o[x][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Ids of this wave's next 64 tiles sit in its lanes.
  int ids = 0, ids_at = t1;
  auto key_of = [&](int t) -> int {   // the tile's first key, -1 if none of its tokens is seen
    if (!p.index) return (t < unit.n0 ? t : unit.s1 + t - unit.n0) * 32;
    if (t >= ids_at + 64 * NW || t < ids_at) {
      ids_at = t;
      const int mine = t + lane * NW;
      ids = mine < t1 ? list[mine >> (p.shift - 5)] : -1;
    }
    const int id = __builtin_amdgcn_readlane(ids, (t - ids_at) / NW);
    const int64_t key = ((int64_t)id << p.shift) + (t & ((1 << (p.shift - 5)) - 1)) * 32;
    return id < 0 || key > last ? -1 : (int)key;
  };
  // A tile's codes in LDS: 16-byte chunk c of row r in slot c ^ swizzle(r). Direct load i fills rows i RPL .. + RPL.
  constexpr int CPR = D / 16, RPL = 64 / CPR, LOADS = 32 / RPL, HALF = 32 * D;
  auto swizzle = [](int r) { return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3; };
  char* const ring = lds + w * 4 * HALF;
  int off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int r = i * RPL + lane / CPR;
    off[i] = r * st + ((lane % CPR) ^ swizzle(r)) * 16;
  }
  const int ky = (l16 & 3) * 4 + (l16 >> 2);   // the key of operand row l16
  struct Tile {
    float ks, vs;
    int key;
  };
  int next = t0 + w;
  auto issue = [&](Tile& x, int stage) {   // the wave's next tile with seen tokens
    x.key = -1;
    while (next < t1 && (x.key = key_of(next)) < 0) next += NW;
    next += NW;
    if (x.key < 0) return;
    // from the last token that any row sees on the codes read as zeros
    const int bytes = (min(32, last + 1 - x.key) - 1) * st + D;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kb + (int64_t)x.key * st), (short)0, bytes, WA_BUF_DWORD3);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vb + (int64_t)x.key * st), (short)0, bytes, WA_BUF_DWORD3);
    char* const to = ring + stage * 2 * HALF;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) lds_dma16(kr, to + i * 1024, off[i]);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) lds_dma16(vr, to + HALF + i * 1024, off[i]);
    x.ks = ksc[x.key >> p.shift];
    x.vs = vsc[x.key >> p.shift];
  };
  // Tile x of `stage`, with tile y behind it on its way: x's place is taken by the tile after y.
  auto use = [&](Tile& x0, const Tile& y0, int stage) {
    const Tile x = x0;
    if (y0.key >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const char* at = ring + stage * 2 * HALF;
    u32x4 kc[2][KL];
    VRow vc[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < KL; ++c) kc[h][c] = *(const u32x4*)(at + (16 * h + ky) * D + ((4 * c + kg) ^ swizzle(ky)) * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = 16 * (e >> 2) + 4 * (e & 3) + kg;
      vc[e] = *(const VRow*)(at + HALF + r * D + (((VC * l16) >> 4) ^ swizzle(r)) * 16 + ((VC * l16) & 15));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < KL; ++c) asm volatile("" : "+v"(kc[h][c]));
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(vc[e]));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before it is filled again
    issue(x0, stage);
    // the halves' keys one after the other: what is converted is used at once
    f32x4 scores[RT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int y = 0; y < RT; ++y) scores[y][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        u32x4 k;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t lo, hi;
          Code::pairs(kc[h][c >> 1][2 * (c & 1) + e], lo, hi);
          k[2 * e] = lo;
          k[2 * e + 1] = hi;
        }
#pragma unroll
        for (int y = 0; y < RT; ++y) scores[y][h] = mma16(__builtin_bit_cast(bf16x8, k), q[y][c], scores[y][h]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool whole = x.key + 31 <= lowest && ((window == 0) | (x.key > last - window) | (x.key + 31 < sink));
    bf16x8 pr[RT];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      const f32x4(&acc)[2] = scores[y];
      float s[8];
      const int key0 = x.key + kg;
      if (p.bend.cap2 > 0.f || p.slopes) {
        Bend bend = p.bend;
        bend.slope2 = slope2[y];
        const float far = (float)(pos[y] - key0);
        float most = 0.f, unused;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[e] = acc[e >> 2][e & 3] * x.ks;
          most = fmaxf(most, fabsf(s[e]));
        }
        by_form<BENDS>(bend, most, [&](auto form) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] = bend.bent<decltype(form)::value>(s[e], far - (float)(16 * (e >> 2) + 4 * (e & 3)), unused);
        });
      } else {
        const float by = p.bend.scale2 * x.ks;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = acc[e >> 2][e & 3] * by;
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // one comparison beside the other: as a chain of branches the window's was compiled to nothing
          const int key = key0 + 16 * (e >> 2) + 4 * (e & 3);
          const bool seen = (key <= pos[y]) & ((key >= from[y]) | (key < sink));
          s[e] = seen ? s[e] : -INFINITY;
        }
      }
      const float top = over_groups(fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))),
                                    [](float a, float c) { return fmaxf(a, c); });
      // the running maximum follows only when a score is 2^kSlack above it: weights of up to 2^kSlack are as exact
      if (__any(top > m[y] + kSlack)) {
        const float up = fmaxf(m[y], top), f = __builtin_amdgcn_exp2f(m[y] - up);
        m[y] = up;
        l[y] *= f;
#pragma unroll
        for (int j = 0; j < VC; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[y][j][r] *= f;
      }
      // weights times the values' scale round to bf16 for their product with the codes; the sum that divides them is of the unrounded ones
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = __builtin_amdgcn_exp2f(s[e] - m[y]);
        pr[y][e] = (bf16_t)(s[e] == -INFINITY ? 0.f : z * x.vs);   // a scale of NaN reaches only rows that see its block
        l[y] += z;
      }
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      uint32_t rows[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) rows[e] = word(vc[e], j / 4);
      const u32x4 vt = Code::column(rows, j % 4);   // channel j of the eight rows
#pragma unroll
      for (int y = 0; y < RT; ++y) o[y][j] = mma16(__builtin_bit_cast(bf16x8, vt), pr[y], o[y][j]);
      if (j % 2) __builtin_amdgcn_sched_barrier(0);
    }
  };
  {
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
      for (int c = 0; c < KC; ++c) asm volatile("" : "+v"(q[x][c]));   // here before the first tiles are asked for
    Tile a, c;
    issue(a, 0);
    issue(c, 1);
    while (a.key >= 0) {
      use(a, c, 0);
      if (c.key < 0) break;
      use(c, a, 1);
    }
  }
  float(*so)[16][D + 4] = (float(*)[16][D + 4])lds;
  // The waves' parts: each to the common maximum, then summed in wave order. Channel VC (4 kg + r) + j of row l16 is register r of
  // accumulator j.
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const float lw = over_groups(l[x], [](float a, float c) { return a + c; });
    if (x > 0) __syncthreads();
    if (kg == 0) {
      sm[w][l16] = m[x];
      sl[w][l16] = lw;
    }
    __syncthreads();
    auto highest = [&](int r) { return fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r])); };
    const float f = __builtin_amdgcn_exp2f(m[x] - highest(l16));
#pragma unroll
    for (int j = 0; j < VC; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[w][l16][VC * (4 * kg + r) + j] = o[x][j][r] * f;
    __syncthreads();
    const int rows = min(16, unit.rows - 16 * x);
    for (int y = tid; y < rows * D; y += 256) {
      const int r = y / D, d = y % D;
      const float top = highest(r);
      float sum = 0.f, all = 0.f;
#pragma unroll
      for (int z = 0; z < NW; ++z) {
        sum += so[z][r][d];
        all += sl[z][r] * __builtin_amdgcn_exp2f(sm[z][r] - top);
      }
      if (alone) {
        write_row(p, b, unit.query(p, 16 * x + r), unit.head(p, 16 * x + r), d, sum, top, all);
      } else {
        float* at = p.part + (slot * 16 * RT + 16 * x + r) * (D + 2);
        at[2 + d] = sum;
        if (d == 0) {
          at[0] = top;
          at[1] = all;
        }
      }
    }
  }
  more = false;
  if (p.even && t1 == unit.tiles) {   // on to the next sequence that sees a token
    const int at = s_end[seq];
    while (seq + 1 < p.B && s_end[seq + 1] == at) ++seq;
    ++seq;
    t0 = 0;
    more = at < upto;
    __syncthreads();   // the outputs' places are the rings'
  }
  }
}

// The parts of units that have several, in their order: one wave per row.
template <int D, int RT>
__global__ void __launch_bounds__(256) join_kernel(AttendParams p, unsigned units) {
  const int lane = threadIdx.x & 63;
  const unsigned x = blockIdx.x * 4 + (threadIdx.x >> 6), u = x / (16 * RT);
  const int r = (int)(x % (16 * RT));
  if (u >= units) return;
  Unit unit;
  unit.init<RT>(p, u);
  if (r >= unit.rows) return;
  int n;
  int64_t first, step, second;   // the parts' places: first, then second + step s
  if (p.even) {
    int before = 0, all = 0;
    for (int y = lane; y < p.B; y += 64) {
      Unit other;
      const int tiles = other.of_sequence(p, y);
      all += tiles;
      before += y < unit.b ? tiles : 0;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      before += __shfl_xor(before, d, 64);
      all += __shfl_xor(all, d, 64);
    }
    const int per = share(all, p.even), from = before / per;
    n = unit.tiles ? (before + unit.tiles - 1) / per - from + 1 : 0;
    if (n == 1) return;
    first = 2 * ((int64_t)from * p.Hk + unit.hk) + 1;
    step = 2 * p.Hk;
    second = first - 1;
  } else {
    if (unit.tiles <= p.per) return;
    n = (unit.tiles + p.per - 1) / p.per;
    first = second = (int64_t)u * p.parts;
    step = 1;
  }
  auto place = [&](int s) { return p.part + ((s ? second + step * s : first) * 16 * RT + r) * (D + 2); };
  float top = kLowest;
  for (int s = lane; s < n; s += 64) top = fmaxf(top, place(s)[0]);
  top = wa_wave_max(top);
  float l = 0.f, o[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float* at = place(s);
    const float f = __builtin_amdgcn_exp2f(at[0] - top);
    l += at[1] * f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] += at[2 + lane + 64 * e] * f;
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e) write_row(p, unit.b, unit.query(p, r), unit.head(p, r), lane + 64 * e, o[e], top, l);
}

// How a call is cut: row tiles of a unit, units, tiles of a part and parts.
struct Cut {
  int rt, units_of;
  int64_t units;
  int per, parts;      // tiles of a part, parts of a unit; or,
  int even;            // with sequences cut evenly, workgroups of a key head at once
  int64_t most, heads; // and in all at most
  int64_t grid() const { return even ? most * heads : units * parts; }
  int64_t slots() const { return even ? 2 * grid() : parts > 1 ? units * parts : 0; }
};

bool sized(const wa_kv8_attend_args& a) {
  const wa_cache8& c = a.cache;
  return c.B >= 1 && a.n >= 1 && c.cap >= 1 && c.cap <= 1 << 30 && c.Hk >= 1 && a.H >= c.Hk && a.H % c.Hk == 0 && a.H <= 65536 && a.n <= 1 << 24 &&
         a.n * (a.H / c.Hk) <= INT32_MAX && c.B <= INT32_MAX / c.Hk &&
         (a.index ? a.n * ((a.H / c.Hk + 15) / 16) : (a.n * (a.H / c.Hk) + 15) / 16) <= INT32_MAX / (c.B * c.Hk) && a.window >= 0 && a.sink >= 0 &&
         (!a.index || (a.topk >= 1 && a.topk <= WA_SELECT_MAX_BLOCKS && a.window == 0));
}

Cut cut(const wa_kv8_attend_args& a) {
  Cut c;
  const int64_t G = a.H / a.cache.Hk, rows = a.index ? G : a.n * G;
  // 64 rows of a unit take 256 registers at D = 64; at D = 128 they would leave one wave a SIMD (8 sequences of 32,000 tokens, 64 rows of 8 key heads:
  // two units of 32 rows 197 us, one of 64 283)
  c.rt = rows <= 16 ? 1 : rows <= 32 || a.cache.D == 128 ? 2 : 4;
  const int64_t of = (rows + 16 * c.rt - 1) / (16 * c.rt);
  c.units_of = (int)of;
  c.units = a.cache.B * a.cache.Hk * of * (a.index ? a.n : 1);
  const int64_t tokens = a.kv_len ? a.cache.cap : std::min(std::max<int64_t>(a.kv_len_all, 0), a.cache.cap);
  // at most: the sinks', and from the first row's window to the last row, each run with a partial tile at either end
  const int64_t seen = a.window > 0 ? std::min(tokens, std::min(a.sink, tokens) + std::min(a.window, tokens) + a.n + 128) : tokens;
  const int64_t tiles = a.index ? a.topk * (a.cache.block_size / 32) : (seen + 31) / 32;
  // workgroups that run at once: what the kernels' registers leave of four a CU (D = 64) or, with their codes' stages, two
  const int64_t at_once = a.cache.D == 128 ? 512 : c.rt == 1 ? 1024 : c.rt == 2 ? 768 : 512;
  c.per = (int)std::min<int64_t>(share(c.units * tiles, at_once), std::max<int64_t>(8, tiles));
  c.parts = (int)std::max<int64_t>(1, (tiles + c.per - 1) / c.per);
  // Sequences of lengths that only the GPU knows, or, whatever the lengths, more tiles than one round takes: cut along all sequences, so that workgroups bring as much each
  // (32 ragged ones of up to 32,768 tokens, 8 key heads of 128: 204 us; cut by the cache's length into parts of 64 tiles 268. 32 of 30,000 and heads
  // of 64: 251 and 311; 16 of 4,000, less than a round: 27 and 23).
  c.heads = a.cache.Hk;
  const bool along = (a.kv_len || c.units * tiles > 64 * at_once) && !a.index && of == 1 && a.cache.B > 1 && a.cache.B <= 256 && c.heads <= at_once;
  c.even = along && a.cache.B * tiles <= INT32_MAX ? (int)(at_once / c.heads) : 0;
  c.most = (std::min<int64_t>(kRounds * c.even, a.cache.B * tiles / 64 + c.even) + kTurn - 1) / kTurn * kTurn;
  return c;
}

template <typename Code, int D, Bends BENDS>
void launch(const AttendParams& p, const Cut& c, hipStream_t s) {
  const dim3 grid((unsigned)c.grid()), block(256);
  const dim3 rows((unsigned)((c.units * 16 * c.rt + 3) / 4));
  if (c.rt == 1) hipLaunchKernelGGL((attend_kernel<Code, D, 1, BENDS>), grid, block, 0, s, p);
  else if (c.rt == 2) hipLaunchKernelGGL((attend_kernel<Code, D, 2, BENDS>), grid, block, 0, s, p);
  else if constexpr (D == 64) hipLaunchKernelGGL((attend_kernel<Code, D, 4, BENDS>), grid, block, 0, s, p);
  if (!c.slots()) return;
  if (c.rt == 1) hipLaunchKernelGGL((join_kernel<D, 1>), rows, block, 0, s, p, (unsigned)c.units);
  else if (c.rt == 2) hipLaunchKernelGGL((join_kernel<D, 2>), rows, block, 0, s, p, (unsigned)c.units);
  else if constexpr (D == 64) hipLaunchKernelGGL((join_kernel<D, 4>), rows, block, 0, s, p, (unsigned)c.units);
}

template <typename Code>
void launch(const AttendParams& p, const Cut& c, bool other, int64_t D, hipStream_t s) {
  if (D == 128 && other) launch<Code, 128, kOther>(p, c, s);
  else if (D == 128) launch<Code, 128, kUsual>(p, c, s);
  else if (other) launch<Code, 64, kOther>(p, c, s);
  else launch<Code, 64, kUsual>(p, c, s);
}

}  // namespace

extern "C" int64_t wa_kv8_attend_workspace_bytes(const wa_kv8_attend_args* a) {
  if (!a || !sized(*a)) return 0;
  const Cut c = cut(*a);
  return c.slots() * 16 * c.rt * (a->cache.D + 2) * 4;
}

extern "C" int wa_kv8_attend(const wa_kv8_attend_args* a, void* stream) {
  WA_CHECK_ARG(a, "kv8_attend: null args");
  const wa_cache8& c = a->cache;
  WA_CHECK_ARG(c.D == 64 || c.D == 128, "kv8_attend: head dim must be 64 or 128, got %lld", (long long)c.D);
  WA_CHECK_ARG(c.block_size == 64 || c.block_size == 128, "kv8_attend: block size must be 64 or 128, got %lld", (long long)c.block_size);
  WA_CHECK_ARG(c.code == WA_CODE_INT8 || c.code == WA_CODE_E4M3, "kv8_attend: unknown code %d", c.code);
  WA_CHECK_ARG(sized(*a), "kv8_attend: bad sizes B %lld n %lld cap %lld heads %lld / %lld window %lld sink %lld, or lists that are not of 1 .. %d ids without a window",
               (long long)c.B, (long long)a->n, (long long)c.cap, (long long)a->H, (long long)c.Hk, (long long)a->window, (long long)a->sink, WA_SELECT_MAX_BLOCKS);
  WA_CHECK_ARG(c.k && c.v && c.k_scale && c.v_scale && wa_aligned16(c.k) && wa_aligned16(c.v) && a->q && a->o && a->lse, "kv8_attend: null or misaligned tensor");
  WA_CHECK_ARG(!a->index == !a->num, "kv8_attend: lists need counts");
  auto rows16 = [](const void* x, int64_t sb, int64_t st, int64_t sh) {
    return wa_aligned16(x) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
  };
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh) && rows16(a->o, a->o_sb, a->o_st, a->o_sh), "kv8_attend: rows must be 16-byte aligned");
  WA_CHECK_ARG(a->scale >= 0.f && a->scale < INFINITY && (a->cap == 0.f || (a->cap >= 1e-6f && a->cap <= 1e6f && a->scale <= 1e30f)),
               "kv8_attend: scale must be finite and not below 0, cap 0 or 1e-6 .. 1e6 (with a scale of at most 1e30)");
  const Cut k = cut(*a);
  WA_CHECK_ARG(k.grid() <= INT32_MAX && k.units * k.parts <= INT32_MAX && k.units * 16 * k.rt <= INT32_MAX, "kv8_attend: too many rows");
  WA_CHECK_ARG(!k.slots() || a->workspace, "kv8_attend: a launch of %d parts needs a workspace", k.parts);
  AttendParams p{};
  p.q = (const bf16_t*)a->q; p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.o = (bf16_t*)a->o; p.o_sb = a->o_sb; p.o_st = a->o_st; p.o_sh = a->o_sh;
  p.lse = a->lse;
  p.k = (const uint8_t*)c.k; p.v = (const uint8_t*)c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
  p.kv_len = a->kv_len; p.kv_len_all = a->kv_len_all; p.cap = c.cap;
  p.index = a->index; p.num = a->num; p.topk = (int)a->topk;
  p.window = std::min(a->window, (int64_t)1 << 30); p.sink = std::min(a->sink, (int64_t)1 << 30);
  p.slopes = a->slopes;
  p.n = (int)a->n; p.H = (int)a->H; p.Hk = (int)c.Hk;
  p.nb = (int)((c.cap + c.block_size - 1) / c.block_size); p.shift = c.block_size == 64 ? 6 : 7;
  p.units = k.units_of; p.parts = k.parts; p.per = k.per; p.even = k.even; p.B = (int)c.B;
  const float scale = a->scale == 0.f ? 1.f / sqrtf((float)c.D) : a->scale;
  p.bend = bend_of(scale, a->cap);
  p.part = (float*)a->workspace;
  hipStream_t s = (hipStream_t)stream;
  const bool other = bends_of(scale, a->cap, a->slopes) == kOther;
  if (c.code == WA_CODE_INT8) launch<Int8>(p, k, other, c.D, s);
  else launch<E4m3>(p, k, other, c.D, s);
  return wa_launch_status("kv8_attend");
}
