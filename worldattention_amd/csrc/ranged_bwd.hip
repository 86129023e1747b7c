// Gradients of the ranged attention (ranged.hip). With P = exp(s - lse), dP = dO V^T and delta = rowsum(O dO) - dlse,
//   dS = P (dP - delta),  dslope = -sum dS |t - j|,  dx = dS (1 - tanh^2),
//   dQ = scale dx K,  dK = scale dx^T Q,  dV = P^T dO   (a shared key head: summed over its query heads).
// Two launches: dQ (with the rows' statistics, and the slopes' gradients in parts), then dK and dV; one more adds up the slopes' parts, and one
// those of dK and dV where their steps are cut. Each of the two forms the scores (dQ twice where a row tile has few steps); that costs two
// products more than forming them once for both, and needs neither atomics nor partial sums of dQ in memory.
#include <algorithm>
#include <type_traits>

#include "ranges.h"
#include "tile.h"

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// dS is carried with this factor: the weights go from one wave to another as fp16 (11 significant bits), and 2^12 keeps weights down to
// 2^-26 among its normal numbers (smaller ones are off by up to 2^-37). It is taken out where the gradients are written.
constexpr float kLift = 4096.f;

// Steps of 128 rows up to which dQ's launch walks them twice, at first for delta alone: rows that see few keys, whose dQ the output's delta leaves
// 2.6e-3 off (of norms, short windows; 2.3e-3 so). Two sequences of 333 tokens: 25 us, 20 in one walk; no difference at thousands of tokens.
constexpr int kFewSteps = 4;

struct BwdParams {
  const bf16_t* q; int64_t q_sb, q_st, q_sh;
  const bf16_t* k; int64_t k_sb, k_st, k_sh;
  const bf16_t* v; int64_t v_sb, v_st, v_sh;
  const bf16_t* o; int64_t o_sb, o_st, o_sh;
  const bf16_t* dout; int64_t d_sb, d_st, d_sh;
  const float* lse; const float* dlse;
  Ranges ranges;
  const float* slopes;
  int B, H, Hk;
  float scale;
  Bend bend;
  bf16_t* dq; bf16_t* dk; bf16_t* dv; float* dslopes;
  // workspace
  float* lse2;    // [B, H, Lq] log-sum-exp in units of log2; +inf where a row sees nothing: its weights come out 0
  float* on;      // [B, H, Lq] 1, or 0 where a row sees a single key: its weight is 1 whatever the score, and its dS exactly 0
  float* delta;   // [B, H, Lq] delta * on; from the output for dQ, which puts it right for dK
  float* slope_part;   // [H][B * q tiles]
  float* part_kv;      // [parts][dK, dV][B, Lk, Hk, D] fp32, with parts > 1
  int parts;
};

// A tile of 64 rows streamed into LDS by direct loads (tile.h's layout): rows from `rows` on read as zeros.
template <int D, int NW>
struct RowTile {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, NI = 64 / (RPI * NW);
  int off[NI];
  __device__ __forceinline__ void init(int64_t st, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = (i * NW + w) * RPI + lane / CPR, pos = lane % CPR;
      off[i] = ((int)(row * st) + (pos ^ dual_swizzle<D>(row)) * 8) * 2;
    }
  }
  __device__ __forceinline__ void issue(bf16_t* lds, const bf16_t* first, int64_t st, int rows, int w) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)first, (short)0, rows > 0 ? (int)((min(rows, 64) - 1) * st + D) * 2 : 0, WA_BUF_DWORD3);
#pragma unroll
    for (int i = 0; i < NI; ++i) lds_dma16(rs, lds + (i * NW + w) * RPI * D, off[i]);
  }
};

// A lane's operands in a 64-row tile whose LDS address is a multiple of its size: rows l32 + 32 x, chunk 2 c + g (tile.h's tile_row8), and
// transposed, rows of 16 c at columns 32 tt + l32 (tile_tr8). With the swizzle's exclusive ors a lane needs one address of either kind: what c and tt
// turn are bits of it, what x and 16 c rows add is a constant (an address for each operand cost registers that the products' operands need).
typedef __attribute__((address_space(3))) const bf16x8 lds_bf16x8;
typedef __attribute__((address_space(3))) wa_s16x4 lds_s16x4;
template <int D>
struct TileReads {
  uint32_t row, col;
  __device__ __forceinline__ void init(int lane) {
    const int l32 = lane & 31, g = lane >> 5, G = lane >> 4, r = (lane & 15) >> 2, q = lane & 3, i = 4 * (G >> 1) + r, at = 16 * (G & 1) + 4 * q;
    row = (uint32_t)(l32 * D + (g ^ dual_swizzle<D>(l32)) * 8) * 2;
    col = (uint32_t)(i * D + ((at >> 3) ^ dual_swizzle<D>(i)) * 8 + (at & 7)) * 2;
  }
  __device__ __forceinline__ static uint32_t address(const bf16_t* tile) { return (uint32_t)(size_t)WA_LDS_PTR(tile); }
  __device__ __forceinline__ bf16x8 row8(uint32_t tile, int c, int x) const { return *(lds_bf16x8*)(size_t)(((tile | row) ^ 32 * c) + 64 * D * x); }
  __device__ __forceinline__ bf16x8 tr8(uint32_t tile, int c, int tt) const {
    bf16x8 a;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {   // eight rows on, whose swizzle differs in the lowest bit
      const uint32_t at = ((tile | col) ^ (64 * tt) ^ (hf ? 16 * D + 16 : 0)) + 32 * D * c;
      const bf16x4 b = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(size_t)at));
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * hf + e] = b[e];
    }
    return a;
  }
};

// Products whose operands are read from LDS two at a time and kAhead pairs ahead: left to itself the compiler waits for each read right behind it.
constexpr int kAhead = 1;
typedef bf16x8 Operands[kAhead + 1][2];
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// acc[x] = rows 32 x .. of the tile times b^T. `first` reads the first operands.
template <int D>
struct RowsProduct {
  static constexpr int N = D / 16;   // pairs: of one chunk c
  __device__ __forceinline__ static void read(const TileReads<D>& rd, uint32_t lds, Operands& a, int i) {
#pragma unroll
    for (int y = 0; y < 2; ++y) a[i % (kAhead + 1)][y] = rd.row8(lds, i, y);
  }
  __device__ __forceinline__ static void first(const TileReads<D>& rd, uint32_t lds, Operands& a) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(rd, lds, a, i);
  }
  __device__ __forceinline__ static void run(const TileReads<D>& rd, uint32_t lds, const bf16x8 (&b)[D / 16], f32x16 (&acc)[2], Operands& a) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + kAhead < N) read(rd, lds, a, i + kAhead);
      in_order();
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[y] = wa_mfma32(a[i % (kAhead + 1)][y], b[i], i == 0 ? f32x16{} : acc[y]);
      in_order();
    }
  }
};
// acc[tt] += (the tile's columns 32 tt ..)^T times b, over the tile's 64 rows.
template <int D>
struct ColsProduct {
  static constexpr int DT = D / 32, N = 2 * DT;
  __device__ __forceinline__ static void read(const TileReads<D>& rd, uint32_t lds, Operands& a, int i) {
#pragma unroll
    for (int y = 0; y < 2; ++y) a[i % (kAhead + 1)][y] = rd.tr8(lds, (2 * i + y) / DT, (2 * i + y) % DT);
  }
  __device__ __forceinline__ static void first(const TileReads<D>& rd, uint32_t lds, Operands& a) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(rd, lds, a, i);
  }
  // B: one operand, or one and what its rounding left of it.
  template <int B>
  __device__ __forceinline__ static void run(const TileReads<D>& rd, uint32_t lds, const bf16x8 (&b)[B][4], f32x16 (&acc)[DT], Operands& a) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + kAhead < N) read(rd, lds, a, i + kAhead);
      in_order();
#pragma unroll
      for (int z = 0; z < B; ++z)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[(2 * i + y) % DT] = wa_mfma32(a[i % (kAhead + 1)][y], b[z][(2 * i + y) / DT], acc[(2 * i + y) % DT]);
      in_order();
    }
  }
};

// a b, and 0 where either is 0, whatever the other.
__device__ __forceinline__ float zero_mul(float a, float b) {
  float x;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(x) : "v"(a), "v"(b));
  return x;
}

// Four values as bf16 into places 4 x .. of an operand.
__device__ __forceinline__ void put4(bf16x8& a, int x, const float (&f)[4]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16x2 p = __builtin_convertvector(f32x2{f[2 * i], f[2 * i + 1]}, bf16x2);
    a[4 * x + 2 * i] = p[0];
    a[4 * x + 2 * i + 1] = p[1];
  }
}

// Top of a step: this wave's tile loads have landed and its LDS reads returned, then the workgroup's.
__device__ __forceinline__ void step_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---------------------------------------------------------------------------------------------
// dQ: one workgroup of four waves per 128 rows of a head over the 64-key steps that they see; K and V through two LDS stages each, a row
// a lane. delta comes from the output, whose weights and self are rounded to bf16, and is off by 2^-9 / sqrt(keys that count); the rows' sums of
// dS, which delta makes the log-sum-exp's gradient, tell by how much: delta is put right for the launch behind, which forms dK, and for the
// slopes' gradients (SLOPES: sums of dS dist and P dist besides). dQ itself takes dS in two bf16 parts, of 16 bits together, so that
// its only other rounding is its own: one product in four more. Rows of few keys: 2.8e-3 from the exact dQ and dK with one part and the
// output's delta, 2.4e-3 so (of norms; 1.7e-3 is the results' rounding). 4,680 tokens in 3 frames, 12 heads of 128: dQ 230 us (one
// part 187); packed documents of 8,190 tokens in all, 16 heads, capped: 152 us (134). A second part only where a weight is above 1/8 cost more
// in registers than it saved.
// ---------------------------------------------------------------------------------------------
template <int D, Bends BENT, bool SLOPES>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) ranged_dq_kernel(BwdParams p) {
  constexpr int NW = 4, DC = D / 16, DT = D / 32, TILE = 64 * D;
  using RT = RowTile<D, NW>;
  __shared__ __attribute__((aligned(2 * TILE))) bf16_t kv0[2 * TILE];
  __shared__ __attribute__((aligned(2 * TILE))) bf16_t kv1[2 * TILE];
  __shared__ float s_part[NW];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  const int per = p.H / p.Hk, nbh = p.B * p.Hk, nq = (p.ranges.Lq + 127) / 128;
  int u = (int)blockIdx.x;
  const int bh = u % nbh;
  u /= nbh;
  const int h = (bh % p.Hk) * per + u % per, b = bh / p.Hk, qt = p.ranges.row_tile(b, u / per);
  Steps st;
  st.init(p.ranges, b, 2 * qt, 2);
  const int qi = qt * 128 + w * 32 + l32;
  const bool q_ok = qi < p.ranges.Lq;
  const int row = q_ok ? qi : 0;
  int4 runs = p.ranges.row(b, row);
  if (!q_ok) runs = int4{0, 0, 0, 0};
  bf16x8 qf[DC], dof[DC];
  float dl = 0.f;
  {
    const bf16_t* qr = p.q + (int64_t)b * p.q_sb + (int64_t)h * p.q_sh + (int64_t)row * p.q_st;
    const bf16_t* dr = p.dout + (int64_t)b * p.d_sb + (int64_t)h * p.d_sh + (int64_t)row * p.d_st;
    const bf16_t* orow = p.o + (int64_t)b * p.o_sb + (int64_t)h * p.o_sh + (int64_t)row * p.o_st;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const bf16x8 a = *(const bf16x8*)(qr + c * 16 + g * 8);
      const bf16x8 d = *(const bf16x8*)(dr + c * 16 + g * 8);
      const bf16x8 o = *(const bf16x8*)(orow + c * 16 + g * 8);
      qf[c] = q_ok ? a : bf16x8{};
      dof[c] = q_ok ? d : bf16x8{};
#pragma unroll
      for (int e = 0; e < 8; ++e) dl = fmaf((float)o[e], (float)d[e], dl);
    }
  }
  dl += __shfl_xor(dl, 32, 64);
  // The row's statistics, for the launch behind too: weights of a row that sees nothing come out 0, and of one that sees a single key 1 whatever
  // its score, so that its dS is 0.
  const int64_t srow = ((int64_t)b * p.H + h) * p.ranges.Lq;
  const float lse = p.lse[srow + row], shift = p.dlse ? p.dlse[srow + row] : 0.f;
  const bool none = !q_ok || lse == -INFINITY, one = (runs.y - runs.x) + (runs.w - runs.z) == 1;
  float lse2 = none ? INFINITY : lse * WA_LOG2E, on = one || !q_ok ? 0.f : 1.f;
  dl = none ? 0.f : one ? -shift : dl - shift;
  if (q_ok && g == 0) {
    p.lse2[srow + row] = lse2;
    p.on[srow + row] = on;
  }
  Bend bend = p.bend;
  int pos = 0;   // the row's position
  if (BENT && p.slopes) {
    bend.slope2 = p.slopes[h] * WA_LOG2E;
    pos = p.ranges.position(b) + qi;
  }
#pragma unroll
  for (int c = 0; c < DC; ++c) asm volatile("" : "+v"(qf[c]), "+v"(dof[c]));
  asm volatile("" : "+v"(lse2), "+v"(dl), "+v"(on), "+v"(runs.x), "+v"(runs.y), "+v"(runs.z), "+v"(runs.w));

  f32x16 dqacc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) dqacc[t] = f32x16{};
  float left = 0.f, a2 = 0.f, a3 = 0.f;   // sums of dS (before the cap's factor), of dS dist and P dist

  RT kt, vt;
  kt.init(p.k_st, w, lane);
  vt.init(p.v_st, w, lane);
  const bf16_t* kb = p.k + (int64_t)b * p.k_sb + (int64_t)(bh % p.Hk) * p.k_sh;
  const bf16_t* vb = p.v + (int64_t)b * p.v_sb + (int64_t)(bh % p.Hk) * p.v_sh;
  auto issue = [&](bf16_t* kv, int t) {
    const int key = st.key(t), rows = st.end(t) - key;
    kt.issue(kv, kb + key * p.k_st, p.k_st, rows, w);
    vt.issue(kv + TILE, vb + key * p.v_st, p.v_st, rows, w);
  };
  TileReads<D> rd;
  rd.init(lane);
  // 32 keys at a time: S^T = K Q^T and dP^T = V dO^T in turn, then dS^T = P^T (dP^T - delta) and what its rounding leaves, packed in accumulator
  // order for the next product
  // (both halves' products first, their exponentials after, took 64 more registers than there are).
  auto half = [&](uint32_t kc, uint32_t vc, int x, int key0, int end, bool whole, bf16x8* dsb, bf16x8* rest) {
    f32x16 s, dp;
    Operands a;
    auto read = [&](int c) {
      a[c % (kAhead + 1)][0] = rd.row8(kc, c, x);
      a[c % (kAhead + 1)][1] = rd.row8(vc, c, x);
    };
#pragma unroll
    for (int c = 0; c < kAhead; ++c) read(c);
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      if (c + kAhead < DC) read(c + kAhead);
      in_order();
      s = wa_mfma32(a[c % (kAhead + 1)][0], qf[c], c == 0 ? f32x16{} : s);
      dp = wa_mfma32(a[c % (kAhead + 1)][1], dof[c], c == 0 ? f32x16{} : dp);
      in_order();
    }
    auto weights = [&](auto form) {
      const RowRuns mine(runs, end);
      const float far = (float)(key0 - pos);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        float out[4], pr[4], turn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * r4 + i;
          turn[i] = 1.f;
          if constexpr (BENT) pr[i] = __builtin_amdgcn_exp2f(bend.bent<decltype(form)::value>(s[r], far + (float)(8 * r4 + i), turn[i]) - lse2);
          else pr[i] = __builtin_amdgcn_exp2f(fmaf(s[r], bend.scale2, -lse2));
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i) pr[i] = mine.sees(key0 + 8 * r4 + i) ? pr[i] : 0.f;
        }
        // products that are 0 where the weight is: what a masked key holds, NaN too, reaches nothing
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = zero_mul(pr[i], fmaf(dp[4 * r4 + i], on, -dl));
        left += (out[0] + out[1]) + (out[2] + out[3]);
        if constexpr (SLOPES) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float dist = fabsf(far + (float)(8 * r4 + i));
            a2 = fmaf(out[i], dist, a2);
            a3 = fmaf(pr[i], dist, a3);
          }
        }
        if constexpr (BENT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = zero_mul(out[i], turn[i]);
        }
        put4(dsb[r4 >> 1], r4 & 1, out);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] -= (float)dsb[r4 >> 1][4 * (r4 & 1) + i];
        put4(rest[r4 >> 1], r4 & 1, out);
        if constexpr (BENT) in_order();
      }
    };
    if constexpr (BENT) {
      float most = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[r]));
      by_form<BENT>(bend, most, weights);
    } else {
      weights(FormTag<kBias>{});
    }
  };
  // P (dP - delta) sums to the log-sum-exp's gradient: what it is beside that is delta's own error, from the rounded output.
  auto error = [&]() {
    const float sum = left + __shfl_xor(left, 32, 64);
    return on > 0.f && lse2 < INFINITY ? sum - (p.dlse ? p.dlse[srow + row] : 0.f) : 0.f;
  };
  // Few steps are walked twice, at first for delta alone.
#pragma unroll 1
  for (int walk = st.total <= kFewSteps ? 0 : 1; walk < 2; ++walk) {
    if (st.total > 0) issue(kv0, 0);
    for (int t = 0; t < st.total; ++t) {
      const uint32_t kc = rd.address(t & 1 ? kv1 : kv0), vc = kc + 2 * TILE;
      step_wait();
      if (t + 1 < st.total) issue(t & 1 ? kv0 : kv1, t + 1);   // the stage of step t - 1
      const int key = st.key(t), end = st.end(t);
      const bool whole = st.whole(key, end);
      bf16x8 dsb[2][4];
      half(kc, vc, 0, key + 4 * g, end, whole, dsb[0], dsb[1]);
      half(kc, vc, 1, key + 32 + 4 * g, end, whole, dsb[0] + 2, dsb[1] + 2);
      if (walk == 0) continue;
      // dQ^T[d, q] += K^T dS^T: A by transpose reads, B from registers (a row a lane)
      Operands a;
      ColsProduct<D>::first(rd, kc, a);
      ColsProduct<D>::run(rd, kc, dsb, dqacc, a);
    }
    if (walk == 1) break;
    dl += error();
    left = a2 = a3 = 0.f;
    __syncthreads();   // the stages are free
  }
  const float off = error();
  if (q_ok && g == 0) p.delta[srow + row] = dl + off;
  if constexpr (SLOPES) {
    a2 += __shfl_xor(a2, 32, 64);
    a3 += __shfl_xor(a3, 32, 64);
    const float mine = a2 - off * a3;
    float sum = g == 0 ? mine : 0.f;
    sum = wa_wave_sum(sum);
    if (lane == 0) s_part[w] = sum;
    __syncthreads();
    if (tid == 0) p.slope_part[((int64_t)h * p.B + b) * nq + qt] = -(s_part[0] + s_part[1] + s_part[2] + s_part[3]);
  }
  // channel 32 tt + 8 rq + 4 g + i of row l32 is register 4 rq + i of accumulator tt
  if (!q_ok) return;
  bf16_t* out = p.dq + (((int64_t)b * p.ranges.Lq + qi) * p.H + h) * D + 4 * g;
#pragma unroll
  for (int tt = 0; tt < DT; ++tt) {
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      bf16x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (bf16_t)(dqacc[tt][4 * rq + i] * p.scale);
      *(bf16x4*)(out + 32 * tt + 8 * rq) = x;
    }
  }
}

// The slopes' gradients: a workgroup a head, its parts added in a fixed order.
__global__ void __launch_bounds__(256) slopes_kernel(BwdParams p, int n) {
  __shared__ double s[256];
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) x += (double)p.slope_part[(int64_t)blockIdx.x * n + i];
  s[threadIdx.x] = x;
  __syncthreads();
  for (int m = 128; m >= 1; m >>= 1) {
    if ((int)threadIdx.x < m) s[threadIdx.x] += s[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.dslopes[blockIdx.x] = (float)s[0];
}

// ---------------------------------------------------------------------------------------------
// dK, dV: one workgroup of eight waves per 128 keys of a key head, over the 64-row tiles that see one of them, for each query head of the
// group in turn. Each 32 keys have two waves, on one SIMD, a key a lane:
//   the S-wave holds the keys and dV. Phase t: S = Q K^T of step t, P = exp2(s - lse2), P (1 - tanh^2) to LDS as fp16, dV += P^T dO;
//   the dP-wave holds the values and dK, a step behind. Phase t: dx of step t - 1 from its dP and the weights in LDS, dK += dx^T Q, then
//   dP = dO V^T of step t.
// So one wave's products run under the other's exponentials, with one barrier a step. Q, dO and the rows' statistics and runs stream two steps ahead
// into rings of four (Q is read by both phases), three and four stages; the weights have two. A workgroup takes 156 KiB of LDS at D = 128.
// parts > 1: the steps are cut into runs for workgroups of their own, whose fp32 sums another launch adds up in their order.
// ---------------------------------------------------------------------------------------------
constexpr int kListMax = 1024;   // row tiles listed at a time: 65,536 rows
constexpr int kKeys = 128;       // of a workgroup, as the order of the key tiles has them

template <int D, Bends BENT>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) ranged_dkv_kernel(BwdParams p) {
  constexpr int NW = 8, DC = D / 16, DT = D / 32, TILE = 64 * D;
  using RT = RowTile<D, NW>;
  constexpr int STATS = 192 + 256;   // floats of a stage: 64 lse2, 64 delta, 64 on, 64 rows' runs
  __shared__ __attribute__((aligned(2 * TILE))) bf16_t s_q[4 * TILE];   // tiles at multiples of their size (TileReads)
  __shared__ __attribute__((aligned(2 * TILE))) bf16_t s_do[3 * TILE];
  __shared__ __attribute__((aligned(1024))) f16x4 s_p[2][4][2][4][64];
  __shared__ __attribute__((aligned(1024))) float s_stats[4 * STATS];
  __shared__ int s_list[kListMax];   // row tile (from `base` on) | rows up to its last that sees anything << 10 | whole << 20
  __shared__ int s_count[NW];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, l32 = lane & 31, kg = w & 3;
  const bool swave = w < 4;   // wave-uniform role
  const int per = p.H / p.Hk, nbh = p.B * p.Hk;
  int u = (int)blockIdx.x;
  const int bh = u % nbh, hk = bh % p.Hk, b = bh / p.Hk;
  u /= nbh;
  const int part = u % p.parts, key0 = p.ranges.key_tile(b, u / p.parts) * kKeys;
  const int kl = kg * 32 + l32, key = key0 + kl;
  const bool k_ok = key < p.ranges.Lk;
  const int key_end = min(key0 + kKeys, p.ranges.Lk);

  bf16x8 kvf[DC];
  {
    const int kr = k_ok ? key : key0;
    const bf16_t* src = swave ? p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh + (int64_t)kr * p.k_st
                              : p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh + (int64_t)kr * p.v_st;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const bf16x8 a = *(const bf16x8*)(src + c * 16 + g * 8);
      kvf[c] = k_ok ? a : bf16x8{};
    }
  }
#pragma unroll
  for (int c = 0; c < DC; ++c) asm volatile("" : "+v"(kvf[c]));
  const int pos0 = BENT && p.slopes ? p.ranges.position(b) : 0;

  f32x16 acc[DT];   // S-wave: dV^T; dP-wave: dK^T (lane = key, registers = channels)
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
  RT qt, dt;
  qt.init(p.q_st, w, lane);
  dt.init(p.d_st, w, lane);
  TileReads<D> rd;
  rd.init(lane);

  for (int base = 0; base < p.ranges.n_tiles; base += kListMax) {
    const int limit = min(base + kListMax, p.ranges.n_tiles);
    int n = 0;
    for (int i0 = base; i0 < limit; i0 += 64 * NW) {
      const int i = i0 + tid;
      bool any = false;
      int entry = 0;
      if (i < limit) {
        const int32_t* r = p.ranges.tile(b, i);
        any = (r[kUpLo] < key_end && r[kUpHi] > key0) || (r[kLowLo] < key_end && r[kLowHi] > key0);
        // rows from Lq on read as zeros, their log-sum-exp too, and with a negative slope their weights may be infinite: masked, by runs of zeros
        const bool whole = ((r[kUpIn0] <= key0 && r[kUpIn1] >= key_end) || (r[kLowIn0] <= key0 && r[kLowIn1] >= key_end)) && (i + 1) * 64 <= p.ranges.Lq;
        entry = (i - base) | min(max(min(r[kRowEnd], p.ranges.Lq) - i * 64, 0), 64) << 10 | (whole ? 1 << 20 : 0);
      }
      const uint64_t mask = __ballot(any);
      __syncthreads();   // s_count of the round before has been read
      if (lane == 0) s_count[w] = __popcll(mask);
      __syncthreads();
      int at = n + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const int c = s_count[x];
        if (x < w) at += c;
        n += c;
      }
      if (any) s_list[at] = entry;
    }
    __syncthreads();
    n = __builtin_amdgcn_readfirstlane(n);
    const int all = n * per;
    const int first = (int)((int64_t)all * part / p.parts), total = (int)((int64_t)all * (part + 1) / p.parts) - first;
    if (total > 0) {
      int next_g = first / n, next_i = first % n, next_do = 0, now_do = 0;   // of the step issued next
      int now_g = next_g, now_i = next_i;
      // The next step's list entry is read while the present one is issued, and a head's addresses are formed once: what an issue takes from the
      // waves is scalar work that nothing hides.
      int next_entry = s_list[next_i];
      const bf16_t* qh = p.q + (int64_t)b * p.q_sb + (int64_t)(hk * per + next_g) * p.q_sh;
      const bf16_t* dh = p.dout + (int64_t)b * p.d_sb + (int64_t)(hk * per + next_g) * p.d_sh;
      const float* stat = w == 0 ? p.lse2 : w == 1 ? p.delta : p.on;   // the row statistics that this wave streams
      stat += ((int64_t)b * p.H + hk * per + next_g) * p.ranges.Lq;
      const int32_t* runs = p.ranges.rows + (int64_t)b * p.ranges.sb * p.ranges.Lq * 4;
      auto issue = [&](int t) {
        if (t >= total) return;
        const int entry = __builtin_amdgcn_readfirstlane(next_entry), rows = entry >> 10 & 127, row0 = (base + (entry & 1023)) * 64;
        const bf16_t *qn = qh, *dn = dh;
        const float* sn = stat;
        if (++next_i == n) {
          next_i = 0;
          qh += p.q_sh;
          dh += p.d_sh;
          stat += p.ranges.Lq;
        }
        next_entry = s_list[next_i];
        qt.issue(s_q + (t & 3) * TILE, qn + row0 * p.q_st, p.q_st, rows, w);
        dt.issue(s_do + next_do * TILE, dn + row0 * p.d_st, p.d_st, rows, w);
        next_do = next_do == 2 ? 0 : next_do + 1;
        if (w < 4) {
          float* to = s_stats + (t & 3) * STATS + 64 * w;
          const int count = min(64, p.ranges.Lq - row0);
          if (w < 3) {
            row_stats_dma(to, sn + row0, count, lane);
          } else {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(runs + (int64_t)row0 * 4), (short)0, count * 16, WA_BUF_DWORD3);
            lds_dma16(rs, to, lane * 16);
          }
        }
      };
      // Top of phase t: this wave's loads of step t have landed (those of step t + 1, five of an S-wave's and four of a dP-wave's at
      // D = 128, may be on their way) and its LDS reads returned, then the workgroup's.
      auto top = [&](int t) {
        if (t + 1 >= total) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else if (swave) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * RT::NI + 1) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * RT::NI) : "memory");
      };
      issue(0);
      issue(1);
      if (swave) {
        Bend bend = p.bend;
        if (BENT && p.slopes) bend.slope2 = p.slopes[hk * per + now_g] * WA_LOG2E;
        for (int t = 0; t < total; ++t) {
          top(t);
          const uint32_t qc = rd.address(s_q + (t & 3) * TILE);
          const uint32_t dc = rd.address(s_do + now_do * TILE);
          const float* st_lse2 = s_stats + (t & 3) * STATS;
          const int4* st_runs = (const int4*)(st_lse2 + 192);
          const int entry = __builtin_amdgcn_readfirstlane(s_list[now_i]);
          const int row0 = (base + (entry & 1023)) * 64;
          // S[q, key] = Q K^T per 32 rows; lane = key, registers = rows 32 x + 8 rq + 4 g + i
          f32x16 sacc[2];
          Operands a;
          RowsProduct<D>::first(rd, qc, a);
          RowsProduct<D>::run(rd, qc, kvf, sacc, a);
          issue(t + 2);
          ColsProduct<D>::first(rd, dc, a);   // under the exponentials
          in_order();
          bf16x8 ab[1][4];
          const bool whole = entry >> 20;
          auto weights = [&](auto form) {
            const float far = (float)(key - pos0 - row0 - 4 * g);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
              for (int rq = 0; rq < 4; ++rq) {
                const int r0 = 32 * x + 8 * rq;
                const f32x4 l4 = *(const f32x4*)(st_lse2 + r0 + 4 * g);
                float pr[4], turn[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float s = sacc[x][rq * 4 + i];
                  turn[i] = 1.f;
                  if constexpr (BENT) pr[i] = __builtin_amdgcn_exp2f(bend.bent<decltype(form)::value>(s, far - (float)(r0 + i), turn[i]) - l4[i]);
                  else pr[i] = __builtin_amdgcn_exp2f(fmaf(s, bend.scale2, -l4[i]));
                }
                if (!whole) {
#pragma unroll
                  for (int i = 0; i < 4; ++i) pr[i] = RowRuns(st_runs[r0 + 4 * g + i], INT32_MAX).sees(key) ? pr[i] : 0.f;
                }
                f16x4 p4;
#pragma unroll
                for (int i = 0; i < 4; ++i) p4[i] = (_Float16)(pr[i] * (BENT ? kLift * turn[i] : kLift));
                put4(ab[0][x * 2 + (rq >> 1)], rq & 1, pr);
                s_p[t & 1][kg][x][rq][lane] = p4;
                if (BENT || rq % 2) in_order();   // few rows' statistics in registers at a time
              }
            }
          };
          if constexpr (BENT) by_form<BENT>(bend, largest<2>(sacc), weights);
          else weights(FormTag<kBias>{});
          // dV^T[d, key] += dO^T P: A by transpose reads, B from registers
          ColsProduct<D>::run(rd, dc, ab, acc, a);
          now_do = now_do == 2 ? 0 : now_do + 1;
          if (++now_i == n) {
            now_i = 0;
            ++now_g;
            if (BENT && p.slopes && now_g < per) bend.slope2 = p.slopes[hk * per + now_g] * WA_LOG2E;
          }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // phase `total`
      } else {
        f32x16 dp[2];
        auto product = [&](int t) {   // dP[q, key] = dO V^T
          const uint32_t dc = rd.address(s_do + now_do * TILE);
          Operands a;
          RowsProduct<D>::first(rd, dc, a);
          RowsProduct<D>::run(rd, dc, kvf, dp, a);
          now_do = now_do == 2 ? 0 : now_do + 1;
        };
        auto gradient = [&](int t) {   // dK^T[d, key] += Q^T dS
          const uint32_t qc = rd.address(s_q + (t & 3) * TILE);
          const float* st_dl = s_stats + (t & 3) * STATS + 64;
          const float* st_on = st_dl + 64;
          bf16x8 ab[1][4];
          Operands a;
          ColsProduct<D>::first(rd, qc, a);
          in_order();
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
              const int r0 = 32 * x + 8 * rq + 4 * g;
              const f32x4 d4 = *(const f32x4*)(st_dl + r0), o4 = *(const f32x4*)(st_on + r0);
              const f16x4 p4 = s_p[t & 1][kg][x][rq][lane];
              float ds[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = rq * 4 + i;
                // a product that is 0 where the weight is: what a masked key holds, NaN too, reaches nothing
                ds[i] = zero_mul((float)p4[i], fmaf(dp[x][r], o4[i], -d4[i]));
              }
              put4(ab[0][x * 2 + (rq >> 1)], rq & 1, ds);
              if (rq % 2) in_order();
            }
          }
          ColsProduct<D>::run(rd, qc, ab, acc, a);
        };
        top(0);
        issue(2);
        product(0);
        for (int t = 1; t < total; ++t) {
          top(t);
          gradient(t - 1);
          issue(t + 2);
          product(t);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        gradient(total - 1);
      }
    }
    __syncthreads();   // the list and the stages are free
  }
  // each lane holds its key's row: channels 32 tt + 8 rq + 4 g .. + 3 of tile tt
  const float osc = swave ? 1.f : p.scale / kLift;
  const int rows = key_end - key0;
  const int64_t at0 = (((int64_t)b * p.ranges.Lk + key0) * p.Hk + hk) * D, st = (int64_t)p.Hk * D;
  if (p.parts > 1) {
    if (!k_ok) return;
    const int64_t size = (int64_t)p.B * p.ranges.Lk * st;
    float* dst = p.part_kv + ((int64_t)part * 2 + (swave ? 1 : 0)) * size + at0 + kl * st + 4 * g;
#pragma unroll
    for (int tt = 0; tt < DT; ++tt) {
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        f32x4 v4;
#pragma unroll
        for (int i = 0; i < 4; ++i) v4[i] = acc[tt][rq * 4 + i] * osc;
        *(f32x4*)(dst + 32 * tt + 8 * rq) = v4;
      }
    }
    return;
  }
  // Rows are staged in LDS, row r's 16-byte chunk c at chunk c ^ swz(r), and written whole.
  auto swz = [](int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); };
  bf16_t* stg = s_q + (swave ? 2 * TILE : 0);   // dK, dV
#pragma unroll
  for (int tt = 0; tt < DT; ++tt) {
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      bf16x4 v4;
#pragma unroll
      for (int i = 0; i < 4; ++i) v4[i] = (bf16_t)(acc[tt][rq * 4 + i] * osc);
      *(bf16x4*)(stg + kl * D + (((4 * tt + rq) ^ swz(kl)) << 3) + 4 * g) = v4;
    }
  }
  __syncthreads();
  constexpr int CPR = D / 8;
  for (int x = tid; x < rows * CPR; x += 64 * NW) {
    const int r = x / CPR, c = x % CPR;
    *(bf16x8*)(p.dk + at0 + r * st + c * 8) = *(const bf16x8*)(s_q + r * D + ((c ^ swz(r)) << 3));
    *(bf16x8*)(p.dv + at0 + r * st + c * 8) = *(const bf16x8*)(s_q + 2 * TILE + r * D + ((c ^ swz(r)) << 3));
  }
}

// dK and dV of a launch in parts: the parts' sums in their order, eight channels a thread.
__global__ void __launch_bounds__(256) parts_kernel(BwdParams p, int64_t size) {
  const int64_t x = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (x >= 2 * size) return;
  const float* src = p.part_kv + x;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  for (int i = 0; i < p.parts; ++i) {
    const f32x4 a = *(const f32x4*)(src + 2 * size * i), c = *(const f32x4*)(src + 2 * size * i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] += a[e];
      s[4 + e] += c[e];
    }
  }
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (bf16_t)s[e];
  *(bf16x8*)(x < size ? p.dk + x : p.dv + (x - size)) = o;
}

// Runs that the steps of 128 keys are cut into: about two workgroups a CU, but none of fewer than four steps, and at most eight (the runs' fp32 sums
// are written and read once more). 8,190 packed tokens, 4 key heads of 128: two runs 221 us and 13 for their sum, uncut 384; two sequences of 333
// tokens, 2 key heads of 64: 16 and 4, uncut 28.
int kv_parts(int64_t B, int64_t H, int64_t Hk, int64_t Lq, int64_t Lk) {
  const int64_t groups = B * Hk * ((Lk + kKeys - 1) / kKeys), steps = H / Hk * ((Lq + 63) / 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / groups, steps / 4, 8}));
}

template <int D, Bends BENT>
void launch_bwd(const BwdParams& p, hipStream_t s) {
  const int64_t nq = (p.ranges.Lq + 127) / 128;
  const dim3 gq((unsigned)(p.B * p.H * nq)), gk((unsigned)((int64_t)p.B * p.Hk * ((p.ranges.Lk + kKeys - 1) / kKeys) * p.parts));
  bool slopes = false;
  if constexpr (BENT) {
    slopes = p.dslopes;
    if (slopes) {
      hipLaunchKernelGGL((ranged_dq_kernel<D, BENT, true>), gq, dim3(256), 0, s, p);
      hipLaunchKernelGGL(slopes_kernel, dim3((unsigned)p.H), dim3(256), 0, s, p, (int)(p.B * nq));
    }
  }
  if (!slopes) hipLaunchKernelGGL((ranged_dq_kernel<D, BENT, false>), gq, dim3(256), 0, s, p);
  hipLaunchKernelGGL((ranged_dkv_kernel<D, BENT>), gk, dim3(512), 0, s, p);
  if (p.parts > 1) {
    const int64_t size = (int64_t)p.B * p.ranges.Lk * p.Hk * D;
    hipLaunchKernelGGL(parts_kernel, dim3((unsigned)((size / 4 + 255) / 256)), dim3(256), 0, s, p, size);
  }
}

template <int D>
void launch_bwd(const BwdParams& p, Bends bends, hipStream_t s) {
  if (bends == kPlain) launch_bwd<D, kPlain>(p, s);
  else if (bends == kUsual) launch_bwd<D, kUsual>(p, s);
  else launch_bwd<D, kOther>(p, s);
}

}  // namespace

extern "C" int64_t wa_ranged_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t Lq, int64_t Lk, int64_t D) {
  if (B < 1 || Hk < 1 || H < Hk || Lq < 1 || Lk < 1) return 0;
  const int parts = kv_parts(B, H, Hk, Lq, Lk);
  const int64_t rows = (B * H * Lq * 12 + B * H * ((Lq + 127) / 128) * 4 + 15) / 16 * 16;
  return rows + (parts > 1 ? parts * 2 * B * Lk * Hk * D * 4 : 0);
}

extern "C" int wa_ranged_bwd(const wa_ranged_bwd_args* a, void* stream) {
  WA_CHECK_ARG(a, "ranged_bwd: null args");
  WA_CHECK_ARG(a->D == 64 || a->D == 128, "ranged_bwd: head dim must be 64 or 128, got %lld", (long long)a->D);
  WA_CHECK_ARG(a->B >= 1 && a->Lq >= 1 && a->Lk >= 1 && a->Lq <= 1 << 30 && a->Lk <= 1 << 30 && a->Hk >= 1 && a->H >= a->Hk && a->H % a->Hk == 0 &&
               a->B <= INT32_MAX / a->H,
               "ranged_bwd: bad sizes B %lld Lq %lld Lk %lld heads %lld / %lld", (long long)a->B, (long long)a->Lq, (long long)a->Lk,
               (long long)a->H, (long long)a->Hk);
  WA_CHECK_ARG(a->q && a->k && a->v && a->o && a->dout && a->lse && a->rows && a->tiles && a->order && a->dq && a->dk && a->dv && a->workspace &&
               wa_aligned16(a->rows), "ranged_bwd: null tensor");
  WA_CHECK_ARG(!a->dslopes || a->slopes, "ranged_bwd: dslopes without slopes");
  auto rows16 = [](const void* x, int64_t sb, int64_t st, int64_t sh) {
    return wa_aligned16(x) && sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
  };
  auto near = [](int64_t st) { return st >= 0 && st <= (int64_t)1 << 23; };
  WA_CHECK_ARG(rows16(a->q, a->q_sb, a->q_st, a->q_sh) && rows16(a->k, a->k_sb, a->k_st, a->k_sh) && rows16(a->v, a->v_sb, a->v_st, a->v_sh) &&
               rows16(a->o, a->o_sb, a->o_st, a->o_sh) && rows16(a->dout, a->d_sb, a->d_st, a->d_sh) && wa_aligned16(a->dq) && wa_aligned16(a->dk) &&
               wa_aligned16(a->dv) && wa_aligned16(a->workspace) && near(a->q_st) && near(a->k_st) && near(a->v_st) && near(a->d_st),
               "ranged_bwd: rows must be 16-byte aligned, at most 2^23 elements apart");
  WA_CHECK_ARG(a->scale >= 0.f && a->scale < INFINITY && (a->cap == 0.f || (a->cap >= 1e-6f && a->cap <= 1e6f && a->scale <= 1e30f)),
               "ranged_bwd: scale must be finite and not below 0, cap 0 or 1e-6 .. 1e6 (with a scale of at most 1e30)");
  WA_CHECK_ARG(a->B * a->H * ((a->Lq + 127) / 128) <= INT32_MAX && a->B * a->H * ((a->Lk + 63) / 64) <= INT32_MAX && a->B * a->Lk * a->Hk * a->D / 1024 <= INT32_MAX && a->B * a->H * a->Lq / 16 <= INT32_MAX,
               "ranged_bwd: too many rows");
  BwdParams p{};
  p.q = (const bf16_t*)a->q; p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.k = (const bf16_t*)a->k; p.k_sb = a->k_sb; p.k_st = a->k_st; p.k_sh = a->k_sh;
  p.v = (const bf16_t*)a->v; p.v_sb = a->v_sb; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.o = (const bf16_t*)a->o; p.o_sb = a->o_sb; p.o_st = a->o_st; p.o_sh = a->o_sh;
  p.dout = (const bf16_t*)a->dout; p.d_sb = a->d_sb; p.d_st = a->d_st; p.d_sh = a->d_sh;
  p.lse = a->lse; p.dlse = a->dlse;
  p.ranges = {a->rows, a->tiles, a->ranges_sb ? 1 : 0, (int)a->Lq, (int)a->Lk, (int)((a->Lq + kRangeRows - 1) / kRangeRows), a->order};
  p.slopes = a->slopes;
  p.B = (int)a->B; p.H = (int)a->H; p.Hk = (int)a->Hk;
  p.scale = a->scale == 0.f ? 1.f / sqrtf((float)a->D) : a->scale;
  p.bend = bend_of(p.scale, a->cap);
  p.dq = (bf16_t*)a->dq; p.dk = (bf16_t*)a->dk; p.dv = (bf16_t*)a->dv; p.dslopes = a->dslopes;
  const int64_t n = a->B * a->H * a->Lq;
  p.lse2 = (float*)a->workspace;
  p.on = p.lse2 + n;
  p.delta = p.on + n;
  p.slope_part = p.delta + n;
  p.parts = kv_parts(a->B, a->H, a->Hk, a->Lq, a->Lk);
  p.part_kv = (float*)((char*)a->workspace + (n * 12 + a->B * a->H * ((a->Lq + 127) / 128) * 4 + 15) / 16 * 16);
  hipStream_t s = (hipStream_t)stream;
  const Bends bends = bends_of(p.scale, a->cap, a->slopes);
  if (a->D == 128) launch_bwd<128>(p, bends, s);
  else launch_bwd<64>(p, bends, s);
  return wa_launch_status("ranged_bwd");
}
