// The software-pipelined step loop of the attention forward kernels (bsa_fwd.hip, ranged.hip): tile
// loads and their LDS layouts, one slot of the loop, and the running maximum's rescaling.
#pragma once
#include "common.h"
#include "tile.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
#define WA_LDS(p) ((__attribute__((address_space(3))) void*)(p))
#define WA_LDS4(p) ((__attribute__((address_space(3))) s16x4*)(p))

// 16-byte chunk swizzles. gfx950 serves a 128-bit LDS read 16 lanes (256 bytes, all 64 banks)
// per cycle, and the transpose read 16 lanes x 8 bytes (128 bytes) per cycle:
//   K row r, D = 128 (256-byte rows): chunk ^ (r & 15) — 16 consecutive keys hit 16 distinct
//     chunk slots of their rows, i.e. all 64 banks;
//   K row r, D = 64 (128-byte rows, two per bank line): chunk ^ ((r >> 1) & 7);
//   V row r: chunk ^ 2 (r & 3) — a transpose read's 16 lanes cover 4 rows x 32 bytes, which this
//     spreads over 4 x 8 distinct banks.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }
__device__ __forceinline__ int v_swizzle(int r) { return 2 * (r & 3); }

// One [64, D] bf16 step tile (64 consecutive key rows) streamed into swizzled LDS with
// direct-to-LDS buffer loads. Wave instruction i moves 1 KiB = RPI whole rows: lane L writes row
// r0(i) + L / CPR, slot L % CPR, and so reads the chunk that the swizzle stores in that slot. The
// per-lane byte offsets within a tile are loop-invariant; a tile is selected by its buffer
// descriptor, which starts at the tile's first row and ends at the slab's end. Rows past a partial
// block's end read either the following keys (finite, masked or multiplied by a zero probability)
// or, past the slab, zeros.
template <int D, int NW>
struct NextTile {
  static constexpr int CPR = D / 8;                  // 16-byte chunks per row
  static constexpr int RPI = 64 / CPR;               // rows per wave instruction (4 or 8)
  static constexpr int NI = 64 / (RPI * NW);         // instructions per wave per tensor
};

// ---------------------------------------------------------------------------------------------
// Software-pipelined step loop. A 64-key step is two 32-key halves, and the loop runs in "slots",
// one half each. Slot (block b, half h) does three independent pieces of work:
//   * the softmax of the half-step whose scores the previous slot produced: S[1 - h] -> the
//     probability chunks P[2(1-h)], P[2(1-h)+1] and the slot's row sum;
//   * the QK product of half h of step b (K stage of step b) -> S[h];
//   * the PV product of half h of step b - 1 (V stage of step b - 1) with P[2h], P[2h+1];
// plus, in the block's first slot, the tile loads of the next block (K of step b + 1, V of step b:
// both stages were last read in block b - 1, so the loads go out a whole block ahead). The softmax (~56 VALU instructions at D = 128)
// interleaves with the 16 products inside the wave, so the SIMD issues VALU work while the MFMA
// pipe is busy instead of after it.
// ---------------------------------------------------------------------------------------------

// Direct-to-LDS 16-byte load through the compiler's builtin: the scheduler sees a memory load (LDS
// reads move freely around it) and the wait-count pass tracks it per LDS array. Every ring stage is
// an array of its own and every access names its stage statically, so a read of one stage never
// waits for loads into another; the kernel still orders loads across waves itself (pipe_sync at the
// top of each block).
__device__ __forceinline__ void pipe_dma16(__amdgpu_buffer_rsrc_t rs, bf16_t* lds, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

// Top of a block: this wave's tile loads (but the AHEAD latest) have landed and its LDS reads have
// returned, then the same for the workgroup: the stages read last may be refilled. The reads are
// waited for by name: the products that consume them are free to move below the barrier (the key-split
// loop's first one does), and a load that hits L1, as one does behind the CU's other workgroup on the
// same keys, can refill the stage sooner than a read in flight returns.
template <int AHEAD>
__device__ __forceinline__ void pipe_sync() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(AHEAD) : "memory");
}

// Instruction-group order of one slot: after a few leading LDS reads, each product is followed by
// up to DSN LDS reads and VAN VALU instructions, and every VMEVERY-th product by one tile load.
template <int I, int N, int DSN, int VAN, int VMEVERY>
__device__ __forceinline__ void pipe_sched() {
  if constexpr (I < N) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);    // MFMA
    __builtin_amdgcn_sched_group_barrier(0x100, DSN, 0);  // LDS read
    __builtin_amdgcn_sched_group_barrier(0x002, VAN, 0);  // VALU
    if constexpr (VMEVERY > 0 && I % VMEVERY == 0) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // VMEM
    pipe_sched<I + 1, N, DSN, VAN, VMEVERY>();
  }
}

// Tile loads of one slot: NI direct-to-LDS loads of a tensor's next tile into stage `lds`.
struct PipeLoad {
  __amdgpu_buffer_rsrc_t rs;
  bf16_t* lds;
};

// One slot (see above) of a wave that owns QT 32-query tiles. SMH: half whose softmax runs (1 - the
// product half). SM / QK / PV / LD switch the pieces on for the pipeline's first and last blocks.
// With QT = 2 every K and V fragment read from LDS feeds two products. rs[qt]: the slot's row sum
// of exponentials of tile qt (this lane's 16 keys).
template <int D, int NW, int QT, int SMH, bool SM, bool QK, bool PV, bool LD, int KROW = -1>
__device__ __forceinline__ void pipe_slot(f32x16 (&S)[2][QT], bf16x8 (&P)[4][QT], f32x16 (&oacc)[QT][D / 32],
                                          const bf16x8 (&qf)[QT][D / 16], const bf16_t* kst, const bf16_t* vst,
                                          const int (&k_rd)[D / 16], const int (&v_rd)[2], const float (&neg_m)[QT],
                                          float scale_log2, const PipeLoad& ldk, const int (&koff)[NextTile<D, NW>::NI],
                                          const PipeLoad& ldv, const int (&voff)[NextTile<D, NW>::NI], int w,
                                          float (&rs)[QT]) {
  constexpr int H = SMH ^ 1, DC = D / 16, DT = D / 32;
  constexpr int RH = KROW < 0 ? H : KROW;  // key half of the K / V rows (the key-split loop fixes it)
  constexpr int NI = NextTile<D, NW>::NI, RPI = NextTile<D, NW>::RPI;
  // operands from LDS: K rows 32 RH + l32 (A of S^T = K Q^T), V^T of keys 32 RH .. +32 (A of O^T += V^T P^T)
  bf16x8 kf[DC];
  if constexpr (QK) {
#pragma unroll
    for (int c = 0; c < DC; ++c) kf[c] = *(const bf16x8*)(kst + k_rd[c] + RH * 32 * D);
  }
  bf16x8 vf[2][DT];
  if constexpr (PV) {
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
#pragma unroll
      for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const s16x4 vv = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              WA_LDS4(vst + v_rd[t & 1] + (16 * (2 * RH + cc) + 8 * hf) * D + (t >> 1) * 64));
          const bf16x4 vb4 = __builtin_bit_cast(bf16x4, vv);
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[cc][t][4 * hf + e] = vb4[e];
        }
      }
    }
  }
  if constexpr (QK) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) S[H][qt] = wa_mfma32(kf[0], qf[qt][0], f32x16{});
#pragma unroll
    for (int c = 1; c < DC; ++c) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) S[H][qt] = wa_mfma32(kf[c], qf[qt][c], S[H][qt]);
    }
  }
  if constexpr (PV) {
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
#pragma unroll
      for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) oacc[qt][t] = wa_mfma32(vf[cc][t], P[2 * H + cc][qt], oacc[qt][t]);
      }
    }
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) rs[qt] = 0.f;
  if constexpr (SM) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float r0 = 0.f, r1 = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pv = __builtin_amdgcn_exp2f(fmaf(S[SMH][qt][r], scale_log2, neg_m[qt]));
        if (r & 1) r1 += pv;
        else r0 += pv;
        P[2 * SMH + (r >> 3)][qt][r & 7] = (bf16_t)pv;
      }
      rs[qt] = r0 + r1;
    }
  }
  if constexpr (LD) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      pipe_dma16(ldk.rs, ldk.lds + (i * NW + w) * RPI * D, koff[i]);
      pipe_dma16(ldv.rs, ldv.lds + (i * NW + w) * RPI * D, voff[i]);
    }
  }
  constexpr int NM = QT * ((QK ? DC : 0) + (PV ? 2 * DT : 0));
  constexpr int NDS = (QK ? DC : 0) + (PV ? 4 * DT : 0);
  if constexpr (NM > 0) {
    __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
    pipe_sched<0, NM, (NDS + NM - 1) / NM, 4, LD ? (NM / (2 * NI) > 0 ? NM / (2 * NI) : 1) : 0>();
  }
}

// Keys of half KH of a step at or past `real` get score -inf (probability 0): lane (l32, g) holds
// keys 32 KH + 8 (r / 4) + 4 g + r % 4 in S[r].
template <int KH, int QT>
__device__ __forceinline__ void pipe_mask(f32x16 (&s)[QT], int real, int g) {
  const int rr = real - 32 * KH - 4 * g;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[qt][r] = 8 * (r >> 2) + (r & 3) >= rr ? -INFINITY : s[qt][r];
  }
}

// A slot whose exponentials failed the sum check: each tile's m_i moves to the running max over its
// half-step s (every half-step the pipeline starts with holds a real key, so the max is finite;
// where it does not exceed m_i the factor is 1 and nothing changes), the output accumulators
// (which already include this slot's PV product) and l_i are rescaled, and the half's
// probabilities P[2 PH], P[2 PH + 1] and row sums are recomputed.
template <int D, int QT, int PH>
__device__ __forceinline__ void pipe_rescale(const f32x16 (&s)[QT], bf16x8 (&P)[4][QT], f32x16 (&oacc)[QT][D / 32],
                                             float (&m_i)[QT], float (&l_i)[QT], float (&rs)[QT], float scale_log2) {
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[qt][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * scale_log2;
    const float m_new = fmaxf(mx, m_i[qt]);
    const float alpha = __builtin_amdgcn_exp2f(m_i[qt] - m_new);
    l_i[qt] *= alpha;
    m_i[qt] = m_new;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) oacc[qt][t] *= alpha;
    float r0 = 0.f, r1 = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float pv = __builtin_amdgcn_exp2f(fmaf(s[qt][r], scale_log2, -m_i[qt]));
      if (r & 1) r1 += pv;
      else r0 += pv;
      P[2 * PH + (r >> 3)][qt][r & 7] = (bf16_t)pv;
    }
    rs[qt] = r0 + r1;
  }
}

template <int QT>
__device__ __forceinline__ bool pipe_check(const float (&rs)[QT]) {
  bool bad = false;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) bad |= !(rs[qt] <= 65536.f);
  return __any(bad);
}

}  // namespace
