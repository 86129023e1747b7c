// A KV cache in 8 bits: written with a scale for each block of tokens and head, and read back. No reference counterpart; the
// attention over it is attend8.hip.
#include <algorithm>

#include "codes.h"

namespace {

__device__ __forceinline__ int64_t per_sequence(const int32_t* t, int64_t all, int b) { return t ? (int64_t)t[b] : all; }

// ---------------------------------------------------------------------------------------------
// Append: one workgroup per (sequence, head, touched block, keys or values), 16 channels of a row a thread. The new rows stay in registers
// from the maximum of their magnitudes to their codes; the block's earlier codes are read for the keys' sums (those of the whole block as it
// is now: rewritten tokens and a grown scale leave nothing stale in them) and, where the scale grows, rounded again. Scales are powers of
// two, so a growth is a shift, and what a token is off by stays below a step: half a step of each scale that it was held at, 1/2 + 1/4 + ...
// Bound by memory for prompts; a single token of each sequence is a few dependent trips to memory.
// ---------------------------------------------------------------------------------------------
struct AppendParams {
  uint8_t* code[2];
  float* scale[2];
  float* sums;
  const void* src[2];
  int64_t sb[2], st[2], sh[2];
  const int32_t* start; int64_t start_all;
  const int32_t* lengths;
  int64_t cap;
  int n, Hk, bs, nb, touched;   // touched: blocks of a sequence, at most
};

template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&f)[16]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const bf16x8 x = *(const bf16x8*)(p + 8 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[8 * c + e] = (float)x[e];
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x4 x = *(const f32x4*)(p + 4 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * c + e] = x[e];
    }
  }
}

template <typename Code, typename T, int D, int BS>
__global__ void __launch_bounds__(256) append_kernel(AppendParams p) {
  constexpr int CPR = D / 16, RPP = 256 / CPR, PASSES = BS / RPP;   // threads of a row; rows of a pass
  static_assert(BS % RPP == 0, "whole passes");
  __shared__ uint32_t s_top[4];
  __shared__ float s_sum[4][D];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c0 = tid % CPR * 16, r0 = tid / CPR;
  int u = (int)blockIdx.x;
  const int kv = u & 1;
  u >>= 1;
  const int h = u % p.Hk;
  u /= p.Hk;
  const int b = u / p.touched;
  const int64_t start = per_sequence(p.start, p.start_all, b);
  const int64_t count = min(max(p.lengths ? (int64_t)p.lengths[b] : (int64_t)p.n, (int64_t)0), (int64_t)p.n);
  if (count == 0 || start < 0 || start + count > p.cap) return;
  const int64_t block = start / BS + u % p.touched, lo = block * BS;
  if (lo >= start + count) return;
  const int first = (int)max(start - lo, (int64_t)0), end = (int)min(start + count - lo, (int64_t)BS);   // the block's new rows

  const T* src = (const T*)p.src[kv] + (int64_t)b * p.sb[kv] + (int64_t)h * p.sh[kv] + (lo - start) * p.st[kv] + c0;
  float x[PASSES][16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + i * RPP;
    if (r >= first && r < end) {
      load16(src + r * p.st[kv], x[i]);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
  if (lane == 0) s_top[w] = top;
  __syncthreads();
  top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
  float* scale_at = p.scale[kv] + ((int64_t)b * p.Hk + h) * p.nb + block;
  const float before = first > 0 ? *scale_at : 0.f;
  const int power = max(Code::power(__uint_as_float((top & 0x7fffffu) | 0x3f800000u), (int)(top >> 23) - 127), -126);
  float now = __uint_as_float((uint32_t)(power + 127) << 23);
  if (top >= 0x7f800000u || !(before < INFINITY)) now = NAN;   // an infinity or NaN among the new values, or one before them
  else if (before > now) now = before;
  const float in = now == now ? 1.f / now : 0.f, again = before * in;
  const bool grown = first > 0 && again != 1.f && now == now;
  __syncthreads();   // every thread has read the scale

  uint8_t* at = p.code[kv] + (((int64_t)b * p.cap + lo) * p.Hk + h) * D + c0;
  const int64_t row = (int64_t)p.Hk * D;
  float sum[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + i * RPP;
    if (r >= end) continue;
    float f[16];
    u32x4 c;
    if (r >= first) {
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] = now == now ? x[i][e] * in : 0.f;
      c = Code::codes(f);
      *(u32x4*)(at + r * row) = c;
    } else {
      if (!grown && kv == 1) continue;   // the values' earlier codes stand
      c = *(const u32x4*)(at + r * row);
      if (grown) {
        Code::floats(c, f);
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] *= again;
        c = Code::codes(f);
        *(u32x4*)(at + r * row) = c;
      }
    }
    if (kv == 0 && p.sums) {
      Code::floats(c, f);
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[e] += f[e];
    }
  }
  if (tid == 0) *scale_at = now;
  if (kv == 1 || !p.sums) return;
  // rows' threads of a wave, then the waves
#pragma unroll
  for (int m = CPR; m < 64; m <<= 1) {
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] += __shfl_xor(sum[e], m, 64);
  }
  if (lane < CPR) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s_sum[w][c0 + e] = sum[e];
  }
  __syncthreads();
  if (tid < D)
    p.sums[(((int64_t)b * p.Hk + h) * p.nb + block) * D + tid] = (s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid]) * now;
}

// ---------------------------------------------------------------------------------------------
// Read: 16 codes a thread, keys and values in one launch. Memory-bound.
// ---------------------------------------------------------------------------------------------
struct ReadParams {
  const uint8_t* code[2];
  const float* scale[2];
  void* out[2];
  const int32_t* start; int64_t start_all;
  const int32_t* kv_len; int64_t kv_len_all;
  int64_t last, window, sink, cap;
  unsigned chunks;   // of 16 codes, of a sequence
  int Hk, bs, nb, D;
};

template <typename Code, typename T>
__global__ void __launch_bounds__(256) read_kernel(ReadParams p) {
  const unsigned u = blockIdx.x * 256 + threadIdx.x;   // of one sequence: (token, head, chunk)
  if (u >= p.chunks) return;
  const int b = (int)blockIdx.y, kv = (int)blockIdx.z, shift = p.D == 128 ? 3 : 2;
  const unsigned row = u >> shift, i = row / (unsigned)p.Hk, h = row % (unsigned)p.Hk, c0 = (u & ((1u << shift) - 1)) * 16;
  const int64_t t = per_sequence(p.start, p.start_all, b) + i;
  if (p.kv_len || p.kv_len_all >= 0) {
    const int64_t len = min(per_sequence(p.kv_len, p.kv_len_all, b), p.cap);   // as the attention takes it
    if (t >= len || (p.window > 0 && t >= p.sink && t <= len - p.last - p.window)) return;
  }
  float f[16];
  if (t >= 0 && t < p.cap) {
    const int64_t at = (((int64_t)b * p.cap + t) * p.Hk + h) * p.D + c0;
    Code::floats(*(const u32x4*)(p.code[kv] + at), f);
    const float s = p.scale[kv][((int64_t)b * p.Hk + h) * p.nb + (t >> (p.bs == 64 ? 6 : 7))];
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] *= s;
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = 0.f;
  }
  T* out = (T*)p.out[kv] + ((int64_t)b * p.chunks + u) * 16;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (bf16_t)f[8 * c + e];
      *(bf16x8*)(out + 8 * c) = x;
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) *(f32x4*)(out + 4 * c) = f32x4{f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]};
  }
}

int check_cache(const char* what, const wa_cache8& c) {
  WA_CHECK_ARG(c.D == 64 || c.D == 128, "%s: head dim must be 64 or 128, got %lld", what, (long long)c.D);
  WA_CHECK_ARG(c.block_size == 64 || c.block_size == 128, "%s: block size must be 64 or 128, got %lld", what, (long long)c.block_size);
  WA_CHECK_ARG(c.code == WA_CODE_INT8 || c.code == WA_CODE_E4M3, "%s: unknown code %d", what, c.code);
  WA_CHECK_ARG(c.B >= 1 && c.Hk >= 1 && c.cap >= 1 && c.cap <= 1 << 30 && c.Hk <= 65536 && c.B <= INT32_MAX / c.Hk, "%s: bad sizes B %lld cap %lld Hk %lld",
               what, (long long)c.B, (long long)c.cap, (long long)c.Hk);
  WA_CHECK_ARG(c.k && c.v && c.k_scale && c.v_scale && wa_aligned16(c.k) && wa_aligned16(c.v), "%s: null or misaligned cache", what);
  return WA_OK;
}

template <typename Code, typename T>
void launch_append(const AppendParams& p, int64_t D, unsigned grid, hipStream_t s) {
  if (D == 128 && p.bs == 128) hipLaunchKernelGGL((append_kernel<Code, T, 128, 128>), dim3(grid), dim3(256), 0, s, p);
  else if (D == 128) hipLaunchKernelGGL((append_kernel<Code, T, 128, 64>), dim3(grid), dim3(256), 0, s, p);
  else if (p.bs == 128) hipLaunchKernelGGL((append_kernel<Code, T, 64, 128>), dim3(grid), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((append_kernel<Code, T, 64, 64>), dim3(grid), dim3(256), 0, s, p);
}

}  // namespace

extern "C" int wa_kv8_append(const wa_kv8_append_args* a, void* stream) {
  WA_CHECK_ARG(a, "kv8_append: null args");
  const int rc = check_cache("kv8_append", a->cache);
  if (rc != WA_OK) return rc;
  const wa_cache8& c = a->cache;
  WA_CHECK_ARG(a->n >= 0 && a->n <= c.cap, "kv8_append: %lld tokens do not fit a cache of %lld", (long long)a->n, (long long)c.cap);
  if (a->n == 0) return WA_OK;
  WA_CHECK_ARG(a->start || (a->start_all >= 0 && a->start_all <= c.cap - a->n), "kv8_append: %lld tokens from %lld on do not fit a cache of %lld",
               (long long)a->n, (long long)a->start_all, (long long)c.cap);
  WA_CHECK_ARG(a->dtype == WA_BF16 || a->dtype == WA_F32, "kv8_append: unknown dtype %d", a->dtype);
  const int64_t unit = a->dtype == WA_BF16 ? 8 : 4;
  auto rows16 = [&](const void* x, int64_t sb, int64_t st, int64_t sh) {
    return x && wa_aligned16(x) && sb % unit == 0 && st % unit == 0 && sh % unit == 0;
  };
  WA_CHECK_ARG(rows16(a->k, a->k_sb, a->k_st, a->k_sh) && rows16(a->v, a->v_sb, a->v_st, a->v_sh), "kv8_append: null or misaligned rows");
  AppendParams p{};
  p.code[0] = (uint8_t*)c.k; p.code[1] = (uint8_t*)c.v;
  p.scale[0] = c.k_scale; p.scale[1] = c.v_scale; p.sums = c.k_sums;
  p.src[0] = a->k; p.sb[0] = a->k_sb; p.st[0] = a->k_st; p.sh[0] = a->k_sh;
  p.src[1] = a->v; p.sb[1] = a->v_sb; p.st[1] = a->v_st; p.sh[1] = a->v_sh;
  p.start = a->start; p.start_all = a->start_all; p.lengths = a->lengths;
  p.cap = c.cap; p.n = (int)a->n; p.Hk = (int)c.Hk; p.bs = (int)c.block_size;
  p.nb = (int)((c.cap + c.block_size - 1) / c.block_size);
  p.touched = a->start ? (int)((a->n + 2 * c.block_size - 2) / c.block_size)
                       : (int)((a->start_all + a->n - 1) / c.block_size - a->start_all / c.block_size + 1);
  const int64_t grid = 2 * c.B * c.Hk * p.touched;
  WA_CHECK_ARG(grid <= INT32_MAX, "kv8_append: too many tokens");
  hipStream_t s = (hipStream_t)stream;
  if (c.code == WA_CODE_INT8) {
    if (a->dtype == WA_BF16) launch_append<Int8, bf16_t>(p, c.D, (unsigned)grid, s);
    else launch_append<Int8, float>(p, c.D, (unsigned)grid, s);
  } else {
    if (a->dtype == WA_BF16) launch_append<E4m3, bf16_t>(p, c.D, (unsigned)grid, s);
    else launch_append<E4m3, float>(p, c.D, (unsigned)grid, s);
  }
  return wa_launch_status("kv8_append");
}

extern "C" int wa_kv8_read(const wa_kv8_read_args* a, void* stream) {
  WA_CHECK_ARG(a, "kv8_read: null args");
  const int rc = check_cache("kv8_read", a->cache);
  if (rc != WA_OK) return rc;
  const wa_cache8& c = a->cache;
  WA_CHECK_ARG(a->n >= 0 && a->n <= 1 << 30 && a->last >= 0 && a->window >= 0 && a->sink >= 0, "kv8_read: bad sizes");
  if (a->n == 0) return WA_OK;
  WA_CHECK_ARG(a->dtype == WA_BF16 || a->dtype == WA_F32, "kv8_read: unknown dtype %d", a->dtype);
  WA_CHECK_ARG(a->k_out && a->v_out && wa_aligned16(a->k_out) && wa_aligned16(a->v_out), "kv8_read: null or misaligned output");
  ReadParams p{};
  p.code[0] = (const uint8_t*)c.k; p.code[1] = (const uint8_t*)c.v;
  p.scale[0] = c.k_scale; p.scale[1] = c.v_scale;
  p.out[0] = a->k_out; p.out[1] = a->v_out;
  // beyond any cache numbers count as just beyond it: the kernel's sums of them stay in 64 bits
  const int64_t far = (int64_t)1 << 31;
  p.start = a->start; p.start_all = std::min(std::max(a->start_all, -far), far); p.kv_len = a->kv_len; p.kv_len_all = a->kv_len_all;
  p.last = std::min(a->last, far); p.window = std::min(a->window, far); p.sink = std::min(a->sink, far); p.cap = c.cap;
  p.Hk = (int)c.Hk; p.bs = (int)c.block_size; p.D = (int)c.D;
  p.nb = (int)((c.cap + c.block_size - 1) / c.block_size);
  const int64_t chunks = a->n * c.Hk * (c.D / 16);
  WA_CHECK_ARG(chunks <= INT32_MAX && c.B <= 65535, "kv8_read: at most 65535 sequences and 2^31 - 1 chunks of 16 channels each");
  p.chunks = (unsigned)chunks;
  const dim3 grid((unsigned)((chunks + 255) / 256), (unsigned)c.B, 2);
  hipStream_t s = (hipStream_t)stream;
  if (c.code == WA_CODE_INT8) {
    if (a->dtype == WA_BF16) hipLaunchKernelGGL((read_kernel<Int8, bf16_t>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((read_kernel<Int8, float>), grid, dim3(256), 0, s, p);
  } else {
    if (a->dtype == WA_BF16) hipLaunchKernelGGL((read_kernel<E4m3, bf16_t>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((read_kernel<E4m3, float>), grid, dim3(256), 0, s, p);
  }
  return wa_launch_status("kv8_read");
}
