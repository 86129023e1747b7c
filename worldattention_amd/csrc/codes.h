// 8-bit codes of a KV cache: int8 or e4m3 (OCP), 16 of them to a 16-byte chunk, with power-of-two scales.
#pragma once
#include "common.h"

namespace {

struct Int8 {
  // 16 codes as floats.
  __device__ __forceinline__ static void floats(const u32x4& c, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = (float)(int8_t)(c[i / 4] >> (8 * (i % 4)));
  }
  // Nearest codes, ties to even; the values fit.
  __device__ __forceinline__ static u32x4 codes(const float (&f)[16]) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) x |= ((uint32_t)(int)rintf(f[4 * i + j]) & 0xffu) << (8 * j);
      c[i] = x;
    }
    return c;
  }
  // Exponent of the smallest power of two that brings m 2^e, 1 <= m < 2, down to 127 = 1.984375 2^6.
  __device__ __forceinline__ static int power(float m, int e) { return m <= 1.984375f ? e - 6 : e - 5; }
  // Four codes as bf16 pairs (codes have at most eight significant bits: the upper halves of their floats).
  __device__ __forceinline__ static void pairs(uint32_t c, uint32_t& lo, uint32_t& hi) {
    const float a = (float)(int8_t)c, b = (float)(int8_t)(c >> 8), d = (float)(int8_t)(c >> 16), e = (float)((int32_t)c >> 24);
    lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
    hi = __builtin_amdgcn_perm(__float_as_uint(e), __float_as_uint(d), 0x07060302);
  }
  // The operand that holds a column of eight rows: column j of the four that each row's word has.
  __device__ __forceinline__ static u32x4 column(const uint32_t (&rows)[8], int j) {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)(rows[2 * e + 1] >> (8 * j))), __float_as_uint((float)(int8_t)(rows[2 * e] >> (8 * j))), 0x07060302);
    return x;
  }
};

struct E4m3 {
  __device__ __forceinline__ static void floats(const u32x4& c, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c[i], true);
      f[4 * i] = a[0];
      f[4 * i + 1] = a[1];
      f[4 * i + 2] = b[0];
      f[4 * i + 3] = b[1];
    }
  }
  __device__ __forceinline__ static u32x4 codes(const float (&f)[16]) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      x = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], x, true);
      c[i] = (uint32_t)x;
    }
    return c;
  }
  // ... down to 448 = 1.75 2^8.
  __device__ __forceinline__ static int power(float m, int e) { return m <= 1.75f ? e - 8 : e - 7; }
  __device__ __forceinline__ static void pairs(uint32_t c, uint32_t& lo, uint32_t& hi) {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true));
  }
  __device__ __forceinline__ static u32x4 column(const uint32_t (&rows)[8], int j) {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t a, b;
      if (j < 2) {
        a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[2 * e], 1.f, false));
        b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[2 * e + 1], 1.f, false));
      } else {
        a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[2 * e], 1.f, true));
        b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rows[2 * e + 1], 1.f, true));
      }
      x[e] = __builtin_amdgcn_perm(b, a, j % 2 ? 0x07060302 : 0x05040100);
    }
    return x;
  }
};

}  // namespace
