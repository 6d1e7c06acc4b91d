// The 8-bit key/value cache: e4m3 numbers (4 significant bits, up to 448, no infinity) under a power of two per block of
// 16 tokens and head. Shared by the kernel that writes the pages and those that read them.
//   K [pages, Hkv, page, D], V [pages, Hkv, D, page] bytes; powers [pages, Hkv, page / 16] bytes, stored with 127 added, so
//   that a byte shifted to a float's exponent is the power itself.
// A power of two changes no digit: a number of the cache stands for a bfloat16 number exactly (4 bits against 8), and a block
// whose power grows is rounded again only where its numbers fall below e4m3's smallest normal one.
#pragma once
#include "common.h"

constexpr int E4_BLOCK = 16;                       // tokens under one power
constexpr int E4_LEAST = -100, E4_MOST = 120;      // powers: bfloat16 keeps 2^-100 times e4m3's least number, and 448 * 2^119 is below its largest
constexpr int E4_BIAS = 127;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

// 2^p for p in [-126, 127]
__device__ __forceinline__ float e4_pow2(int p) { return __uint_as_float((uint32_t)(p + E4_BIAS) << 23); }

// The least power p with amax <= 448 * 2^p = 1.75 * 2^(8 + p), within bounds; amax is finite and not negative.
__device__ __forceinline__ int e4_power(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int p = (int)(u >> 23) - E4_BIAS - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(p, E4_LEAST), E4_MOST);
}

// What counts for a block's largest number: infinities and NaN do not (they are stored as NaN).
__device__ __forceinline__ float e4_size(float x) {
  const float s = fabsf(x);
  return s < INFINITY ? s : 0.f;
}
// x * scale is at most 448 in size where x is finite; an infinity has no e4m3 number and becomes NaN.
__device__ __forceinline__ float e4_scaled(float x, float scale) { return fabsf(x) < INFINITY ? x * scale : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t e4_pack(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// Four stored numbers times a power of two, rounded again.
__device__ __forceinline__ uint32_t e4_again(uint32_t w, float scale) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return e4_pack(lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale);
}
