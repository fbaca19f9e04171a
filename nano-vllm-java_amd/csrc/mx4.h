// The 4-bit form of include/nva.h on the device (included by .hip sources only): 32 values as e2m1
// codes beside one power of two.  The converters of gfx950 do the rounding (nearest, ties to even) and
// the reading; their results were compared with the definition for every code and scale byte, subnormal
// and NaN scales included.
#pragma once

#include <hip/hip_runtime.h>

#include "nva_device.h"

namespace nva {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Scale byte of a block whose largest magnitude has these bits (sign cleared): the smallest 2^e,
// -127 <= e <= 125, with top <= 6 * 2^e, from the exponent and whether the significand passes 1.5;
// 255 where the block holds a value that is not finite.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int e = (int)(top >> 23) - ((top & 0x7fffffu) > 0x400000u ? 1 : 2);
  return (uint32_t)min(max(e, 0), 252);
}

// The largest magnitude's bits of 8 values (NaN above infinity above the finite ones).
__device__ __forceinline__ uint32_t mx4_top8(const float *x) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) t = max(t, __float_as_uint(x[i]) & 0x7fffffffu);
  return t;
}

// The maximum over the four lanes of a quad.
__device__ __forceinline__ uint32_t max_quad(uint32_t t) {
  t = max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0xB1, 0xF, 0xF, false));
  return max(t, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)t, 0x4E, 0xF, 0xF, false));
}

// Codes of 8 values under a scale byte.  x * 2^-e is exact, or so small that its code is 0.
__device__ __forceinline__ uint32_t mx4_codes8(const float *x, uint32_t scale) {
  if (scale == 255u) return 0u;
  const float inv = __uint_as_float((254u - scale) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * inv, x[1] * inv, 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * inv, x[3] * inv, 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * inv, x[5] * inv, 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * inv, x[7] * inv, 1.0f, 3);
}

// A scale byte as the operand of the converters.
__device__ __forceinline__ float mx4_unit(uint32_t scale) { return __uint_as_float(scale << 23); }

// The two values of byte B of a word, as bf16 (exact: two significant bits).
template <int B> __device__ __forceinline__ uint32_t mx4_pair(uint32_t word, float unit) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, unit, B));
}

// The 8 values of a word in order, a matrix operand.
__device__ __forceinline__ bf16x8 mx4_frag(uint32_t word, float unit) {
  u32x4 r;
  r.x = mx4_pair<0>(word, unit);
  r.y = mx4_pair<1>(word, unit);
  r.z = mx4_pair<2>(word, unit);
  r.w = mx4_pair<3>(word, unit);
  return __builtin_bit_cast(bf16x8, r);
}

// 8 values as fp32.
__device__ __forceinline__ void mx4_values8(uint32_t word, float unit, float *x) {
#define NVA_PAIR(B)                                                               \
  {                                                                               \
    const uint32_t p = mx4_pair<B>(word, unit);                                   \
    x[2 * B] = __uint_as_float(p << 16), x[2 * B + 1] = __uint_as_float(p & 0xffff0000u); \
  }
  NVA_PAIR(0) NVA_PAIR(1) NVA_PAIR(2) NVA_PAIR(3)
#undef NVA_PAIR
}

// The largest magnitude of three (where one is NaN: of the others, or NaN).
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// x less its top half, exactly: the halves of a pair by a dot product with (-1, 0) and (0, -1), one
// instruction where taking the half apart and subtracting it are two.  (The masks stay in registers: as
// constants they would be read as fp32 ones.)
__device__ __forceinline__ float less_half(uint32_t halves, uint32_t minus, float x) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, halves),
                                         __builtin_bit_cast(bf16x2, minus), x, false);
}

// fp32 values as three bf16 parts whose sum they are: the top 8 bits of the significand, of what is left
// and of what is left then (cut off, not rounded, so nothing overflows).  w[p] holds the pairs' parts p.
// FINITE: the values are finite, or the NaNs among them may reach their neighbour too; otherwise an
// infinity is its first part alone.  (A NaN less its top half is a quiet NaN.)
template <bool FINITE, int PAIRS>
__device__ __forceinline__ void split3_pairs(const float *x, uint32_t (*w)[PAIRS]) {
  bool odd = false;
  if (!FINITE) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) top = max3_abs(top, x[2 * i], x[2 * i + 1]);
    odd = __any(!(top < INFINITY));
  }
  if (odd) {
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      float a = x[2 * i], b = x[2 * i + 1];
      // NaNs whose payload is below the top half keep being one.
      if (a != a) a = __uint_as_float(0x7fc00000u);
      if (b != b) b = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int p = 0; p < 3; p++) {
        const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
        w[p][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
        a -= __uint_as_float(ua & 0xffff0000u);
        b -= __uint_as_float(ub & 0xffff0000u);
        if (a != a) a = 0.f;  // (an infinity less itself)
        if (b != b) b = 0.f;
      }
    }
    return;
  }
  uint32_t first = 0x0000bf80u, second = 0xbf800000u;
  asm("" : "+s"(first));
  asm("" : "+s"(second));
#pragma unroll
  for (int i = 0; i < PAIRS; i++) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; p++) {
      w[p][i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);  // a below
      if (p < 2) {
        a = less_half(w[p][i], first, a);
        b = less_half(w[p][i], second, b);
      }
    }
  }
}

// 8 values; parts[p] holds parts p.
template <bool FINITE> __device__ __forceinline__ void split3(const float *x, bf16x8 *parts) {
  uint32_t w[3][4];
  split3_pairs<FINITE, 4>(x, w);
#pragma unroll
  for (int p = 0; p < 3; p++)
    parts[p] = __builtin_bit_cast(bf16x8, u32x4{w[p][0], w[p][1], w[p][2], w[p][3]});
}

}  // namespace nva
