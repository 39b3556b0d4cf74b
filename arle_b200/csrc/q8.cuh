// The 8-bit cache: e4m3 codes [pages, heads, page_size, width] and one float32 scale, a power of two, for each page and head; a number is code * scale.
// The scale of a page is the least 2^e with max |x| <= 448 * 2^e (448 is the largest e4m3 number), e in [-100, 119]: 448 * 2^119 is finite in float32
// and a product with 2^100 does not overflow.  Powers of two cost nothing in e4m3 (a code's relative step does not depend on its exponent) and make
// every product with a scale, its reciprocal or the ratio of two exact: a page whose scale grows is rounded again only where a code falls below 2^-6.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace arle {

constexpr int kQ8Low = -100, kQ8High = 119;

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // e in [-126, 127]

// The least power of two that carries numbers of up to `most` (finite, not negative).
__device__ __forceinline__ float q8_scale(float most) {
  const uint32_t b = __float_as_uint(most);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);      // 448 = 1.75 * 2^8
  return exp2_int(min(max(e, kQ8Low), kQ8High));
}

// Two numbers as e4m3 codes: to nearest even, what is larger than 448 to 448, NaN stays.
__device__ __forceinline__ uint32_t q8_codes2(float lo, float hi) { return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d) { return q8_codes2(a, b) | (q8_codes2(c, d) << 16); }

// Four codes as float16 numbers, exactly: the first two and the last two.
__device__ __forceinline__ void q8_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;}\n" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ uint32_t q8_half2(uint32_t codes) {      // the low 16 bits
  uint32_t r;
  asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;}\n" : "=r"(r) : "r"(codes));
  return r;
}

__device__ __forceinline__ float2 q8_float2(uint32_t codes) {
  const uint32_t h = q8_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

constexpr uint32_t kInfBits = 0x7f800000u;

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The bits of |v|, 0 where v is not finite.  (Bits of numbers without their sign are ordered as the numbers are.)
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = abs_bits(v);
  return b < kInfBits ? b : 0u;
}
__device__ __forceinline__ float finite_or_nan(float v) { return abs_bits(v) < kInfBits ? v : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ float inverse_scale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }      // of a power of two in 2^-100 .. 2^119
__device__ __forceinline__ uint8_t exponent_byte(float s) { return (uint8_t)(__float_as_uint(s) >> 23); }                   // the same as e8m0

// The gates of a feed-forward in float32.  Silu's exponential is 2^(-g log2 e) by the special function unit: off by |g| 2^-24 of itself beside its two steps, as much
// as sums of some thousand products are (expf, which keeps that, cost the gated product of 4,096 rows 2 % of its time); the quotient is good to two steps and 0
// beyond 2^126, which is what silu is there.
__device__ __forceinline__ float q8_silu(float g) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(g * -1.4426950408889634f));
  return __fdividef(g, 1.0f + e);
}
__device__ __forceinline__ float q8_gelu_tanh(float g) { return 0.5f * g * (1.0f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g))); }

__device__ __forceinline__ float q8_float(uint8_t code) { return q8_float2(code).x; }

}  // namespace arle
