// Values of 4-bit weights on the device.
#pragma once
#include "mixture_device.h"

typedef __attribute__((ext_vector_type(2))) f16_t f16x2;

// The 8 values of a word of codes, scale * (code - zero) rounded once to T.
//
// f16: a code in the low bits of 1024's significand is 1024 + code, the
// subtraction is exact and the product is the one rounding; two values an
// instruction. bf16 has no such arithmetic, so code * scale - zero * scale goes
// through a float fma: 4 bits times 8, so every term and the result are exact,
// and the conversion is the one rounding. (Scales are at most 2^120 there, or
// NaN, so zero * scale does not overflow.) 15 and 23 instructions a word.
template <class T>
struct FourScale;
template <>
struct FourScale<f16_t> {
  f16_t s, minus;  // -(1024 + zero)
  __device__ inline FourScale(f16_t scale, uint32_t zero) : s(scale), minus((f16_t)(-1024.0f - (float)zero)) {}
};
template <>
struct FourScale<bf16_t> {
  float s, minus;  // -zero * scale
  __device__ inline FourScale(bf16_t scale, uint32_t zero) : s((float)scale), minus(-(float)zero * s) {}
};
__device__ inline f16x8 four_values(uint32_t q, const FourScale<f16_t>& f) {
  f16x8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 c = __builtin_bit_cast(f16x2, (q >> (4 * i) & 0x000f000fu) | 0x64006400u);
    const f16x2 d = (c + f16x2{f.minus, f.minus}) * f16x2{f.s, f.s};
    v[2 * i] = d[0];
    v[2 * i + 1] = d[1];
  }
  return v;
}
__device__ inline bf16x8 four_values(uint32_t q, const FourScale<bf16_t>& f) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) bf16_t bf16x2;
  // bytes: columns 0, 4, 1, 5 and 2, 6, 3, 7 of the word
  uint32_t even = q & 0x0f0f0f0fu, odd = q >> 4 & 0x0f0f0f0fu;
  asm("" : "+v"(even), "+v"(odd));  // left as they are: a byte's conversion then needs no instruction to cut it out
  bf16x8 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i % 2 ? odd : even;
    const f32x2 c = {fmaf((float)(w >> (8 * (i / 2)) & 0xff), f.s, f.minus),
                     fmaf((float)(w >> (16 + 8 * (i / 2)) & 0xff), f.s, f.minus)};
    const bf16x2 b = __builtin_convertvector(c, bf16x2);
    v[2 * i] = b[0];
    v[2 * i + 1] = b[1];
  }
  return v;
}
// Codes 0 .. 15 of 8 columns to their word.
__device__ inline uint32_t four_word(const uint32_t (&c)[8]) {
  uint32_t q = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) q |= c[i] << (4 * (i / 2) + 16 * (i % 2));
  return q;
}
