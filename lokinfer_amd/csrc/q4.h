// Values held in 4 bits: x = s (c - 8), a code c of 0 .. 15 and its group's scale s >= 0, an f16 of at most 8 significant
// bits, so that s (c - 8) (8 + 3 bits; -8 s is a shift) is exact in f16: a kernel may multiply by s before or after its
// products without another rounding.
//
// A group's scale is the smallest such s with 7 s >= its largest and 8 s >= minus its smallest value (bounded by 8128, so
// that -8 s is finite: a magnitude over 56896 is held as 56896 or 65024), its codes 8 + floor(x / s + 1/2), clamped to
// 0 .. 15. x / s, an 11-bit by an 8-bit number, is k + 1/2 or at least 2^-13 away from it, so the f32 quotient decides as the
// exact one does. A group that holds an infinity or a NaN gets s = NaN.
//
// Eight codes of consecutive values go into one 32-bit word, the even ones at bits 0, 4, 8, 12 and the odd ones 16 above:
// an `and` with 0x000F000F then leaves a pair of codes where a pair of f16 has its mantissas.
#pragma once

#include "f16.h"

namespace lkd {

typedef h16 half2v __attribute__((ext_vector_type(2)));

// hi >= 0, lo <= 0: the group's largest and smallest value (0 among them)
__device__ __forceinline__ float q4Scale(float hi, float lo) {
  const float a = fmaxf(hi / 7.0f, lo * -0.125f);
  float s = __uint_as_float((__float_as_uint(a) + 0xFFFFu) & 0xFFFF0000u);  // up to 8 significant bits
  if (s < 0x1p-17f) s = ceilf(a * 0x1p24f) * 0x1p-24f;                      // f16's smallest step
  return fminf(s, 8128.0f);
}

__device__ __forceinline__ unsigned q4Code(float x, float s) {
  if (!(s > 0.0f)) return 8u;
  const float c = fminf(fmaxf(floorf(x / s + 0.5f), -8.0f), 7.0f);
  return static_cast<unsigned>(static_cast<int>(c) + 8);
}

// bit position of the word's j-th code
__device__ __forceinline__ constexpr int q4Shift(int j) { return 4 * (j >> 1) + 16 * (j & 1); }

// The constants of q4Ints in registers: as literals they would not fit one and-or instruction. Made once, at a kernel's start.
struct Q4Masks {
  unsigned low = 0x000F000Fu, high = 0x00F000F0u, magic = 0x64006400u;
  __device__ __forceinline__ Q4Masks() { asm("" : "+v"(low), "+v"(high), "+v"(magic)); }
};

// the 8 integers c - 8 of a word, in order, exact in f16: a code under the mantissa of 1024 reads 1024 + c, four bits
// higher 1024 + 16 c
__device__ __forceinline__ half8 q4Ints(unsigned w, const Q4Masks& m) {
  const half2v k0 = {static_cast<h16>(-1032.0f), static_cast<h16>(-1032.0f)};
  const half2v k1 = {static_cast<h16>(-72.0f), static_cast<h16>(-72.0f)};
  const half2v r = {static_cast<h16>(0.0625f), static_cast<h16>(0.0625f)};
  const unsigned v = w >> 8;
  const half2v a = __builtin_bit_cast(half2v, (w & m.low) | m.magic) + k0;
  const half2v b = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w & m.high) | m.magic), r, k1);
  const half2v c = __builtin_bit_cast(half2v, (v & m.low) | m.magic) + k0;
  const half2v d = __builtin_elementwise_fma(__builtin_bit_cast(half2v, (v & m.high) | m.magic), r, k1);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace lkd
