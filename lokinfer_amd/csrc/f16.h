// Device helpers shared by the f16 kernels: types, the contract's roundings, RMSNorm and RoPE arithmetic in the one order
// that every kernel using them keeps (so fused ops and their compositions give the same bits).
#pragma once

#include "common.h"

// No fp contraction from here on (every intended fma is an explicit fmaf).
#pragma clang fp contract(off)

namespace lkd {

typedef _Float16 h16;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));


// The contract's output rounding: the f32 result, then f16. The empty asm makes the f32 value opaque, so the compiler
// cannot fold the operation producing it and the conversion into one mixed-precision instruction (v_fma_mix*),
// which rounds once, straight to f16, and differs near f16 midpoints; fused ops and their compositions then round
// alike.
__device__ __forceinline__ h16 toH16(float v) {
  asm volatile("" : "+v"(v));
  return static_cast<h16>(v);
}

__device__ __forceinline__ half8 ld8(const h16* p) { return *reinterpret_cast<const half8*>(p); }
// weight rows streamed once per call (decode GEMVs: gigabytes per token, far above the last-level cache)
__device__ __forceinline__ half8 ldStream8(const h16* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const half8*>(p));
}
__device__ __forceinline__ void st8(h16* p, half8 v) { *reinterpret_cast<half8*>(p) = v; }

// Sum of squares of a row of k values (k % 8 == 0, 16-byte aligned) over one wave.
__device__ __forceinline__ float rowSumSq(const h16* x, int64_t k, int lane) {
  float s = 0.0f;
  for (int64_t c = lane; c < k / 8; c += 64) {
    const half8 v = ld8(x + 8 * c);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(static_cast<float>(v[e]), static_cast<float>(v[e]), s);
  }
  return waveSum(s);
}

__device__ __forceinline__ float rmsFactor(float sumSq, int64_t k, float eps) {
  return 1.0f / sqrtf(sumSq / static_cast<float>(k) + eps);
}

// HF Qwen3RMSNorm with the contract's roundings: h = f16(x r), y = f16(g h)
__device__ __forceinline__ h16 rmsElem(h16 x, h16 g, float r) {
  const h16 h = toH16(static_cast<float>(x) * r);
  return toH16(static_cast<float>(g) * static_cast<float>(h));
}

// ---- RoPE: angle = f32(p) * invFreq[j] (f32 product), cos / sin of it in double, rounded to f32 ------------
struct RopeTable {
  float invf[64];
};

__device__ __forceinline__ void ropeAngle(int64_t p, float invf, float& c, float& s) {
  const float ang = static_cast<float>(p) * invf;
  double sd, cd;
  sincos(static_cast<double>(ang), &sd, &cd);  // one routine in every kernel (the compiler may merge sin + cos)
  c = static_cast<float>(cd), s = static_cast<float>(sd);
}

__device__ __forceinline__ void ropeRotate(float lo, float hi, float c, float s, h16& olo, h16& ohi) {
  // explicit fma forms: every kernel that rotates computes the same bits (no contraction choice left to the
  // compiler, which could fuse either product)
  olo = toH16(fmaf(lo, c, -(hi * s)));
  ohi = toH16(fmaf(hi, c, lo * s));
}

__device__ __forceinline__ void ropePair(float lo, float hi, int64_t p, float invf, h16& olo, h16& ohi) {
  float c, s;
  ropeAngle(p, invf, c, s);
  ropeRotate(lo, hi, c, s, olo, ohi);
}

__device__ __forceinline__ float siluMul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

typedef h16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// 4 consecutive rows x 16 consecutive halves per 16 lanes, transposed: lane i passes the address of row i / 4,
// halves 4 (i % 4) .. and gets the 4 rows' values of half i
__device__ __forceinline__ half4 ldsTranspose4(const h16* a) {
  typedef short short4v __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4v* Lds;
  return __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (Lds)(reinterpret_cast<short4v*>(const_cast<h16*>(a)))));
}

}  // namespace lkd
