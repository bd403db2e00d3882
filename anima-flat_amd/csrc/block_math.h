// Device arithmetic shared by the block's operators (adaln.hip, int8_rows.hip,
// ckpt8.hip): wave reductions in the vector ALU, GELU, 8-bit encodings.
#pragma once

#include "aa_common.h"

namespace aa {

// Reductions over the 64 lanes of a wave that leave the result in every lane:
// four DPP rotations inside the rows of 16 lanes, then the permlane swaps
// across rows. No LDS access (a ds_bpermute per step costs about 10 times a
// DPP move's latency, and a row's norm needs two to four reductions in a row).
// Every step combines the same two values in both lanes of a pair, so all
// lanes end with the same bits.
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_mov(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, false);
}
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e;  // quad_perm [1 0 3 2], [2 3 0 1]
constexpr int kDppRor = 0x120;                   // row_ror:n is kDppRor + n

template <class Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t x, Op op) {
  x = op(x, dpp_mov<kDppRor + 8>(x));
  x = op(x, dpp_mov<kDppRor + 4>(x));
  x = op(x, dpp_mov<kDppRor + 2>(x));
  x = op(x, dpp_mov<kDppRor + 1>(x));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return op(b[0], b[1]);
}
__device__ __forceinline__ float wave_sum(float x) {
  return __uint_as_float(wave_reduce(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  return wave_reduce(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// Magnitudes are compared as bit patterns: among non-negative floats the order
// is the same, and a NaN stands above infinity instead of being dropped.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// GELU(x) = x Phi(x) with Phi the normal distribution function. For a = |x|
//   Q(a) = 1 - Phi(a) = exp(-a^2 / 2) F(a),  F(a) = erfcx(a / sqrt 2) / 2,
// and F(a) = t P(t) with t = 1 / (1 + 0.31 a): P is a polynomial of degree 5
// fitted to a relative error of 4.7e-6 over 0 <= a <= 14 (minimax, by linear
// programming against scipy's erfcx), below which Q is under 2^-126. The error
// is relative, so that the lower tail of GELU keeps its digits; it is a
// hundredth of a bf16 rounding (2^-9).
struct Phi {
  float p;  // Phi(x)
  float e;  // exp(-x^2 / 2)
};
__device__ __forceinline__ Phi normal_cdf(float x) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.31f, fabsf(x), 1.0f));
  const float e = __builtin_amdgcn_exp2f((x * x) * (-0.5f * kLog2e));
  float f = fmaf(t, -0.07393838465213776f, 0.18047693371772766f);
  f = fmaf(t, f, 0.01571611687541008f);
  f = fmaf(t, f, 0.13344404101371765f);
  f = fmaf(t, f, 0.12043801695108414f);
  f = fmaf(t, f, 0.12386097013950348f);
  const float q = f * t * e;
  return {x < 0.f ? q : 1.0f - q, e};
}
// x Phi(x); -inf gives its limit 0 (the product alone would be -inf * 0).
__device__ __forceinline__ float gelu(float x) {
  return fmaxf(x, -0x1p+100f) * normal_cdf(x).p;
}
// d GELU / dx = Phi(x) + x phi(x), phi(x) = exp(-x^2 / 2) / sqrt(2 pi).
__device__ __forceinline__ float gelu_slope(float x) {
  const Phi n = normal_cdf(x);
  return fmaf(x * 0.3989422804014327f, n.e, n.p);
}

// The low byte of the result's bits is round-to-nearest-even(x) in two's
// complement for |x| <= 127: adding 1.5 * 2^23 leaves the integer in the low
// mantissa bits.
__device__ __forceinline__ uint32_t round_bits(float x) { return __float_as_uint(x + 12582912.0f); }
// The low bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
  const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return ab | cd;
}

// Per-token int8 codes: with s = max(max |y|, 1e-12) / 127, the code of y is
// round-to-nearest-even(y / s), |code| <= 127. The quotient is rounded
// correctly before it is rounded to an integer, as a division would (ties of
// the second rounding would otherwise fall either way): from the correctly
// rounded reciprocal, q0 = RN(y rcp), e = y - q0 s exact in an FMA, and
// RN(q0 + e rcp) is the quotient (Markstein) as long as no remainder
// underflows, which holds for max |y| >= 2^-60 where it decides a code.
// A row with a value that is not finite has the scale NaN and codes 0.
struct RowScale {
  float s, rcp;
  bool divide;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  RowScale r;
  r.s = amax_bits >= kInfBits ? __builtin_nanf("") : fmaxf(amax, 1e-12f) / 127.0f;
  r.rcp = 1.0f / r.s;
  r.divide = amax < 0x1p-60f;
  return r;
}
template <bool kDivide>
__device__ __forceinline__ uint32_t int8_code(float y, const RowScale& r) {
  float t;
  if constexpr (kDivide) {
    t = y / r.s;
  } else {
    const float q0 = y * r.rcp;
    t = fmaf(fmaf(-q0, r.s, y), r.rcp, q0);
  }
  return round_bits(t);
}
// Eight values' codes. NaN scale: every quotient is NaN, whose bits + magic
// have a zero low byte (the quiet NaN 0x7fc00000).
__device__ __forceinline__ u32x2 int8_codes8(const float* y, const RowScale& r) {
  uint32_t c[8];
  if (r.divide) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = int8_code<true>(y[i], r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = int8_code<false>(y[i], r);
  }
  return u32x2{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}

}  // namespace aa
