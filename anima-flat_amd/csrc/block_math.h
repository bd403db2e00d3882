// Device arithmetic shared by the block's operators (adaln.hip, int8_linear.hip,
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

// max(a, |b|, |c|) that is NaN if one of them is.
__device__ __forceinline__ float max3abs_nan(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Magnitudes are compared as bit patterns: among non-negative floats the order
// is the same, and a NaN stands above infinity instead of being dropped.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// GELU(x) = x Phi(x) with Phi the normal distribution function. For a = |x|
//   Q(a) = 1 - Phi(a) = exp(-a^2 / 2) F(a),  F(a) = erfcx(a / sqrt 2) / 2,
// and F(a) = t P(t) with t = 1 / (1 + 0.3625 a): P is a polynomial of degree 6
// fitted to a relative error of 7.7e-7 over 0 <= a <= 14 (minimax, by linear
// programming against scipy's erfcx), below which Q is under 2^-126; 1.0e-6 with
// fp32 rounding. The error is relative, so that the lower tail of GELU keeps its
// digits. Then, for either sign of x,
//   GELU(x) = max(x, 0) - a Q(a).
// 14 vector instructions and two transcendental ones a value. Degree 4 (3.1e-5, 12
// instructions) moved 1% of the results to the other side of a bf16 rounding.
struct Tail {
  float a;  // |x|, or 2^100
  float f;  // Q / e
  float e;  // exp(-x^2 / 2); NaN for NaN
};
__device__ __forceinline__ Tail normal_tail(float x) {
  // Bounded so that infinity times Q's zero is no NaN. (fminf and fmaxf would
  // quiet their operand first, an instruction each; NaN comes through e.)
  const float a = __builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.f, 0x1p+100f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3625f, a, 1.0f));
  const float e = __builtin_amdgcn_exp2f((x * (-0.5f * kLog2e)) * x);
  float f = fmaf(t, 0.04806283116340637f, -0.17974217236042023f);
  f = fmaf(t, f, 0.17510363459587097f);
  f = fmaf(t, f, 0.029682673513889313f);
  f = fmaf(t, f, 0.13925662636756897f);
  f = fmaf(t, f, 0.14293640851974487f);
  f = fmaf(t, f, 0.14470037817955017f);
  return {a, f * t, e};
}
__device__ __forceinline__ float gelu(float x) {
  const Tail n = normal_tail(x);
  return fmaf(-n.a, n.f * n.e, __builtin_amdgcn_fmed3f(x, 0.f, __builtin_inff()));
}
// d GELU / dx = Phi(x) + x phi(x), phi(x) = exp(-x^2 / 2) / sqrt(2 pi): with
// d = Q(a) - a phi(a), it is d for negative x and 1 - d otherwise.
__device__ __forceinline__ float gelu_slope(float x) {
  const Tail n = normal_tail(x);
  const float d = fmaf(-0.3989422804014327f, n.a, n.f) * n.e;
  return x < 0.f ? d : 1.0f - d;
}

// GELU for 8-bit codes whose step is at least 1e-12 / 127: log2 Q(a) is a polynomial of
// degree 8 up to a = 9 (minimax, by linear programming against scipy's log_ndtr: 6e-6 of
// Q, 1.4e-5 with fp32 rounding), where a Q is under 2e-18, far below half a step, and
// stays there. 1 code in 10^6 of normal rows is another than the 64-bit formula's. One
// transcendental instruction and 11 others a value against the two and 14 above: the row
// quantiser is bound by them (degree 10, 1.3e-6 near 0, took 3 to 7% longer). NaN comes
// through the maximum.
__device__ __forceinline__ float gelu_coarse(float x) {
  const float a = __builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.f, 9.0f);
  float p = fmaf(a, 7.462385553935746e-08f, -3.6554802136379294e-06f);
  p = fmaf(p, a, 7.943361561046913e-05f);
  p = fmaf(p, a, -0.001020022202283144f);
  p = fmaf(p, a, 0.008750777691602707f);
  p = fmaf(p, a, -0.05430452153086662f);
  p = fmaf(p, a, -0.4582415819168091f);
  p = fmaf(p, a, -1.1512950658798218f);
  p = fmaf(p, a, -0.999996542930603f);
  float top;
  asm("v_maximum3_f32 %0, %1, 0, 0" : "=v"(top) : "v"(x));
  return fmaf(-a, __builtin_amdgcn_exp2f(p), top);
}

// x + kRoundMagic for |x| <= 127, rounded to nearest even, has round(x) in two's
// complement in the low byte of its bits: 1.5 * 2^23 leaves the integer in the
// low mantissa bits.
constexpr float kRoundMagic = 12582912.0f;
// The low bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
  const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return ab | cd;
}

// Per-token int8 codes: with m = max(max |y|, 1e-12) the scale is m / 127, rounded to
// fp32, and the code of y is round-to-nearest-even(127 y / m): from one FMA with the
// row's rcp, 127 / m rounded up to fp32, whose product with y is exact in it.
// For a bf16 y that is the rule's code in exact arithmetic, ties included. 127 y / m is
// either a tie or 2^-17 away from one, relatively (8-bit mantissas), far more than rcp's
// 2^-23. Ties are y = +-m / 2, 63.5, where the rounding up leaves a product of at
// least that, so 64, the even one; and rows with 127 in m, where rcp is a power of
// two and exact. (With 1 / s rounded either way instead, half of the values at m / 2,
// up to 0.1% of a row, got 63.) An fp32 y's code is the rule's unless its quotient is
// within 2^-16 of a half. |y rcp| <= 127 (1 + 2^-22), so |code| <= 127. A row with a
// value that is not finite has the scale NaN and codes 0 (NaN + magic is 0x7fc00000).
struct RowScale {
  float s, rcp;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const float m = fmaxf(__uint_as_float(amax_bits), 1e-12f);
  RowScale r;
  r.s = m / 127.0f;
  r.rcp = 127.0f / m;  // rounded to nearest: the FMA's sign says which way
  if (fmaf(r.rcp, m, -127.0f) < 0.f) r.rcp = __uint_as_float(__float_as_uint(r.rcp) + 1u);
  if (amax_bits >= kInfBits) r.s = r.rcp = __builtin_nanf("");
  return r;
}
__device__ __forceinline__ u32x2 int8_codes8(const float* y, const RowScale& r) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(fmaf(y[i], r.rcp, kRoundMagic));
  return u32x2{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}

}  // namespace aa
