// Device helpers in 64 bits for choices that hang on values next to a border (routing, sampling).
#pragma once
#include "common.h"

namespace ifd {

// exp(x) for x <= 0 (NaN: NaN), relative error below 1e-15: Cody and Waite's reduction x = n ln 2 + r, |r| <= ln 2 / 2, with ln 2 in
// two parts (its first 32 bits, so that n times them is exact, and the rest), and the Taylor polynomial of exp(r) to degree 12 (its remainder 1.7e-16).
__device__ __forceinline__ double exp_neg(double x) {
  const double n = __builtin_rint(fmax(x, -1100.0) * 1.4426950408889634074);
  double r = __builtin_fma(-n, 0.6931471806019545, fmax(x, -1100.0));
  r = __builtin_fma(-n, -4.2009150726810846e-11, r);
  double p = 1.0 / 479001600;
  p = __builtin_fma(p, r, 1.0 / 39916800);
  p = __builtin_fma(p, r, 1.0 / 3628800);
  p = __builtin_fma(p, r, 1.0 / 362880);
  p = __builtin_fma(p, r, 1.0 / 40320);
  p = __builtin_fma(p, r, 1.0 / 5040);
  p = __builtin_fma(p, r, 1.0 / 720);
  p = __builtin_fma(p, r, 1.0 / 120);
  p = __builtin_fma(p, r, 1.0 / 24);
  p = __builtin_fma(p, r, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// 2^y for y <= 0 as a whole number of 2^-44 (NaN and y < -64: 0), from 2^y to 4e-14: the nearest whole number n of y (the low
// bits of y + 44 + 1.5 2^52) and a polynomial of degree 9 on [-1/2, 1/2] that takes 2^r - 1 over r at the Chebyshev points;
// n + 44 is added to the exponent, and the sum with 2^52 has the result in its low bits. Conversions and ldexp run at a quarter
// of the rate of these. 2^0 is 2^44 exactly.
__device__ __forceinline__ uint64_t exp2_fixed44(double y) {
  constexpr double kRound = 0x1.8p52 + 44;
  y = fmax(y, -64.0);
  const double m = y + kRound, r = y - (m - kRound);
  double p = 1.0203121063391729e-07;
  p = __builtin_fma(p, r, 1.3255224878668817e-06);
  p = __builtin_fma(p, r, 1.525268684626772e-05);
  p = __builtin_fma(p, r, 0.00015403455852453838);
  p = __builtin_fma(p, r, 0.0013333558179043112);
  p = __builtin_fma(p, r, 0.009618129159402558);
  p = __builtin_fma(p, r, 0.055504108664760424);
  p = __builtin_fma(p, r, 0.2402265069581299);
  p = __builtin_fma(p, r, 0.6931471805599453);
  p = __builtin_fma(p, r, 1.0);
  u32x2 q = __builtin_bit_cast(u32x2, p);
  q[1] += __builtin_bit_cast(u32x2, m)[0] << 20;
  q = __builtin_bit_cast(u32x2, __builtin_bit_cast(double, q) + 0x1p52);
  q[1] &= 0xfffffu;
  return __builtin_bit_cast(uint64_t, q);
}

// 1 / d for 1 <= d <= 1e300: the reciprocal estimate and two Newton steps.
__device__ __forceinline__ double rcp64(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// 64-bit values across lanes. A DPP move of both halves (lanes without a source get `id`):
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t id, uint64_t v) {
  const u32x2 i = __builtin_bit_cast(u32x2, id), u = __builtin_bit_cast(u32x2, v);
  u32x2 r;
  r[0] = (uint32_t)__builtin_amdgcn_update_dpp((int)i[0], (int)u[0], CTRL, ROWS, 0xf, false);
  r[1] = (uint32_t)__builtin_amdgcn_update_dpp((int)i[1], (int)u[1], CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(uint64_t, r);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double id, double v) {
  return __builtin_bit_cast(double, dpp_u64<CTRL, ROWS>(__builtin_bit_cast(uint64_t, id), __builtin_bit_cast(uint64_t, v)));
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int lane) {
  const u32x2 u = __builtin_bit_cast(u32x2, v);
  u32x2 r;
  r[0] = (uint32_t)__builtin_amdgcn_readlane((int)u[0], lane);
  r[1] = (uint32_t)__builtin_amdgcn_readlane((int)u[1], lane);
  return __builtin_bit_cast(uint64_t, r);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  return __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, v), lane));
}
// Inclusive prefix sums over a wave (the steps of dpp_reduce_i, which leave each lane the sum up to it).
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v += dpp_u64<0x111, 0xf>(0, v);
  v += dpp_u64<0x112, 0xf>(0, v);
  v += dpp_u64<0x114, 0xf>(0, v);
  v += dpp_u64<0x118, 0xf>(0, v);
  v += dpp_u64<0x142, 0xa>(0, v);
  return v + dpp_u64<0x143, 0xc>(0, v);
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v += dpp_f64<0x111, 0xf>(0.0, v);
  v += dpp_f64<0x112, 0xf>(0.0, v);
  v += dpp_f64<0x114, 0xf>(0.0, v);
  v += dpp_f64<0x118, 0xf>(0.0, v);
  v += dpp_f64<0x142, 0xa>(0.0, v);
  return v + dpp_f64<0x143, 0xc>(0.0, v);
}
__device__ __forceinline__ double dpp_sum_f64(double v) { return readlane_f64(wave_scan_f64(v), 63); }
__device__ __forceinline__ uint64_t dpp_sum_u64(uint64_t v) { return readlane_u64(wave_scan_u64(v), 63); }

// Unsigned keys in the order of the values; -0 as +0, NaN as -infinity.
__device__ __forceinline__ float order_value(float v) { return v != v ? -INFINITY : v + 0.f; }
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(order_value(v));
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

}  // namespace ifd
