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

// 1 / d for 1 <= d <= 1e300: the reciprocal estimate and two Newton steps.
__device__ __forceinline__ double rcp64(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// A DPP move of both halves (lanes without a source keep `id`).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double id, double v) {
  const uint64_t i = __builtin_bit_cast(uint64_t, id), u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)i, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(i >> 32), (int)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Wave-wide sum, the same order in every call (see dpp_reduce_i).
__device__ __forceinline__ double dpp_sum_f64(double v) {
  v += dpp_f64<0x111, 0xf>(0.0, v);
  v += dpp_f64<0x112, 0xf>(0.0, v);
  v += dpp_f64<0x114, 0xf>(0.0, v);
  v += dpp_f64<0x118, 0xf>(0.0, v);
  v += dpp_f64<0x142, 0xa>(0.0, v);
  v += dpp_f64<0x143, 0xc>(0.0, v);
  return readlane_f64(v, 63);
}

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
