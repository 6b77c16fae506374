// What a linear's epilogue does with a sum y (fp32): act(y + bias) + residual, rounded once to the output's type.
// It rides on the products' stores (or on the sums of a split K), so it costs no pass over C: against the plain product
// 10.1 us for 9.8 (1 row, 5120 x 5120, bias and residual), 28.6 for 28.2 (12 rows, 8-bit, 17408 x 5120, bias and SILU), 18.9
// for 18.6 (32 rows, 17408 x 5120, bias and GELU_TANH), 155 for 158 of the product with mode 1 (777 rows, 5120 x 17408, bias
// and residual).
#pragma once
#include "common.h"

namespace ifd {

// A row of a K split's partials in the decode GEMV with an epilogue: whole 16-byte quads.
__host__ __device__ inline int epi_part_row(int N) { return (N + 3) / 4 * 4; }

enum EpiAct { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

struct Epi {
  const uint16_t* bias = nullptr;  // bf16 [N], or null
  const uint16_t* res = nullptr;   // bf16 [M][ldr], or null; may be C itself
  int ldr = 0;
  int act = kActNone;
  int f32 = 0;  // C is fp32, else bf16
};

// 2^x and 1 / x to one unit in the last place by the hardware's estimates (results below 2^-126 are 0). Off the device
// (the tests run some kernels' source on the host) the library's.
#ifdef __HIP__
__device__ __forceinline__ float epi_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float epi_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
#else
inline float epi_exp2(float x) { return exp2f(x); }
inline float epi_rcp(float x) { return 1.f / x; }
#endif

// The activations in as few instructions as fp32 takes (an epilogue of a GEMM whose waves stand alone on their SIMD pays
// about 5 cycles for each): 5 for SILU, 7 for GELU_TANH, 15 for GELU. Infinities and NaN as the formulas have them.
__device__ __forceinline__ float act_silu(float x) { return x * epi_rcp(1.f + epi_exp2(x * -1.44269504f)); }
// x / (1 + exp(-2 sqrt(2 / pi) (x + 0.044715 x^3)))
__device__ __forceinline__ float act_gelu_tanh(float x) {
  return x * epi_rcp(1.f + epi_exp2(x * __builtin_fmaf(x * x, -0.102943240f, -2.30220819f)));
}
// x Phi(x): with t = 1 / (1 + p z), z = |x| / sqrt 2, Phi(-|x|) = exp(-z^2) t (a1 + t (a2 + ..)) / 2 to 7.5e-8
// (Abramowitz and Stegun 7.1.26). The error falls with exp(-z^2): relative to the value 5e-5 at x = -3, 1.6e-3 at -5, 3.6e-3 at -6
// (half a bf16 step is 3.9e-3, and the value 6e-9).
__device__ __forceinline__ float act_gelu(float x) {
  const float t = epi_rcp(__builtin_fmaf(fabsf(x), 0.3275911f * 0.707106781f, 1.f));
  float q = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = __builtin_fmaf(q, t, 0.5f * 1.421413741f);
  q = __builtin_fmaf(q, t, 0.5f * -0.284496736f);
  q = __builtin_fmaf(q, t, 0.5f * 0.254829592f);
  q = q * t * epi_exp2(x * x * (-0.5f * 1.44269504f));
  return x * (x < 0.f ? q : 1.f - q);
}

// act is uniform over a launch: one branch for all N values. CLASS: the activations that are compiled in (kEpiAny, or one
// of the others, by epi_class): a kernel that unrolls its epilogue over many registers takes one class.
enum EpiClass { kEpiLinear, kEpiSigmoid, kEpiErf, kEpiAny };
__host__ __device__ inline int epi_class(int act) {
  return act <= kActRelu ? kEpiLinear : act == kActGelu ? kEpiErf : kEpiSigmoid;
}
template <int N, int CLASS = kEpiAny>
__device__ __forceinline__ void epi_act(float (&v)[N], int act) {
  constexpr bool any = CLASS == kEpiAny;
  if ((any || CLASS == kEpiLinear) && act == kActNone) return;
  if ((any || CLASS == kEpiLinear) && act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = v[i] < 0.f ? 0.f : v[i];
  } else if ((any || CLASS == kEpiSigmoid) && act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = act_silu(v[i]);
  } else if ((any || CLASS == kEpiErf) && act == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = act_gelu(v[i]);
  } else if (any || CLASS == kEpiSigmoid) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = act_gelu_tanh(v[i]);
  }
}

// N values of one row from column col on (o: the first's place in C), of which n lie in the row.
template <int N>
__device__ __forceinline__ void epi_store(const Epi& e, void* C, size_t o, int row, int col, int n, float (&v)[N]) {
  float b[N], r[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    b[i] = e.bias && i < n ? bf2f(e.bias[col + i]) : 0.f;
    r[i] = e.res && i < n ? bf2f(e.res[(size_t)row * e.ldr + col + i]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < N; i++) v[i] += b[i];
  epi_act(v, e.act);
#pragma unroll
  for (int i = 0; i < N; i++)
    if (i < n) store_mode(C, o + i, e.res ? v[i] + r[i] : v[i], e.f32 ? 2 : 0);
}

}  // namespace ifd
