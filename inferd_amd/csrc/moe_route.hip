// Routing with a balance bias, expert groups and sigmoid scores (ifd_moe_route_ex), beside the plain softmax top-k of
// moe.hip.
//
// Per token, over its logits l_e:
//   s_e = exp(l_e - max) / sum exp(l - max)   or   1 / (1 + exp(-l_e))
//   c_e = s_e + b_e; without a bias the logit itself, which has the order of its scores
//   a group's value: its largest c, or the sum of its two largest (of s where there is no bias)
//   picks: the k largest c among the topk_group best groups; weight s / sum of the picks' s, times a scale
// Every choice is made in 64 bits, so that it is the formula's and not that of a rounding: in fp32 one token in some
// thousands has two candidates a rounding apart.
#include "common.h"
#include "f64_dev.h"
#include "host.h"
#include "kernels.h"

namespace ifd {

struct RouteExArgs {
  const void* logits;
  int T, E, k, stride;
  const float* bias;
  int groups, topk_groups, norm, shared_gate;
  float scale;
  int* idx;
  float* wt;
  float* sg;
};

// Signed keys in the order of the values (64 bits; values are not NaN, -0 never enters).
__device__ __forceinline__ int64_t key64(double v) {
  const int64_t u = __builtin_bit_cast(int64_t, v);
  return u ^ (int64_t)((uint64_t)(u >> 63) >> 1);
}
constexpr int64_t kRouteGone = INT64_MIN;  // below every value's key: picked, cut off, or past E

// One wave per token; lane l holds experts PER l .. + PER - 1 (PER = 1, 2, 4, 8 by E <= 512), so that a lane's logits are
// one load and a tie goes to the lowest lane.
template <int PER, bool BF16, bool SOFTMAX, int GTOP>
__global__ __launch_bounds__(256) void k_moe_route_ex(RouteExArgs p) {
  __shared__ double s_score[4][64 * PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x * 4 + wave;
  if (t >= p.T) return;  // no block-wide barrier follows
  const int e0 = lane * PER;
  float l[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const size_t o = (size_t)t * p.stride + min(e0 + i, p.E - 1);
    const float v = BF16 ? bf2f(((const uint16_t*)p.logits)[o]) : ((const float*)p.logits)[o];
    l[i] = order_value(e0 + i < p.E ? v : -INFINITY);
  }
  // scores. A row without a finite maximum of its own: +infinity counts as 1 (shared by all that have it), and where every
  // logit is -infinity every score is 0.
  double s[PER];
  if constexpr (SOFTMAX) {
    float mx = l[0];
#pragma unroll
    for (int i = 1; i < PER; i++) mx = fmaxf(mx, l[i]);
    mx = dpp_max_f(mx);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      s[i] = l[i] == -INFINITY ? 0.0 : l[i] == mx ? 1.0 : exp_neg((double)l[i] - mx);
      sum += s[i];
    }
    sum = dpp_sum_f64(sum);
    const double r = sum > 0 ? rcp64(sum) : 0.0;
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] *= r;
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const double x = exp_neg(-fabs((double)l[i])), r = rcp64(1 + x);
      s[i] = l[i] < 0 ? x * r : r;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; i++) s_score[wave][e0 + i] = s[i];
  int64_t key[PER];
  double c[PER];  // what the groups are ranked by
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const float b = p.bias ? order_value(p.bias[min(e0 + i, p.E - 1)]) : 0.f;
    c[i] = p.bias ? s[i] + b : GTOP == 2 ? s[i] : (double)l[i];
    key[i] = e0 + i < p.E ? key64(p.bias ? c[i] : (double)l[i]) : kRouteGone;
  }
  if (p.groups > 1) {
    const int gs = p.E / p.groups;
    double mine = -INFINITY;  // lane g: group g's value
    for (int g = 0; g < p.groups; g++) {
      // this lane's two largest values in the group
      double a = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const bool in = e0 + i >= g * gs && e0 + i < (g + 1) * gs;
        const double v = in ? c[i] : -INFINITY;
        b = fmax(b, fmin(a, v)), a = fmax(a, v);
      }
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const double a2 = __shfl_xor(a, o, 64), b2 = __shfl_xor(b, o, 64);
        b = fmax(fmin(a, a2), fmax(b, b2)), a = fmax(a, a2);
      }
      if (lane == g) mine = GTOP == 1 ? a : b == -INFINITY ? b : a + b;
    }
    int rank = 0;  // groups above this one: larger values, and equal ones of lower groups
    for (int g = 0; g < p.groups; g++) {
      const double v = readlane_f64(mine, g);
      rank += v > mine || (v == mine && g < lane);
    }
    const uint64_t keep = __ballot(lane < p.groups && rank < p.topk_groups);
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (e0 + i < p.E && !(keep >> ((e0 + i) / gs) & 1)) key[i] = kRouteGone;
  }
  int who = 0;
  for (int j = 0; j < p.k; j++) {
    int64_t best = key[0];
    int bi = 0;
#pragma unroll
    for (int i = 1; i < PER; i++)
      if (key[i] > best) best = key[i], bi = i;
    const int hi = (int)(best >> 32);
    const int hm = dpp_reduce_i(hi, INT32_MIN, [](int a, int b) { return max(a, b); });
    uint64_t hit = __ballot(hi == hm);
    if (hit & (hit - 1)) {  // equal upper halves: the lower ones decide, then the lowest lane
      const int lo = hi == hm ? (int)((uint32_t)best ^ 0x80000000u) : INT32_MIN;
      const int lm = dpp_reduce_i(lo, INT32_MIN, [](int a, int b) { return max(a, b); });
      hit = __ballot(hi == hm && lo == lm);
    }
    const int w = __ffsll((long long)hit) - 1;
    const int e = __builtin_amdgcn_readlane(e0 + bi, w);
    if (lane == j) who = e;
    if (lane == w) {
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (i == bi) key[i] = kRouteGone;
    }
  }
  __builtin_amdgcn_wave_barrier();
  // lane j < k <= 16: pick j
  const bool live = lane < p.k;
  double v = live ? s_score[wave][who] : 0.0;
  if (p.norm) {
    const double sum = dpp_sum_f64(v);
    v = sum > 0 ? v / sum : 0.0;
  }
  if (live) {
    p.idx[(size_t)t * p.k + lane] = who;
    p.wt[(size_t)t * p.k + lane] = (float)(v * (double)p.scale);
  }
  if (lane == 0) {
    float g = 1.f;
    if (p.shared_gate) {
      const size_t o = (size_t)t * p.stride + p.E;
      const double x = BF16 ? bf2f(((const uint16_t*)p.logits)[o]) : ((const float*)p.logits)[o];
      const double y = exp_neg(-fabs(x));
      g = (float)(x != x ? x : x < 0 ? y / (1 + y) : 1 / (1 + y));
    }
    p.sg[t] = g;
  }
}

template <int PER, bool BF16>
static void launch_route_per(const RouteExArgs& a, int softmax, int group_top, hipStream_t st) {
  const dim3 grid((a.T + 3) / 4), block(256);
  if (softmax) {
    if (group_top == 2) hipLaunchKernelGGL((k_moe_route_ex<PER, BF16, true, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_moe_route_ex<PER, BF16, true, 1>), grid, block, 0, st, a);
  } else {
    if (group_top == 2) hipLaunchKernelGGL((k_moe_route_ex<PER, BF16, false, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_moe_route_ex<PER, BF16, false, 1>), grid, block, 0, st, a);
  }
}
template <bool BF16>
static void launch_route_bf(const RouteExArgs& a, int softmax, int group_top, hipStream_t st) {
  if (a.E <= 64) launch_route_per<1, BF16>(a, softmax, group_top, st);
  else if (a.E <= 128) launch_route_per<2, BF16>(a, softmax, group_top, st);
  else if (a.E <= 256) launch_route_per<4, BF16>(a, softmax, group_top, st);
  else launch_route_per<8, BF16>(a, softmax, group_top, st);
}

int launch_moe_route_ex(const void* logits, int logits_bf16, int T, int E, int k, int stride, int softmax,
                        const float* bias, int groups, int topk_groups, int group_top, int norm, float scale,
                        int shared_gate, int* idx, float* wt, float* sg, hipStream_t st) {
  if (T == 0) return IFD_OK;
  const RouteExArgs a{logits, T, E, k, stride, bias, groups, topk_groups, norm, shared_gate, scale, idx, wt, sg};
  if (logits_bf16) launch_route_bf<true>(a, softmax, group_top, st);
  else launch_route_bf<false>(a, softmax, group_top, st);
  return check_launch("moe_route_ex");
}

}  // namespace ifd
