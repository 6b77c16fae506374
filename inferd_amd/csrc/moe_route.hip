// Routing with a balance bias, expert groups and sigmoid scores (ifd_moe_route_ex), beside the plain softmax top-k of
// moe.hip.
//
// Per token, over its logits l_e:
//   s_e = exp(l_e - max) / sum exp(l - max)   or   1 / (1 + exp(-l_e))
//   c_e = s_e + b_e; without a bias the logit itself, which has the order of its scores
//   a group's value: its largest c, or the sum of its two largest (of s where there is no bias)
//   picks: the k largest c among the topk_group best groups; weight s / sum of the picks' s, times a scale
// Every choice is that of the formula in 64 bits, and not that of a rounding: in fp32 one token in some thousands has two
// candidates a rounding apart.
//
// k_moe_route_fast takes the k + 1 largest in fp32, and where two neighbours among them are within the error of the fp32
// scores (one token in some hundreds) orders them anew by their scores in 64 bits. Where that does not settle it (the next
// one is as near to the last pick, or a group that stays to one that does not: one token in ten thousands) the token is done
// again in 64 bits by a whole wave, with the code of k_moe_route_ex. Without a bias the logits themselves are compared.
//
// What bounds it: up to some hundreds of tokens a launch and one token's chain of loads, sort and k + 1 rounds (1 token of
// 512 experts 7.5 us a call, 16 of 256 in 8 groups 7.9); then issue: about 350 vector instructions per token (16384 tokens of
// 256 in 8 groups, bf16: 15 to 16.5 us, 0.55 TB/s, where the bytes alone take 1.9). All in 64 bits by a wave per token they
// took 12.5, 13.2 and 41.8 us.
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

// LDS written by other lanes of this wave is read after it (a wave's LDS operations are in order: no instruction).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Signed keys in the order of the values (64 bits; values are not NaN, -0 never enters).
__device__ __forceinline__ int64_t key64(double v) {
  const int64_t u = __builtin_bit_cast(int64_t, v);
  return u ^ (int64_t)((uint64_t)(u >> 63) >> 1);
}
constexpr int64_t kRouteGone = INT64_MIN;  // below every value's key: picked, cut off, or past E

// One token by one wave; lane l holds experts PER l .. + PER - 1 (PER = 1, 2, 4, 8 by E <= 512), so that a lane's logits are
// one load and a tie goes to the lowest lane.
template <int PER, bool BF16, bool SOFTMAX, int GTOP>
__device__ __forceinline__ void route_exact(const RouteExArgs& p, int t, double* score) {
  const int lane = threadIdx.x & 63;
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
  for (int i = 0; i < PER; i++) score[e0 + i] = s[i];
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
  wave_fence();
  // lane j < k <= 16: pick j
  const bool live = lane < p.k;
  double v = live ? score[who] : 0.0;
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

template <int PER, bool BF16, bool SOFTMAX, int GTOP>
__global__ __launch_bounds__(256) void k_moe_route_ex(RouteExArgs p) {
  __shared__ double score[4][64 * PER];
  const int wave = threadIdx.x >> 6, t = blockIdx.x * 4 + wave;
  if (t < p.T) route_exact<PER, BF16, SOFTMAX, GTOP>(p, t, score[wave]);  // no block-wide barrier in it
}

// ---- several tokens per wave, in fp32 ------------------------------------------------------------------------------
// LPR lanes per token (16, 32 or 64), lane c of them holding experts PER c .. + PER - 1 (PER <= 16).

// Reductions over a token's lanes, every lane getting the result: rotations by 8, 4, 2, 1 within 16 lanes, then rows of 16
// and halves exchanged.
template <int LPR, class Op>
__device__ __forceinline__ uint32_t all_lanes(uint32_t v, Op op) {
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  v = op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
  if constexpr (LPR >= 32) {
    const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(x[0], x[1]);
  }
  if constexpr (LPR == 64) {
    const auto x = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(x[0], x[1]);
  }
  return v;
}
template <int LPR>
__device__ __forceinline__ uint32_t all_max(uint32_t v) {
  return all_lanes<LPR>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int LPR>
__device__ __forceinline__ float all_max_f(float v) {
  return __uint_as_float(all_lanes<LPR>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int LPR>
__device__ __forceinline__ float all_sum_f(float v) {
  return __uint_as_float(all_lanes<LPR>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
// The sum over 16 lanes, in all of them.
__device__ __forceinline__ double row_sum_f64(double v) {
  v += dpp_f64<0x128, 0xf>(0.0, v);
  v += dpp_f64<0x124, 0xf>(0.0, v);
  v += dpp_f64<0x122, 0xf>(0.0, v);
  return v + dpp_f64<0x121, 0xf>(0.0, v);
}

// PER values of a row from column col on, as they are (a lane that reaches past E: -infinity there).
template <int PER, class T>
__device__ __forceinline__ void load_run(const T* row, int col, int E, T pad, T (&v)[PER]) {
  typedef T V __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
  if (col + PER <= E) {
    const V x = *(const V*)(row + col);
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = x[i];
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = col + i < E ? row[min(col + i, E - 1)] : pad;
  }
}

// Falling order of N values by Batcher's odd-even merges.
template <int N>
__device__ __forceinline__ void sort_falling(uint32_t (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; i++)
          if (j + i + k < N && (j + i) / (2 * p) == (j + i + k) / (2 * p)) {
            const uint32_t x = v[j + i], y = v[j + i + k];
            v[j + i] = max(x, y), v[j + i + k] = min(x, y);
          }
}

// Whether two fp32 choices, or sums of two, may be in the other order. A sigmoid is off by less than 2^-22 (the exponential's
// argument and its last place, the reciprocal's), a softmax by less than 2^-19 of the largest one, `top` (21 additions more; the
// argument's rounding grows with it, but less than the exponential falls); the bias's addition and that of a group's two values
// by 2^-24 of their result; the last four bits of a key hide 2^-19 of a value. Equal infinities are exact.
template <bool SOFTMAX, bool KEYS>
__device__ __forceinline__ bool too_near(float hi, float lo, float top) {
  const float m = __builtin_fmaf(fabsf(hi) + fabsf(lo), KEYS ? 0x1p-18f : 0x1p-23f, SOFTMAX ? 0x1p-16f * top : 0x1p-20f);
  return !(hi - lo > m) && !(hi == lo && fabsf(hi) == INFINITY);
}

// A lane's choices become 32-bit keys in the order of the values whose last four bits hold 15 - i, so that a sort takes two
// instructions per exchange; the lanes' sorted keys lie in LDS, and each round takes the largest head by its upper 28 bits, the
// lowest lane's where they are equal. That is exact for bf16 logits without a bias; else a gap that the four bits might hide
// is a near one.
template <int LPR, int PER, bool BF16, bool SOFTMAX, int GTOP>
__global__ __launch_bounds__(256) void k_moe_route_fast(RouteExArgs p) {
  static_assert(PER <= 16 && LPR >= 16, "four bits for a lane's experts, a lane for each of 16 picks");
  constexpr int RW = 64 / LPR;  // tokens per wave
  constexpr uint64_t kLanes = LPR == 64 ? ~0ull : (1ull << (LPR % 64)) - 1;
  // per wave: the tokens' choices (for the groups), then their lanes' sorted keys [PER][64], or a token's scores in 64 bits
  __shared__ __align__(16) uint64_t mem[4][64 * PER];
  __shared__ int s_pick[4][RW][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane / LPR, c = lane % LPR, e0 = c * PER;
  const int t0 = (blockIdx.x * 4 + wave) * RW, t = t0 + r;
  if (t0 >= p.T) return;  // no block-wide barrier follows
  const size_t row = (size_t)min(t, p.T - 1) * p.stride;
  float bias[PER];
  if (p.bias) load_run<PER, float>(p.bias, e0, p.E, -INFINITY, bias);
  float l[PER];
  if constexpr (BF16) {
    uint16_t h[PER];
    load_run<PER, uint16_t>((const uint16_t*)p.logits + row, e0, p.E, 0xff80u, h);
#pragma unroll
    for (int i = 0; i < PER; i++) l[i] = bf2f(h[i]);
  } else {
    load_run<PER, float>((const float*)p.logits + row, e0, p.E, -INFINITY, l);
  }
#pragma unroll
  for (int i = 0; i < PER; i++) l[i] = fmaxf(l[i], -INFINITY) + 0.f;  // NaN: -infinity; -0: +0
  const bool scores = p.bias != nullptr || (p.groups > 1 && GTOP == 2);
  float mx = 0.f, top = 1.f, s[PER];  // the largest logit and score
  if constexpr (SOFTMAX) {
    mx = l[0];
#pragma unroll
    for (int i = 1; i < PER; i++) mx = fmaxf(mx, l[i]);
    mx = all_max_f<LPR>(mx);
  }
  if (scores) {
    if constexpr (SOFTMAX) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        s[i] = l[i] == mx ? 1.f : __builtin_amdgcn_exp2f((l[i] - mx) * 1.44269504f);
        sum += e0 + i < p.E ? s[i] : 0.f;
      }
      const float rs = mx == -INFINITY ? 0.f : __builtin_amdgcn_rcpf(all_sum_f<LPR>(sum));
#pragma unroll
      for (int i = 0; i < PER; i++) s[i] *= rs;
      top = rs;
    } else {
#pragma unroll
      for (int i = 0; i < PER; i++) s[i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(l[i] * -1.44269504f));
    }
  }
  // v: what is compared
  float v[PER];
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = s[i] + (fmaxf(bias[i], -INFINITY) + 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < PER; i++) v[i] = l[i];
  }
  bool redo_me = false;
  uint32_t gone = 0;  // bit i: expert e0 + i is cut off
  if (p.groups > 1) {
    // every group by q = 2^n of the token's lanes, through LDS: whatever the groups' size
    const int gs = p.E / p.groups, q = 1 << (31 - __builtin_clz(LPR / p.groups)), g = c / q, part = c % q;
    float* const ch = (float*)mem[wave] + r * (LPR * PER);
#pragma unroll
    for (int i = 0; i < PER; i++) ch[e0 + i] = GTOP == 2 && !p.bias ? s[i] : v[i];
    wave_fence();
    float a = -INFINITY, b = -INFINITY;  // the two largest
    for (int i0 = 0; i0 < gs; i0 += 8 * q) {  // eight reads in flight
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; u++) x[u] = ch[min(g, p.groups - 1) * gs + min(i0 + q * u + part, gs - 1)];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        x[u] = i0 + q * u + part < gs ? x[u] : -INFINITY;
        b = __builtin_amdgcn_fmed3f(a, b, x[u]), a = fmaxf(a, x[u]);
      }
    }
    for (int o = 1; o < q; o *= 2) {
      const float a2 = __shfl_xor(a, o, 64), b2 = __shfl_xor(b, o, 64);
      b = fmaxf(fminf(a, a2), fmaxf(b, b2)), a = fmaxf(a, a2);
    }
    const float mine = GTOP == 1 ? a : b == -INFINITY ? b : a + b;
    int rank = 0;
    for (int o0 = 0; o0 < p.groups; o0 += 4) {
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; u++) x[u] = __shfl(mine, r * LPR + min((o0 + u) * q, LPR - 1), 64);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int og = o0 + u;
        const bool other = og < p.groups && og != g;
        rank += other && (x[u] > mine || (x[u] == mine && og < g));
      }
    }
    if (p.bias || GTOP == 2) {  // a group that stays against those that do not
      const float out = all_max_f<LPR>(g < p.groups && rank >= p.topk_groups ? mine : -INFINITY);
      redo_me = g < p.groups && rank < p.topk_groups && p.topk_groups < p.groups && too_near<SOFTMAX, false>(mine, out, top);
    }
    const uint64_t keep = __ballot(g < p.groups && rank < p.topk_groups) >> (r * LPR);
    int eg = e0 / gs, left = gs - e0 % gs;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      gone |= (keep >> (min(eg, p.groups - 1) * q) & 1) ? 0u : 1u << i;
      if (--left == 0) eg++, left = gs;
    }
    wave_fence();
  }
  uint32_t x[PER];  // 0: cut off, or past E (below every value's key)
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const uint32_t u = __float_as_uint(v[i]);
    const uint32_t k = (u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) & ~15u;
    x[i] = e0 + i < p.E && !(gone >> i & 1) ? k | (15u - i) : 0u;
  }
  sort_falling<PER>(x);
  uint32_t* const sorted = (uint32_t*)mem[wave] + lane;
#pragma unroll
  for (int i = 1; i < PER; i++) sorted[64 * i] = x[i];
  wave_fence();
  uint32_t head = x[0], picked = 0, m = 0, last = 0, rest = 0;  // keys: of the c-th largest, of the k-th, the one behind it
  int next = 1;
  const uint64_t below = ((1ull << c) - 1) << (r * LPR);
  for (int j = 0; j <= p.k + 1; j++) {
    const uint32_t hk = head & ~15u;
    m = all_max<LPR>(hk);
    if (j > p.k) break;
    const bool best = hk == m;
    const uint64_t same = __ballot(best);
    picked = c == j ? m : picked;
    last = j == p.k - 1 ? m : last, rest = m;
    if (best && !(same & below)) {  // of equal choices the lowest lane's
      s_pick[wave][r][j] = m ? e0 + 15 - (int)(head & 15u) : 0;  // (m = 0: nothing is left, j = k)
      head = next < PER ? sorted[64 * next] : 0u;
      next++;
    }
  }
  wave_fence();
  const int who = s_pick[wave][r][min(c, p.k)];
  // the c-th score in 64 bits, and what is compared
  const int few = min(p.k + 1, LPR);
  double w = 0, y = 0;
  if (c < few) {
    const size_t o = row + who;
    y = order_value(BF16 ? bf2f(((const uint16_t*)p.logits)[o]) : ((const float*)p.logits)[o]);
    if constexpr (SOFTMAX) {
      w = y == -INFINITY ? 0.0 : y == (double)mx ? 1.0 : exp_neg(y - (double)mx);
    } else {
      const double z = exp_neg(-fabs(y)), q = rcp64(1 + z);
      w = y < 0 ? z * q : q;
    }
  }
  // the softmax's sum in 64 bits, which divides the scores (and cancels where the weights are divided by the picks' own sum)
  auto total = [&] {
    double all = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) all += l[i] == -INFINITY ? 0.0 : l[i] == mx ? 1.0 : exp_neg((double)l[i] - (double)mx);
    all = row_sum_f64(all);
    if constexpr (LPR >= 32) all += __shfl_xor(all, 16, 64);
    if constexpr (LPR == 64) all += __shfl_xor(all, 32, 64);
    return all;
  };
  if constexpr (SOFTMAX)
    if (!p.norm) {
      const double all = total();
      w = all > 0 ? w / all : 0.0;
    }
  int at = c;  // the place of this lane's expert among the few
  if (p.bias || !BF16) {
    // logits themselves: only equal keys are in doubt
    auto doubt = [&](uint32_t hi, uint32_t lo) {
      return lo != 0 && (p.bias ? too_near<SOFTMAX, true>(key_value(hi), key_value(lo), top) : hi == lo);
    };
    const uint32_t after = (uint32_t)__shfl_down((int)picked, 1, 64);
    const bool near = c + 1 < few && doubt(picked, after);
    redo_me |= doubt(last, few > p.k ? m : rest);  // the one behind the few
    if (__ballot(near)) {
      double mine = y;
      if (p.bias) {
        mine = w;
        if (SOFTMAX && p.norm) {
          const double all = total();
          mine = all > 0 ? w / all : 0.0;
        }
        mine += (double)order_value(p.bias[who]);
      }
      at = 0;
      for (int j = 0; j < few; j++) {
        const double x = __shfl(mine, r * LPR + j, 64);
        const int e = __shfl(who, r * LPR + j, 64);
        at += __shfl((int)picked, r * LPR + j, 64) != 0 && (x > mine || (x == mine && e < who));
      }
    }
  }
  const uint64_t redo = __ballot(redo_me && t < p.T);
  auto redo_row = [&](int rr) { return (redo >> (rr * LPR) & kLanes) != 0; };
  const bool live = c < few && picked != 0 && at < p.k && t < p.T && !redo_row(r);
  if (p.norm) {
    double sum = row_sum_f64(c < few && at < p.k ? w : 0.0);
    if constexpr (LPR >= 32) sum += __shfl_xor(sum, 16, 64);  // the 17th lane's
    w = sum > 0 ? w / sum : 0.0;
  }
  if (live) {
    p.idx[(size_t)t * p.k + at] = who;
    p.wt[(size_t)t * p.k + at] = (float)(w * (double)p.scale);
  }
  if (c == 0 && t < p.T && !redo_row(r)) {
    float g = 1.f;
    if (p.shared_gate) {
      const double y = BF16 ? bf2f(((const uint16_t*)p.logits)[row + p.E]) : ((const float*)p.logits)[row + p.E];
      const double z = exp_neg(-fabs(y));
      g = (float)(y != y ? y : y < 0 ? z / (1 + z) : 1 / (1 + z));
    }
    p.sg[t] = g;
  }
  if (redo == 0) return;
  for (int rr = 0; rr < RW; rr++)
    if (redo_row(rr)) {
      wave_fence();
      route_exact<LPR * PER / 64, BF16, SOFTMAX, GTOP>(p, t0 + rr, (double*)mem[wave]);
    }
}

// The lanes per token by E: as few as hold the experts, 16 to a lane (16384 tokens of 256: 16 lanes 15.7 us, 32 lanes of 8
// experts 17.6, 64 of 4 28; one token: all within 0.2). Groups of which a token has more than lanes go by waves.
template <int LPR, int PER, bool BF16, bool SOFTMAX, int GTOP>
static void launch_route_cfg(const RouteExArgs& a, hipStream_t st) {
  constexpr int rows = 4 * 64 / LPR;
  if (a.groups <= LPR)
    hipLaunchKernelGGL((k_moe_route_fast<LPR, PER, BF16, SOFTMAX, GTOP>), dim3((a.T + rows - 1) / rows), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_moe_route_ex<LPR * PER / 64, BF16, SOFTMAX, GTOP>), dim3((a.T + 3) / 4), dim3(256), 0, st, a);
}
template <bool BF16, bool SOFTMAX, int GTOP>
static void launch_route_e(const RouteExArgs& a, hipStream_t st) {
  if (a.E <= 64) launch_route_cfg<16, 4, BF16, SOFTMAX, GTOP>(a, st);
  else if (a.E <= 128) launch_route_cfg<16, 8, BF16, SOFTMAX, GTOP>(a, st);
  else if (a.E <= 256) launch_route_cfg<16, 16, BF16, SOFTMAX, GTOP>(a, st);
  else launch_route_cfg<32, 16, BF16, SOFTMAX, GTOP>(a, st);
}
template <bool BF16>
static void launch_route_bf(const RouteExArgs& a, int softmax, int group_top, hipStream_t st) {
  if (softmax) group_top == 2 ? launch_route_e<BF16, true, 2>(a, st) : launch_route_e<BF16, true, 1>(a, st);
  else group_top == 2 ? launch_route_e<BF16, false, 2>(a, st) : launch_route_e<BF16, false, 1>(a, st);
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
