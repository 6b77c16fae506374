// Sampling of the next token from a head's logits, with temperature, top-k, top-p and min-p, from given random numbers.
//
// Per row: w_i = exp((l_i - max) / temperature). In the order of falling logits (equal ones: rising index) every filter
// keeps a prefix: the first k; of these the shortest whose weights reach p times theirs all; of these the w_i >= min_p
// (the largest w is 1). Then, in the order of the vocabulary, the token is the first whose sum of kept weights passes u times
// their total.
// The weights are fixed-point numbers of 44 fraction bits (from 64-bit exponentials), their sums whole numbers: exact
// whatever the order, so blocks and atomics may add them in any order, and 512 K of them fit in 63 bits. What 2^-45 of the
// largest weight or less rounds to nothing is never drawn.
#include "common.h"
#include "f64_dev.h"
#include "host.h"
#include "kernels.h"

namespace ifd {

constexpr int kSampleMaxV = 1 << 19;

struct SampleArgs {
  const void* logits;
  int T, V, ld;
  const float* temperature;  // any of these null: off
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* token;
  float* prob;  // or null
};

struct RowPar {
  double rt;      // 1 / temperature
  double min_p;
  double top_p;
  int k;          // V: off
  bool greedy;
};
__device__ __forceinline__ RowPar row_par(const SampleArgs& p, int t) {
  RowPar r;
  const float tau = p.temperature ? p.temperature[t] : 1.f;
  r.greedy = !(tau > 0.f);
  r.rt = r.greedy ? 1.0 : 1.0 / (double)tau;
  r.k = p.top_k ? p.top_k[t] : 0;
  if (r.k <= 0 || r.k > p.V) r.k = p.V;
  const float tp = p.top_p ? p.top_p[t] : 1.f, mp = p.min_p ? p.min_p[t] : 0.f;
  r.top_p = tp < 1.f ? fmax((double)tp, 0.0) : tp >= 1.f ? 1.0 : 0.0;
  r.min_p = mp > 0.f ? fmin((double)mp, 1.0) : 0.0;
  return r;
}
// a row's random number, inside [0, 1)
__device__ __forceinline__ double row_u(const SampleArgs& p, int t) {
  return (double)fminf(fmaxf(p.u[t], 0.f), 1.f - 0x1p-24f);
}

template <bool BF16>
__device__ __forceinline__ float load_logit(const SampleArgs& p, int t, int i) {
  const size_t o = (size_t)t * p.ld + i;
  return order_value(BF16 ? bf2f(((const uint16_t*)p.logits)[o]) : ((const float*)p.logits)[o]);
}
// w of a logit of a row with a maximum above -infinity
__device__ __forceinline__ double weight(float l, float mx, double rt) {
  return l == mx ? 1.0 : exp_neg(((double)l - (double)mx) * rt);
}
__device__ __forceinline__ uint64_t fixed(double w) { return (uint64_t)__builtin_rint(w * 0x1p44); }

// ---- one block per row ---------------------------------------------------------------------------------------------
constexpr int kRowThreads = 1024, kRowBins = 2048;
struct RowLds {
  uint64_t w[kRowBins];
  uint32_t n[kRowBins];
  uint64_t wsum[64];
  uint32_t nsum[64];
  uint64_t wpart[16];
  uint32_t npart[16];
  uint32_t key, ties;
  uint64_t total;
  int at;
};

// Block-wide exclusive prefix of (w, n) by thread; the totals in W, Nn.
__device__ __forceinline__ void row_scan(RowLds& s, uint64_t& w, uint32_t& n, uint64_t& W, uint32_t& Nn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t iw = w;
  uint32_t in = n;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint64_t a = __shfl_up(iw, o, 64);
    const uint32_t b = __shfl_up(in, o, 64);
    if (lane >= o) iw += a, in += b;
  }
  __syncthreads();
  if (lane == 63) s.wpart[wave] = iw, s.npart[wave] = in;
  __syncthreads();
  uint64_t bw = 0;
  uint32_t bn = 0;
  W = 0, Nn = 0;
  for (int i = 0; i < kRowThreads / 64; i++) {
    if (i == wave) bw = W, bn = Nn;
    W += s.wpart[i], Nn += s.npart[i];
  }
  w = bw + iw - w, n = bn + in - n;
}

// A prefix of the order: all with a key above `key`, and the first `ties` with that key.
struct Border {
  uint32_t key, ties;
};

// The border of the k first (by_count), or of the shortest prefix of the prefix `in` whose weight reaches `want`. Three
// passes over the row narrow the border's key 11, 11 and 10 bits at a time.
template <bool BF16>
__device__ Border row_border(RowLds& s, const SampleArgs& p, int t, float mx, double rt, bool by_count, uint32_t k,
                             double want, Border in) {
  uint32_t prefix = 0, nabove = 0;
  uint64_t wabove = 0;
  for (int level = 0; level < 3; level++) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bins = level == 2 ? 1024 : 2048;
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) s.w[i] = 0, s.n[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.V; i += kRowThreads) {
      const float l = load_logit<BF16>(p, t, i);
      const uint32_t key = order_key(l);
      if (level && (key >> (shift + (level == 2 ? 10 : 11))) != prefix) continue;
      if (key < in.key) continue;
      const int b = (key >> shift) & (bins - 1);
      if (!by_count && key == in.key) continue;  // its `ties` ones are added below
      atomicAdd(&s.n[b], 1u);
      if (!by_count) {
        const uint64_t w = fixed(weight(l, mx, rt));
        if (w) atomicAdd((unsigned long long*)&s.w[b], (unsigned long long)w);
      }
    }
    __syncthreads();
    if (!by_count && threadIdx.x == 0 && in.ties &&
        (level == 0 || (in.key >> (shift + (level == 2 ? 10 : 11))) == prefix)) {
      const int b = (in.key >> shift) & (bins - 1);
      s.n[b] += in.ties;
      s.w[b] += in.ties * fixed(weight(key_value(in.key), mx, rt));
    }
    __syncthreads();
    // bins from the top, two per thread; the bin in which the prefix reaches its end
    uint64_t w[2], ws, W;
    uint32_t n[2], ns, Nn;
    for (int q = 0; q < 2; q++) {
      const int b = bins - 1 - (2 * (int)threadIdx.x + q);
      w[q] = b >= 0 ? s.w[b] : 0, n[q] = b >= 0 ? s.n[b] : 0;
    }
    ws = w[0] + w[1], ns = n[0] + n[1];
    row_scan(s, ws, ns, W, Nn);
    if (threadIdx.x == 0) s.key = 0xffffffffu;
    __syncthreads();
    for (int q = 0; q < 2; q++) {
      const int b = bins - 1 - (2 * (int)threadIdx.x + q);
      if (b >= 0 && n[q]) {
        const bool starts = by_count ? nabove + ns < k : (double)(wabove + ws) < want || nabove + ns == 0;
        const bool ends = by_count ? nabove + ns + n[q] >= k : (double)(wabove + ws + w[q]) >= want;
        if (starts && ends) s.key = (uint32_t)b, s.wsum[0] = wabove + ws, s.nsum[0] = nabove + ns;
      }
      ws += w[q], ns += n[q];
    }
    __syncthreads();
    prefix = prefix << (level == 2 ? 10 : 11) | s.key;
    wabove = s.wsum[0], nabove = s.nsum[0];
    __syncthreads();
  }
  // the ties of the border's key that are still needed
  Border b{prefix, 0};
  const uint32_t have = s.n[prefix & 1023];
  if (by_count) {
    b.ties = k - nabove;
  } else {
    const double w = (double)fixed(weight(key_value(prefix), mx, rt));
    const double r = w > 0 ? ceil((want - (double)wabove) / w) : 1.0;
    b.ties = (uint32_t)fmin(fmax(r, 1.0), (double)have);
  }
  __syncthreads();
  return b;
}

template <bool BF16>
__device__ void row_sample(RowLds& s, const SampleArgs& p, int t) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const RowPar r = row_par(p, t);
  float mx = -INFINITY;
  int at = 0x7fffffff;
  for (int i = threadIdx.x; i < p.V; i += kRowThreads) {
    const float l = load_logit<BF16>(p, t, i);
    if (l > mx) mx = l, at = i;
  }
  const float wm = dpp_max_f(mx);
  const int wat = dpp_min_i(mx == wm ? at : 0x7fffffff);
  if (lane == 0) s.npart[wave] = __float_as_uint(wm), s.nsum[wave] = (uint32_t)wat;
  __syncthreads();
  mx = -INFINITY, at = 0x7fffffff;
  for (int i = 0; i < kRowThreads / 64; i++) {
    const float v = __uint_as_float(s.npart[i]);
    if (v > mx || (v == mx && (int)s.nsum[i] < at)) mx = v, at = (int)s.nsum[i];
  }
  __syncthreads();
  if (mx == -INFINITY || r.greedy) {
    if (threadIdx.x == 0) {
      p.token[t] = mx == -INFINITY ? -1 : at;
      if (p.prob) p.prob[t] = mx == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  Border b{order_key(-INFINITY), (uint32_t)p.V};  // everything
  if (r.k < p.V) b = row_border<BF16>(s, p, t, mx, r.rt, true, (uint32_t)r.k, 0.0, Border{0, 0});
  const int parts = 64, per = (p.V + parts - 1) / parts;
  // kept weights and border ties of 64 runs of the vocabulary
  auto sums = [&](double min_p) {
    if (threadIdx.x < 64) s.wsum[threadIdx.x] = 0, s.nsum[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < p.V; i += kRowThreads) {
      const float l = load_logit<BF16>(p, t, i);
      const uint32_t key = order_key(l);
      if (key < b.key) continue;
      if (key == b.key) {
        atomicAdd(&s.nsum[i / per], 1u);
        continue;
      }
      const double w = weight(l, mx, r.rt);
      const uint64_t f = fixed(w);
      if (w >= min_p && f) atomicAdd((unsigned long long*)&s.wsum[i / per], (unsigned long long)f);
    }
    __syncthreads();
  };
  const uint64_t wb_all = fixed(weight(key_value(b.key), mx, r.rt));
  if (r.top_p < 1.0) {
    sums(0.0);
    uint64_t total = 0;
    for (int i = 0; i < parts; i++) total += s.wsum[i];
    total += b.ties * wb_all;
    __syncthreads();
    b = row_border<BF16>(s, p, t, mx, r.rt, false, 0, r.top_p * (double)total, b);
  }
  sums(r.min_p);
  const double wbd = weight(key_value(b.key), mx, r.rt);
  const uint64_t wb = wbd >= r.min_p ? fixed(wbd) : 0;
  if (threadIdx.x == 0) {  // the run in which u times the total is passed
    uint64_t total = 0;
    uint32_t left = b.ties;
    for (int i = 0; i < parts; i++) {
      const uint32_t n = min(left, s.nsum[i]);
      left -= n;
      s.wsum[i] += n * wb;
      total += s.wsum[i];
    }
    const double want = row_u(p, t) * (double)total;
    uint64_t c = 0;
    int i = 0;
    left = b.ties;
    for (; i < parts - 1 && !((double)(c + s.wsum[i]) > want); i++) c += s.wsum[i], left -= min(left, s.nsum[i]);
    s.at = i, s.total = total, s.wpart[0] = c, s.ties = left;
  }
  __syncthreads();
  const int run = s.at;
  const uint64_t total = s.total;
  uint64_t c = s.wpart[0];
  uint32_t left = s.ties;
  const double want = row_u(p, t) * (double)total;
  __syncthreads();
  if (threadIdx.x == 0) s.at = 0x7fffffff;
  for (int i0 = run * per; i0 < min((run + 1) * per, p.V); i0 += kRowThreads) {
    const int i = i0 + (int)threadIdx.x;
    const bool in = i < min((run + 1) * per, p.V);
    const float l = in ? load_logit<BF16>(p, t, i) : -INFINITY;
    const uint32_t key = order_key(l);
    uint32_t tie = in && key == b.key, tn = tie, N1;
    uint64_t zero = 0, W1;
    row_scan(s, zero, tn, W1, N1);  // ties before this one
    const double wd = in ? weight(l, mx, r.rt) : 0.0;
    uint64_t w = in && key > b.key && wd >= r.min_p ? fixed(wd) : tie && tn < left ? wb : 0, before = w, W;
    uint32_t dn = 0, N2;
    row_scan(s, before, dn, W, N2);
    if (w && (double)(c + before + w) > want) atomicMin(&s.at, i);
    __syncthreads();
    if (s.at != 0x7fffffff) {
      if (s.at == i) {
        p.token[t] = i;
        if (p.prob) p.prob[t] = (float)((double)w / (double)total);
      }
      return;
    }
    c += W, left -= min(left, N1);
    __syncthreads();
  }
}

template <bool BF16>
__global__ __launch_bounds__(kRowThreads) void k_sample_row(SampleArgs p) {
  __shared__ RowLds s;
  row_sample<BF16>(s, p, blockIdx.x);
}

size_t sample_workspace(int T, int V) { return 0; }

int launch_sample(const void* logits, int logits_bf16, int T, int V, int ld, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const float* u, int* token, float* prob, void* ws,
                  size_t ws_bytes, hipStream_t st) {
  if (T == 0) return IFD_OK;
  const SampleArgs a{logits, T, V, ld, temperature, top_k, top_p, min_p, u, token, prob};
  if (logits_bf16) hipLaunchKernelGGL(k_sample_row<true>, dim3(T), dim3(kRowThreads), 0, st, a);
  else hipLaunchKernelGGL(k_sample_row<false>, dim3(T), dim3(kRowThreads), 0, st, a);
  return check_launch("sample");
}

}  // namespace ifd
