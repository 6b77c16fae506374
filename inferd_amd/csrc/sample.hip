// Sampling of the next token from a head's logits, with temperature, top-k, top-p and min-p, from given random numbers.
//
// Per row: w_i = exp((l_i - max) / temperature). In the order of falling logits (equal ones: rising index) every filter
// keeps a prefix: the first k; of these the shortest whose weights reach p times theirs all; of these the w_i >= min_p
// (the largest w is 1). Then, in the order of the vocabulary, the token is the first whose sum of kept weights passes u times
// their total.
// The weights are fixed-point numbers of 44 fraction bits (from 64-bit exponentials), their sums whole numbers: exact
// whatever the order, so blocks and atomics may add them in any order, and 512 K of them fit in 63 bits. What 2^-45 of the
// largest weight or less rounds to nothing is never drawn.
#include <algorithm>

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

// ---- many blocks per row -------------------------------------------------------------------------------------------
// One block reads a row of 248320 at the rate of a single CU, seven times over for a border in 32-bit keys. Here every row
// is spread over the device, in up to four launches:
//   k_sample_max     maxima of runs of 4, 16 or 64 logits and of tiles of 1024 (one wave each)
//   k_sample_border  (with top-k or top-p) where the border lies, roughly. top-k: the k-th largest run maximum bounds the
//                    k-th largest logit from below, so what lies under its bin is out. top-p: a histogram of the row over
//                    2048 bins of (max - l) / temperature, 1/64 wide; a bin's sum is kept relative to exp at its upper
//                    end as a whole number of 2^-12, so one 32-bit LDS addition per logit gives weights to 2^-13.
//   k_sample_collect the tiles' sums of what is surely kept, and a list of the logits that may lie at the border
//   k_sample_draw    one block per row sorts the list, finds the border exactly, and then the token: first its tile, from
//                    the sums, then its place.
// The estimate only chooses what is listed: k_sample_draw checks that the exact border lies inside. Where it does not, or
// the list is full (thousands of equal logits at the border, top_p within 4e-4 of 1 on a flat row) or top_k is past 1024,
// it takes the one-block path above. Both give the same token.
constexpr int kTile = 1024, kList = 4096, kMaxK = 1024, kBins = 2048, kTauBins = 1024;
constexpr int kRowsPerLaunch = 512;

struct RowInfo {  // what the launches of a call hand on, per row
  uint64_t before, all;  // sums of the weights in the bins above blo, and of all
  uint32_t n;            // listed logits
  int tau;               // top-k: the last bin (1/32 wide) that is listed
  int blo, bhi;          // top-p: the bins that are listed
};
struct SampleWs {
  char* base;
  size_t row;  // bytes per row: [RowInfo | list | hist | tile sums | tile maxima | run maxima]
  int tiles, runs, run;  // run: logits per run (4, 16 or 64)
  __host__ __device__ char* at(int t) const { return base + (size_t)t * row; }
  __device__ RowInfo* info(int t) const { return (RowInfo*)at(t); }
  __device__ uint64_t* list(int t) const { return (uint64_t*)(at(t) + 64); }
  __device__ uint32_t* hist(int t) const { return (uint32_t*)(at(t) + 64 + kList * 8); }
  __device__ uint64_t* tsum(int t) const { return (uint64_t*)(at(t) + 64 + kList * 8 + kBins * 4); }
  __device__ float* tmax(int t) const { return (float*)(tsum(t) + tiles); }
  __device__ float* rmax(int t) const { return tmax(t) + tiles; }
};
static_assert(sizeof(RowInfo) <= 64, "row header");

static SampleWs sample_ws(int V) {
  SampleWs w{};
  w.tiles = (V + kTile - 1) / kTile;
  w.run = V > 65536 ? 64 : V > 16384 ? 16 : 4;  // at least kMaxK runs once a row is longer than the list
  w.runs = w.tiles * (kTile / w.run);
  w.row = align_up(64 + (size_t)kList * 8 + kBins * 4 + (size_t)w.tiles * 12 + (size_t)w.runs * 4, 256);
  return w;
}

// What a row asks for. Its filters may differ from its neighbours'.
enum RowKind { kGreedy, kTopK, kTopP, kFull, kOneBlock };
__device__ __forceinline__ int row_kind(const RowPar& r, int V) {
  if (r.greedy) return kGreedy;
  if (r.k < V) return r.k <= kMaxK ? kTopK : kOneBlock;
  return r.top_p < 1.0 ? kTopP : kFull;
}

// The 16 logits of a lane in a tile: q's four are at 256 q + 4 lane (past V: -infinity).
template <bool BF16>
__device__ __forceinline__ void load_tile(const SampleArgs& p, int t, int tile, float (&l)[16]) {
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint16_t h4 __attribute__((ext_vector_type(4), aligned(2)));
  const int lane = threadIdx.x & 63;
  const size_t row = (size_t)t * p.ld;
  if ((tile + 1) * kTile <= p.V) {
    if constexpr (BF16) {
      h4 v[4];
#pragma unroll
      for (int q = 0; q < 4; q++) v[q] = *(const h4*)((const uint16_t*)p.logits + row + tile * kTile + 256 * q + 4 * lane);
#pragma unroll
      for (int e = 0; e < 16; e++) l[e] = order_value(bf2f(v[e / 4][e % 4]));
    } else {
      f4 v[4];
#pragma unroll
      for (int q = 0; q < 4; q++) v[q] = *(const f4*)((const float*)p.logits + row + tile * kTile + 256 * q + 4 * lane);
#pragma unroll
      for (int e = 0; e < 16; e++) l[e] = order_value(v[e / 4][e % 4]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int i = tile * kTile + 256 * (e / 4) + 4 * lane + e % 4;
      const float v = load_logit<BF16>(p, t, min(i, p.V - 1));
      l[e] = i < p.V ? v : -INFINITY;
    }
  }
}
__device__ __forceinline__ int tile_at(int e) { return 256 * (e / 4) + 4 * (int)(threadIdx.x & 63) + e % 4; }

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o, 64);
  return v;
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_sample_max(SampleArgs p, SampleWs ws) {
  const int lane = threadIdx.x & 63, t = blockIdx.y, tile = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (blockIdx.x == 0) {
    uint32_t* const h = ws.hist(t);
    for (int i = threadIdx.x; i < kBins; i += 256) h[i] = 0;
    if (threadIdx.x == 0) *ws.info(t) = RowInfo{};
  }
  if (tile >= ws.tiles) return;
  float l[16], m[4];
  load_tile<BF16>(p, t, tile, l);
  float* const rm = ws.rmax(t) + (size_t)tile * (kTile / ws.run);
#pragma unroll
  for (int q = 0; q < 4; q++) m[q] = fmaxf(fmaxf(l[4 * q], l[4 * q + 1]), fmaxf(l[4 * q + 2], l[4 * q + 3]));
  if (p.top_k) {
    if (ws.run == 4) {
#pragma unroll
      for (int q = 0; q < 4; q++) rm[64 * q + lane] = m[q];
    } else {
      const int n = ws.run / 4;  // lanes per run
#pragma unroll
      for (int q = 0; q < 4; q++) {
        float v = m[q];
        v = fmaxf(v, __shfl_xor(v, 1, 64));
        v = fmaxf(v, __shfl_xor(v, 2, 64));
        if (n == 16) v = fmaxf(v, __shfl_xor(v, 4, 64)), v = fmaxf(v, __shfl_xor(v, 8, 64));
        if (lane % n == 0) rm[64 / n * q + lane / n] = v;
      }
    }
  }
  const float v = dpp_max_f(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
  if (lane == 0) ws.tmax(t)[tile] = v;
}

// The row's maximum, by every thread of a block of W waves.
template <int W>
__device__ __forceinline__ float row_max(const SampleWs& ws, int t, float* s) {
  const float* const tm = ws.tmax(t);
  float m = -INFINITY;
  for (int i = threadIdx.x; i < ws.tiles; i += 64 * W) m = fmaxf(m, tm[i]);
  m = dpp_max_f(m);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
  m = s[0];
#pragma unroll
  for (int i = 1; i < W; i++) m = fmaxf(m, s[i]);
  return m;
}
// (max - l) / temperature in bins of 1 / scale, the last of which holds all that is left; monotone in l
__device__ __forceinline__ float bin_of(float l, float mx, float rt_scale, int bins) {
  return l == mx ? 0.f : fminf((mx - l) * rt_scale, (float)(bins - 1));
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_sample_border(SampleArgs p, SampleWs ws) {
  __shared__ uint32_t h[kBins];
  __shared__ float s[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const RowPar r = row_par(p, t);
  const int kind = row_kind(r, p.V);
  if (kind != kTopP && !(kind == kTopK && blockIdx.x == 0)) return;
  for (int i = threadIdx.x; i < kBins; i += 256) h[i] = 0;
  const float mx = row_max<4>(ws, t, s);  // with a barrier
  if (mx == -INFINITY) return;
  if (kind == kTopK) {
    const float sc = (float)(r.rt * 32.0);
    const float* const rm = ws.rmax(t);
    for (int i = threadIdx.x; i < ws.runs; i += 256) {
      const int b = (int)bin_of(rm[i], mx, sc, kTauBins);
      if (b < kTauBins - 1) atomicAdd(&h[b], 1u);
    }
    __syncthreads();
    if (wave == 0) {  // the first bin at which k runs have been seen; without one, all that has a weight
      uint32_t n[16], own = 0;
#pragma unroll
      for (int i = 0; i < 16; i++) own += n[i] = h[16 * lane + i];
      uint32_t c = own;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const uint32_t a = __shfl_up(c, o, 64);
        if (lane >= o) c += a;
      }
      const uint64_t hit = __ballot(c >= (uint32_t)r.k);
      if (hit == 0) {
        if (lane == 0) ws.info(t)->tau = kTauBins - 2;
      } else if (lane == __ffsll((long long)hit) - 1) {
        uint32_t x = c - own;
        int b = 0;
        for (; b < 15 && x + n[b] < (uint32_t)r.k; b++) x += n[b];
        ws.info(t)->tau = min(16 * lane + b, kTauBins - 2);
      }
    }
    return;
  }
  const float sc = (float)(r.rt * 64.0);
  for (int tile = blockIdx.x * 4 + wave; tile < ws.tiles; tile += 4 * gridDim.x) {
    float l[16];
    load_tile<BF16>(p, t, tile, l);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float y = bin_of(l[e], mx, sc, kBins);
      const int b = (int)y;
      const float f = y - (float)b;
      // exp(-f / 64) to 1e-6
      if (b < kBins - 1) atomicAdd(&h[b], (uint32_t)(4096.5f + f * (-64.f + 0.5f * f)));
    }
  }
  __syncthreads();
  uint32_t* const g = ws.hist(t);
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (h[i]) atomicAdd(&g[i], h[i]);
}

// The bins in which the border of top-p may lie: the histogram's sums are within 1.4e-4, and lo and hi 4e-4 off.
__device__ __forceinline__ void top_p_bins(const uint32_t* g, double top_p, double* part, int* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double w[8], own = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int b = 8 * (int)threadIdx.x + i;
    w[i] = (double)g[b] * (double)expf((float)b * -0.015625f);
    own += w[i];
  }
  double c = own;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const double a = __shfl_up(c, o, 64);
    if (lane >= o) c += a;
  }
  if (lane == 63) part[wave] = c;
  if (threadIdx.x == 0) out[0] = out[1] = kBins - 2;  // (nothing in the last bin has a weight)
  __syncthreads();
  double all = 0, base = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (i == wave) base = all;
    all += part[i];
  }
  double x = base + c - own;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const double want = top_p * all * (k ? 1 + 4e-4 : 1 - 4e-4);
    double y = x;
    int at;
#pragma unroll
    for (int i = 7; i >= 0; i--) y += w[i];  // (this thread's end)
    if (y >= want) {
      y = x, at = 8 * (int)threadIdx.x + 7;
      for (int i = 0; i < 7; i++) {
        y += w[i];
        if (y >= want) {
          at = 8 * (int)threadIdx.x + i;
          break;
        }
      }
      atomicMin(&out[k], at);
    }
  }
  __syncthreads();
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_sample_collect(SampleArgs p, SampleWs ws) {
  __shared__ float s[4];
  __shared__ double part[4];
  __shared__ int bins[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const RowPar r = row_par(p, t);
  const int kind = row_kind(r, p.V);
  if (kind == kGreedy || kind == kOneBlock) return;
  const float mx = row_max<4>(ws, t, s);
  if (mx == -INFINITY) return;
  RowInfo* const info = ws.info(t);
  uint64_t* const list = ws.list(t);
  // bins (of 1 / 32 for top-k) up to `sure` are kept whole, and those up to `last` listed
  int sure = kBins, last = -1;
  float sc = (float)(r.rt * 64.0);
  if (kind == kTopK) {
    sure = -1, last = info->tau, sc = (float)(r.rt * 32.0);
  } else if (kind == kTopP) {
    top_p_bins(ws.hist(t), r.top_p, part, bins);
    sure = bins[0] - 1, last = bins[1];
    if (blockIdx.x == 0 && threadIdx.x == 0) info->blo = bins[0], info->bhi = bins[1];
  }
  const int nbins = kind == kTopK ? kTauBins : kBins;
  uint64_t before = 0, all = 0;
  for (int tile = blockIdx.x * 4 + wave; tile < ws.tiles; tile += 4 * gridDim.x) {
    float l[16];
    load_tile<BF16>(p, t, tile, l);
    uint64_t keep = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int b = (int)bin_of(l[e], mx, sc, nbins);
      if (kind != kTopK) {
        const double w = weight(l[e], mx, r.rt);
        const uint64_t f = fixed(w);
        all += f;
        if (b <= sure) {
          before += f;
          keep += w >= r.min_p ? f : 0;
        }
      }
      const bool add = b > sure && b <= last && l[e] != -INFINITY;
      const uint64_t who = __ballot(add);
      if (who) {
        uint32_t at = 0;
        if (lane == __ffsll((long long)who) - 1) at = atomicAdd(&info->n, (uint32_t)__popcll(who));
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, __ffsll((long long)who) - 1);
        at += (uint32_t)__popcll(who & ((1ull << lane) - 1));
        if (add && at < kList)
          list[at] = (uint64_t)~order_key(l[e]) << 32 | (uint32_t)(tile * kTile + tile_at(e));
      }
    }
    if (kind != kTopK) {
      keep = wave_sum_u64(keep);
      if (lane == 0) ws.tsum(t)[tile] = keep;
    }
  }
  if (kind == kTopP) {
    before = wave_sum_u64(before), all = wave_sum_u64(all);
    if (lane == 0) {
      if (before) atomicAdd((unsigned long long*)&info->before, (unsigned long long)before);
      if (all) atomicAdd((unsigned long long*)&info->all, (unsigned long long)all);
    }
  }
}

// Sorts a[0 .. n - 1] in LDS, rising (space up to the next power of two, which is filled with ones).
__device__ __forceinline__ void sort_lds(uint64_t* a, int n) {
  int n2 = 2;
  while (n2 < n) n2 *= 2;
  for (int i = n + (int)threadIdx.x; i < n2; i += kRowThreads) a[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= n2; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int i = threadIdx.x; i < n2 / 2; i += kRowThreads) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const uint64_t x = a[lo], y = a[hi];
        if ((x > y) == ((lo & k) == 0)) a[lo] = y, a[hi] = x;
      }
      __syncthreads();
    }
}

struct DrawLds {
  union {
    RowLds row;
    struct {
      uint64_t a[kList];
      uint64_t w[kMaxK];
      uint64_t tile[kSampleMaxV / kTile];
    } f;
  };
  uint64_t wpart[16];
  uint32_t npart[16];
  float s[16];
  uint64_t border;
  int at, ok;
};

// Exclusive block-wide prefix of w by thread; the total in W.
__device__ __forceinline__ uint64_t draw_scan(DrawLds& s, uint64_t w, uint64_t& W) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t c = w;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const uint64_t a = __shfl_up(c, o, 64);
    if (lane >= o) c += a;
  }
  __syncthreads();
  if (lane == 63) s.wpart[wave] = c;
  __syncthreads();
  uint64_t base = 0;
  W = 0;
  for (int i = 0; i < kRowThreads / 64; i++) {
    if (i == wave) base = W;
    W += s.wpart[i];
  }
  return base + c - w;
}

template <bool BF16>
__global__ __launch_bounds__(kRowThreads) void k_sample_draw(SampleArgs p, SampleWs ws) {
  __shared__ DrawLds s;
  const int t = blockIdx.x, tid = threadIdx.x;
  const RowPar r = row_par(p, t);
  const int kind = row_kind(r, p.V);
  const float mx = row_max<16>(ws, t, s.s);
  const double u = row_u(p, t);
  if (tid == 0) s.at = 0x7fffffff, s.ok = 1;
  __syncthreads();
  auto done = [&](int token, float prob) {
    p.token[t] = token;
    if (p.prob) p.prob[t] = prob;
  };
  if (mx == -INFINITY) {
    if (tid == 0) done(-1, 0.f);
    return;
  }
  if (kind == kGreedy) {  // the first tile with the maximum, and its place there
    for (int i = tid; i < ws.tiles; i += kRowThreads)
      if (ws.tmax(t)[i] == mx) atomicMin(&s.at, i);
    __syncthreads();
    const int i = s.at * kTile + tid;
    __syncthreads();
    if (tid == 0) s.at = 0x7fffffff;
    __syncthreads();
    if (i < p.V && load_logit<BF16>(p, t, i) == mx) atomicMin(&s.at, i);
    __syncthreads();
    if (tid == 0) done(s.at, 1.f);
    return;
  }
  RowInfo in = *ws.info(t);
  const int n = (int)min(in.n, (uint32_t)kList + 1);
  if (kind == kOneBlock || n > kList) {
    __syncthreads();
    row_sample<BF16>(s.row, p, t);
    return;
  }
  auto entry_key = [](uint64_t a) { return ~(uint32_t)(a >> 32); };
  if (kind == kTopK) {
    for (int i = tid; i < n; i += kRowThreads) s.f.a[i] = ws.list(t)[i];
    sort_lds(s.f.a, n);
    // thread i: the i-th largest of the first k <= 1024
    const bool in_k = tid < min(n, r.k);
    const uint64_t a = s.f.a[in_k ? tid : 0];
    const double wd = in_k ? weight(key_value(entry_key(a)), mx, r.rt) : 0.0;
    const uint64_t w = in_k ? fixed(wd) : 0;
    uint64_t all, total, before = draw_scan(s, w, all);
    const bool in_p = r.top_p >= 1.0 || tid == 0 || (double)before < r.top_p * (double)all;
    const uint64_t f = in_k && in_p && wd >= r.min_p ? w : 0;
    draw_scan(s, f, total);
    // in the order of the vocabulary
    const int m = min(n, r.k);
    s.f.w[tid] = f;
    __syncthreads();
    if (tid < m) s.f.a[tid] = (a & 0xffffffffu) << 32 | (uint32_t)tid;
    __syncthreads();
    sort_lds(s.f.a, m);
    const uint64_t b = s.f.a[tid < m ? tid : 0];
    const uint64_t fw = tid < m ? s.f.w[(uint32_t)b] : 0;
    uint64_t W;
    before = draw_scan(s, fw, W);
    if (fw && (double)(before + fw) > u * (double)total) atomicMin(&s.at, tid);
    __syncthreads();
    if (tid == s.at) done((int)(b >> 32), (float)((double)fw / (double)total));
    return;
  }
  // kept: what comes before or at the border entry in the order, and has min_p
  uint64_t border = ~0ull;
  for (int i = tid; i < ws.tiles; i += kRowThreads) s.f.tile[i] = ws.tsum(t)[i];
  if (kind == kTopP) {
    for (int i = tid; i < n; i += kRowThreads) s.f.a[i] = ws.list(t)[i];
    sort_lds(s.f.a, n);
    const double want = r.top_p * (double)in.all;
    if (in.before != 0 && !((double)in.before < want)) s.ok = 0;  // the border lies above what is listed
    if (tid == 0) s.border = 0;
    uint64_t c = in.before;
    for (int i0 = 0; i0 < n; i0 += kRowThreads) {
      const int i = i0 + tid;
      const uint64_t a = s.f.a[min(i, n - 1)];
      const double wd = i < n ? weight(key_value(entry_key(a)), mx, r.rt) : 0.0;
      const uint64_t w = fixed(wd);
      uint64_t W;
      const uint64_t before = c + draw_scan(s, w, W);
      if (i < n && ((double)before < want || before == 0)) {
        if (i == 0 || before != 0) atomicMax((unsigned long long*)&s.border, (unsigned long long)a);
        if (wd >= r.min_p && (i == 0 || before != 0))
          atomicAdd((unsigned long long*)&s.f.tile[(uint32_t)a / kTile], (unsigned long long)w);
      }
      c += W;
    }
    if ((double)c < want) s.ok = 0;  // or below
    __syncthreads();
    border = s.border;
    if (!s.ok) {
      __syncthreads();
      row_sample<BF16>(s.row, p, t);
      return;
    }
  }
  __syncthreads();
  uint64_t total, W;
  const uint64_t mine = tid < ws.tiles ? s.f.tile[tid] : 0;
  uint64_t before = draw_scan(s, mine, total);
  const double want = u * (double)total;
  if (mine && (double)(before + mine) > want) atomicMin(&s.at, tid);
  __syncthreads();
  const int tile = min(s.at, ws.tiles - 1);
  if (tid == tile) s.border = before;
  __syncthreads();
  const uint64_t base = s.border;
  if (tid == 0) s.at = 0x7fffffff;
  const int i = tile * kTile + tid;
  const float l = i < p.V ? load_logit<BF16>(p, t, i) : -INFINITY;
  const double wd = i < p.V ? weight(l, mx, r.rt) : 0.0;
  const uint64_t a = (uint64_t)~order_key(l) << 32 | (uint32_t)i;
  const uint64_t f = a <= border && wd >= r.min_p ? fixed(wd) : 0;
  before = base + draw_scan(s, f, W);
  if (f && (double)(before + f) > want) atomicMin(&s.at, i);
  __syncthreads();
  if (i == s.at) done(i, (float)((double)f / (double)total));
}

size_t sample_workspace(int T, int V) { return (size_t)std::min(T, kRowsPerLaunch) * sample_ws(V).row; }

template <bool BF16>
static int launch_sample_rows(const SampleArgs& a, const SampleWs& ws, hipStream_t st) {
  const int quads = (ws.tiles + 3) / 4;
  const dim3 block(256), grid(quads, a.T), some(std::min(quads, std::max(1, 1024 / a.T)), a.T);
  hipLaunchKernelGGL(k_sample_max<BF16>, grid, block, 0, st, a, ws);
  if (a.top_k || a.top_p) hipLaunchKernelGGL(k_sample_border<BF16>, some, block, 0, st, a, ws);
  hipLaunchKernelGGL(k_sample_collect<BF16>, some, block, 0, st, a, ws);
  hipLaunchKernelGGL(k_sample_draw<BF16>, dim3(a.T), dim3(kRowThreads), 0, st, a, ws);
  return check_launch("sample");
}

int launch_sample(const void* logits, int logits_bf16, int T, int V, int ld, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const float* u, int* token, float* prob, void* mem,
                  size_t ws_bytes, hipStream_t st) {
  SampleWs ws = sample_ws(V);
  ws.base = (char*)mem;
  if (T && (!mem || ws_bytes < sample_workspace(T, V)))
    return fail(IFD_ERR_WORKSPACE, "sample needs %zu bytes of workspace, got %zu", sample_workspace(T, V), ws_bytes);
  for (int t = 0; t < T; t += kRowsPerLaunch) {
    auto off = [&](auto* q) { return q ? q + t : q; };
    const SampleArgs a{(const char*)logits + (size_t)t * ld * (logits_bf16 ? 2 : 4), std::min(T - t, kRowsPerLaunch), V, ld,
                       off(temperature), off(top_k), off(top_p), off(min_p), off(u), off(token), off(prob)};
    IFD_TRY(logits_bf16 ? launch_sample_rows<true>(a, ws, st) : launch_sample_rows<false>(a, ws, st));
  }
  return IFD_OK;
}

}  // namespace ifd
