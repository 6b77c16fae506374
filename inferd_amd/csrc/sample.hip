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

// w 2^44 of a logit of a row with a maximum above -infinity; rt = log2(e) / temperature
__device__ __forceinline__ uint64_t weight(float l, float mx, double rt) {
  return l == mx ? 1ull << 44 : exp2_fixed44(((double)l - (double)mx) * rt);
}
struct RowPar {
  double rt;      // log2(e) / temperature
  uint64_t min_w;  // min_p
  double top_p;
  int k;          // V: off
  bool greedy;
};
__device__ __forceinline__ RowPar row_par(const SampleArgs& p, int t) {
  RowPar r;
  const float tau = p.temperature ? p.temperature[t] : 1.f;
  r.greedy = !(tau > 0.f);
  r.rt = 1.4426950408889634074 / (r.greedy ? 1.0 : (double)tau);
  r.k = p.top_k ? p.top_k[t] : 0;
  if (r.k <= 0 || r.k > p.V) r.k = p.V;
  const float tp = p.top_p ? p.top_p[t] : 1.f, mp = p.min_p ? p.min_p[t] : 0.f;
  r.top_p = tp < 1.f ? fmax((double)tp, 0.0) : tp >= 1.f ? 1.0 : 0.0;
  r.min_w = mp > 0.f ? (uint64_t)__builtin_rint(fmin((double)mp, 1.0) * 0x1p44) : 0;
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
// ---- one block per row ---------------------------------------------------------------------------------------------
constexpr int kRowThreads = 512, kRowBins = 2048;
struct RowLds {
  uint64_t w[kRowBins];
  uint32_t n[kRowBins];
  uint64_t wsum[64];
  uint32_t nsum[64];
  uint64_t wpart[kRowThreads / 64];
  uint32_t npart[kRowThreads / 64];
  uint32_t key, ties;
  uint64_t total;
  int at;
};

// Block-wide exclusive prefix of (w, n) by thread; the totals in W, Nn.
__device__ __forceinline__ void row_scan(RowLds& s, uint64_t& w, uint32_t& n, uint64_t& W, uint32_t& Nn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t iw = wave_scan_u64(w);
  const uint32_t in = wave_scan_u32(n);
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
        const uint64_t w = weight(l, mx, rt);
        if (w) atomicAdd((unsigned long long*)&s.w[b], (unsigned long long)w);
      }
    }
    __syncthreads();
    if (!by_count && threadIdx.x == 0 && in.ties &&
        (level == 0 || (in.key >> (shift + (level == 2 ? 10 : 11))) == prefix)) {
      const int b = (in.key >> shift) & (bins - 1);
      s.n[b] += in.ties;
      s.w[b] += in.ties * weight(key_value(in.key), mx, rt);
    }
    __syncthreads();
    // bins from the top, some per thread; the bin in which the prefix reaches its end
    constexpr int PER = kRowBins / kRowThreads;
    uint64_t w[PER], ws = 0, W;
    uint32_t n[PER], ns = 0, Nn;
    for (int q = 0; q < PER; q++) {
      const int b = bins - 1 - (PER * (int)threadIdx.x + q);
      w[q] = b >= 0 ? s.w[b] : 0, n[q] = b >= 0 ? s.n[b] : 0;
    }
    for (int q = 0; q < PER; q++) ws += w[q], ns += n[q];
    row_scan(s, ws, ns, W, Nn);
    if (threadIdx.x == 0) s.key = 0xffffffffu;
    __syncthreads();
    for (int q = 0; q < PER; q++) {
      const int b = bins - 1 - (PER * (int)threadIdx.x + q);
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
    const double w = (double)weight(key_value(prefix), mx, rt);
    const double r = w > 0 ? ceil((want - (double)wabove) / w) : 1.0;
    b.ties = (uint32_t)fmin(fmax(r, 1.0), (double)have);
  }
  __syncthreads();
  return b;
}

template <bool BF16>
__device__ __attribute__((noinline)) void row_sample(RowLds& s, const SampleArgs& p, int t) {
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
  auto sums = [&](uint64_t min_w) {
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
      const uint64_t f = weight(l, mx, r.rt);
      if (f >= min_w && f) atomicAdd((unsigned long long*)&s.wsum[i / per], (unsigned long long)f);
    }
    __syncthreads();
  };
  const uint64_t wb_all = weight(key_value(b.key), mx, r.rt);
  if (r.top_p < 1.0) {
    sums(0);
    uint64_t total = 0;
    for (int i = 0; i < parts; i++) total += s.wsum[i];
    total += b.ties * wb_all;
    __syncthreads();
    b = row_border<BF16>(s, p, t, mx, r.rt, false, 0, r.top_p * (double)total, b);
  }
  sums(r.min_w);
  const uint64_t wbf = weight(key_value(b.key), mx, r.rt), wb = wbf >= r.min_w ? wbf : 0;
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
    const uint64_t f = in ? weight(l, mx, r.rt) : 0;
    uint64_t w = in && key > b.key && f >= r.min_w ? f : tie && tn < left ? wb : 0, before = w, W;
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
//                    bins of (max - l) / temperature, 1/128 wide; a bin's sum is kept relative to exp at its upper end as a
//                    whole number of 2^-12, so one 32-bit LDS addition per logit gives weights to 2^-13.
//   k_sample_collect the tiles' sums of what is surely kept, and a list of the logits that may lie at the border
//   k_sample_draw    one block per row finds the border exactly in the list, and then the token: first its tile, from the
//                    sums, then its place.
// The estimate only chooses what is listed: k_sample_draw checks that the exact border lies inside. Where it does not, or
// the list is full (thousands of equal logits at the border, top_p within 4e-4 of 1 on a flat row), top_k is past 1024 or
// the maximum infinite, it takes the one-block path above. Both give the same token. A row no longer than the list is its own
// list, and k_sample_draw alone does it.
//
// What bounds it, us per kernel (max / border / collect / draw; fp32 logits unless noted):
//   1 row of 248320, top-k and top-p       3.7 / 3.1 / 5.0 / 8.8   dependent launches, each a chain of memory latencies
//   7 rows of 50021 (bf16), min-p          2.6 / -   / 5.9 / 7.4   the same
//   32 rows of 151936, filters mixed       6.5 / 5.5 / 12 / 14     the same, and the longest row's draw
//   128 rows of 248320, top-p              24  / 23  / 52 / 18     max reads at 5.3 TB/s; border and collect read again (from the
//                                          last cache) and issue: some 12 and 35 vector instructions per logit, 20 us of
//                                          collect's for the 64-bit exponentials
// One block per row took 401, 46, 436 and 928 us a call; these launches 20, 15, 37 and 110.
constexpr int kTile = 1024, kList = 4096, kMaxK = 1024, kBins = 4096;
constexpr float kBinScale = 128.f;  // bins per unit of (max - l) / temperature
constexpr int kRowsPerLaunch = 512, kSomeWaves = 8, kCollect = 768;

struct RowInfo {  // what the launches of a call hand on, per row
  uint64_t before, all;  // sums of the weights in the bins above the listed ones, and of all
  uint32_t n;            // listed logits
  int tau;               // top-k: the last bin that is listed
};
struct SampleWs {
  char* base;
  size_t row;  // bytes per row: [RowInfo | list | hist | tile sums | tile maxima | run maxima]
  int tiles, runs, run;  // run: logits per run (4, 16 or 64)
  __device__ char* at(int t) const { return base + (size_t)t * row; }
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
enum RowKind { kGreedy, kTopK, kTopP, kFull, kOneBlock, kNothing };
__device__ __forceinline__ int row_kind(const RowPar& r, int V, float mx) {
  if (mx == -INFINITY) return kNothing;
  if (r.greedy) return kGreedy;
  if (mx == INFINITY) return kOneBlock;
  if (r.k < V) return r.k <= kMaxK ? kTopK : kOneBlock;
  return r.top_p < 1.0 ? kTopP : kFull;
}

// The 16 logits of a lane in a tile: q's four are at 256 q + 4 lane (past V: -infinity). NaN stay NaN: no maximum takes them,
// no comparison below holds for them, and their weight is 0.
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
      for (int e = 0; e < 16; e++) l[e] = bf2f(v[e / 4][e % 4]);
    } else {
      f4 v[4];
#pragma unroll
      for (int q = 0; q < 4; q++) v[q] = *(const f4*)((const float*)p.logits + row + tile * kTile + 256 * q + 4 * lane);
#pragma unroll
      for (int e = 0; e < 16; e++) l[e] = v[e / 4][e % 4];
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

template <bool BF16>
__global__ __launch_bounds__(256) void k_sample_max(SampleArgs p, SampleWs ws) {
  const int lane = threadIdx.x & 63, t = blockIdx.y, tile = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (blockIdx.x == 0) {
    uint32_t* const h = ws.hist(t);
    if (p.top_p)
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
// Bins per unit of the logits (finite, so that the maximum itself is in bin 0; log2(e) is taken out of rt again).
__device__ __forceinline__ float bin_scale(const RowPar& r, float scale) {
  return (float)fmin(r.rt * 0.69314718055994531 * scale, 3e38);
}

template <bool BF16>
__global__ __launch_bounds__(64 * kSomeWaves) void k_sample_border(SampleArgs p, SampleWs ws) {
  __shared__ uint32_t h[kBins], part[kSomeWaves];
  __shared__ float s[kSomeWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const RowPar r = row_par(p, t);
  // (a maximum above -infinity and below infinity: whether it is that comes after the rows that have no work here)
  int kind = row_kind(r, p.V, 0.f);
  if (kind != kTopP && !(kind == kTopK && blockIdx.x == 0)) return;
  for (int i = threadIdx.x; i < kBins; i += 64 * kSomeWaves) h[i] = 0;
  // the first loads go out before the row's maximum is waited for
  constexpr int T = 64 * kSomeWaves, U = 8;
  const float* const rm = ws.rmax(t);
  float l[16];
  if (kind == kTopK) {
#pragma unroll
    for (int u = 0; u < U; u++) l[u] = rm[min(T * u + (int)threadIdx.x, ws.runs - 1)];
  } else {
    load_tile<BF16>(p, t, min((int)blockIdx.x * kSomeWaves + wave, ws.tiles - 1), l);
  }
  const float mx = row_max<kSomeWaves>(ws, t, s);  // with a barrier
  if (row_kind(r, p.V, mx) != kind) return;
  const float sc = bin_scale(r, kBinScale);
  if (kind == kTopK) {
    auto count = [&](float m) {
      const float y = (mx - m) * sc;
      if (y < (float)(kBins - 1)) atomicAdd(&h[(int)y], 1u);
    };
#pragma unroll
    for (int u = 0; u < U; u++)
      if (T * u + (int)threadIdx.x < ws.runs) count(l[u]);
    for (int i = T * U + threadIdx.x; i < ws.runs; i += T) count(rm[i]);
    __syncthreads();
    // the first bin at which k runs have been seen; without one, all that has a weight
    constexpr int PER = kBins / T;
    uint32_t n[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) own += n[i] = h[PER * threadIdx.x + i];
    const uint32_t c = wave_scan_u32(own);
    if (lane == 63) part[wave] = c;
    __syncthreads();
    uint32_t x = c - own, all = 0;
#pragma unroll
    for (int i = 0; i < kSomeWaves; i++) {
      x += i < wave ? part[i] : 0;
      all += part[i];
    }
    const uint32_t k = (uint32_t)r.k;
    if (threadIdx.x == 0 && all < k) ws.info(t)->tau = kBins - 2;
    if (x < k && x + own >= k) {
      int b = 0;
      for (; b < PER - 1 && x + n[b] < k; b++) x += n[b];
      ws.info(t)->tau = min(PER * (int)threadIdx.x + b, kBins - 2);
    }
    return;
  }
  for (int tile = blockIdx.x * kSomeWaves + wave; tile < ws.tiles; tile += kSomeWaves * gridDim.x) {
    if (tile >= kSomeWaves * (int)gridDim.x) load_tile<BF16>(p, t, tile, l);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const float y = (mx - l[e]) * sc;
      if (y < (float)(kBins - 1)) {  // beyond: no weight
        const int b = (int)y;
        const float f = y - (float)b;
        // 4096 exp(-f / 128), to 1e-7
        atomicAdd(&h[b], (uint32_t)__builtin_fmaf(f, __builtin_fmaf(f, 0.125f, -32.f), 4096.5f));
      }
    }
  }
  __syncthreads();
  uint32_t* const g = ws.hist(t);
  for (int i = threadIdx.x; i < kBins; i += 64 * kSomeWaves)
    if (h[i]) atomicAdd(&g[i], h[i]);
}

// The first and last bin in which the border of top-p may lie: the histogram's sums are within 1.4e-4 of the weights', and
// the sought ones 4e-4 off to either side.
__device__ __forceinline__ void top_p_bins(const uint32_t* g, double top_p, double* part, int* out) {
  constexpr int PER = kBins / (64 * kSomeWaves);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = PER * (int)threadIdx.x;
  float w[PER];
  double own = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    w[i] = (float)g[b0 + i] * __builtin_amdgcn_exp2f((float)(b0 + i) * (-1.44269504f / kBinScale));
    own += w[i];
  }
  const double c = wave_scan_f64(own);
  if (lane == 63) part[wave] = c;
  if (threadIdx.x == 0) out[0] = out[1] = kBins - 2;  // (nothing in the last bin has a weight)
  __syncthreads();
  double all = 0, base = 0;
#pragma unroll
  for (int i = 0; i < kSomeWaves; i++) {
    if (i == wave) base = all;
    all += part[i];
  }
  const double x = base + c - own;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const double want = top_p * all * (k ? 1 + 4e-4 : 1 - 4e-4);
    if (x + own >= want && (x < want || threadIdx.x == 0)) {
      double y = x;
      int i = 0;
      for (; i < PER - 1; i++) {
        y += w[i];
        if (y >= want) break;
      }
      atomicMin(&out[k], b0 + i);
    }
  }
  __syncthreads();
}

template <bool BF16>
__global__ __launch_bounds__(64 * kSomeWaves) void k_sample_collect(SampleArgs p, SampleWs ws) {
  __shared__ float s[kSomeWaves];
  __shared__ double part[kSomeWaves];
  __shared__ int bins[2];
  __shared__ uint64_t found[kList];  // this block's part of the list (a global atomic per entry costs its latency)
  __shared__ uint32_t nfound, at0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const RowPar r = row_par(p, t);
  if (r.greedy) return;
  const int tau = ws.info(t)->tau;
  const float mx = row_max<kSomeWaves>(ws, t, s);
  const int kind = row_kind(r, p.V, mx);
  if (kind != kTopK && kind != kTopP && kind != kFull) return;
  RowInfo* const info = ws.info(t);
  if (threadIdx.x == 0) nfound = 0;
  __syncthreads();
  // y = (max - l) scale: below `sure` kept whole, from there to below `last` listed
  float sure = INFINITY, last = INFINITY;
  const float sc = bin_scale(r, kBinScale);
  if (kind == kTopK) {
    sure = 0.f, last = (float)(tau + 1);
  } else if (kind == kTopP) {
    top_p_bins(ws.hist(t), r.top_p, part, bins);
    sure = (float)bins[0], last = (float)(bins[1] + 1);
  }
  auto add_to_list = [&](int tile, const float (&l)[16], const float (&y)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const bool add = y[e] >= sure && y[e] < last;
      const uint64_t who = __ballot(add);
      if (who) {
        uint32_t at = 0;
        if (lane == __ffsll((long long)who) - 1) at = atomicAdd(&nfound, (uint32_t)__popcll(who));
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, __ffsll((long long)who) - 1);
        at += (uint32_t)__popcll(who & ((1ull << lane) - 1));
        if (add && at < kList)
          found[at] = (uint64_t)~order_key(l[e]) << 32 | (uint32_t)(tile * kTile + tile_at(e));
      }
    }
  };
  uint64_t before = 0, all = 0;
  for (int tile = blockIdx.x * kSomeWaves + wave; tile < ws.tiles; tile += kSomeWaves * gridDim.x) {
    float l[16], y[16];
    if (kind == kTopK && (mx - ws.tmax(t)[tile]) * sc >= last) continue;
    load_tile<BF16>(p, t, tile, l);
    bool any = false;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      y[e] = kind == kFull ? 0.f : (mx - l[e]) * sc;
      any |= y[e] >= sure && y[e] < last;
    }
    if (__ballot(any)) add_to_list(tile, l, y);
    if (kind == kTopK) continue;
    // sums of what is above the listed bins, and of that with min_p; of all
    uint64_t in = 0, keep = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const uint64_t f = exp2_fixed44(((double)l[e] - (double)mx) * r.rt), g = y[e] < sure ? f : 0;
      all += f;
      in += g;
      if (r.min_w) keep += g >= r.min_w ? g : 0;
    }
    before += in;
    keep = dpp_sum_u64(r.min_w ? keep : in);
    if (lane == 0) ws.tsum(t)[tile] = keep;
  }
  __syncthreads();
  const uint32_t n = nfound;
  if (n) {
    if (threadIdx.x == 0) at0 = atomicAdd(&info->n, n);
    __syncthreads();
    uint64_t* const list = ws.list(t);
    for (uint32_t i = threadIdx.x; i < n && at0 + i < kList; i += 64 * kSomeWaves) list[at0 + i] = found[i];
  }
  if (kind == kTopP) {
    before = dpp_sum_u64(before), all = dpp_sum_u64(all);
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

constexpr int kSub = kRowThreads;  // sub-bins of the list's range, one per thread
struct DrawLds {
  union {
    RowLds row;
    struct {
      uint64_t few[kList];  // the entries of the border's sub-bin
      uint64_t w[kSub];
      uint64_t tile[kSampleMaxV / kTile];
      uint32_t n[kSub];
    } f;
  };
  uint64_t wpart[kRowThreads / 64];
  uint32_t npart[kRowThreads / 64];
  float s[kRowThreads / 64];
  uint64_t border, base, upto;  // upto: the sum of the weights up to the border entry
  int at, bin, nfew;
};

// Exclusive block-wide prefix of (w, n) by thread; the totals in W and Nn.
__device__ __forceinline__ void draw_scan(DrawLds& s, uint64_t& w, uint32_t& n, uint64_t& W, uint32_t& Nn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t c = wave_scan_u64(w);
  const uint32_t d = wave_scan_u32(n);
  __syncthreads();
  if (lane == 63) s.wpart[wave] = c, s.npart[wave] = d;
  __syncthreads();
  uint64_t base = 0;
  uint32_t bn = 0;
  W = 0, Nn = 0;
  for (int i = 0; i < kRowThreads / 64; i++) {
    if (i == wave) base = W, bn = Nn;
    W += s.wpart[i], Nn += s.npart[i];
  }
  w = base + c - w, n = bn + d - n;
}

// A list entry: ~key in the upper half, its place in the vocabulary in the lower, so that rising entries are the order.
__device__ __forceinline__ float entry_logit(uint64_t a) { return key_value(~(uint32_t)(a >> 32)); }

// The value of the lane whose number differs in bit M.
template <int M>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
  if constexpr (M == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);  // quad_perm 1 0 3 2
  else if constexpr (M == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);  // 2 3 0 1
  else if constexpr (M == 4) return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x101F);  // xor 4
  else if constexpr (M == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false);  // row_ror:8
  else if constexpr (M == 16) {
    const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? x[0] : x[1];
  } else {
    const auto x = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? x[0] : x[1];
  }
}
// One exchange of a bitonic sort over a wave: runs of K lanes rise and fall in turn; w goes along with v.
template <int K, int M>
__device__ __forceinline__ void exchange(uint64_t& v, uint64_t& w) {
  const u32x2 a = __builtin_bit_cast(u32x2, v), b = __builtin_bit_cast(u32x2, w);
  const uint64_t x = __builtin_bit_cast(uint64_t, u32x2{xor_lane<M>(a[0]), xor_lane<M>(a[1])});
  const uint64_t y = __builtin_bit_cast(uint64_t, u32x2{xor_lane<M>(b[0]), xor_lane<M>(b[1])});
  const bool low = ((threadIdx.x & M) == 0) == ((threadIdx.x & K) == 0);  // this lane keeps the smaller
  if (low ? x < v : x > v) v = x, w = y;
}
template <int K, int M>
__device__ __forceinline__ void merge_lanes(uint64_t& v, uint64_t& w) {
  exchange<K, M>(v, w);
  if constexpr (M > 1) merge_lanes<K, M / 2>(v, w);
}
// Sorts v over the 64 lanes, rising, w going along.
__device__ __forceinline__ void sort_lanes(uint64_t& v, uint64_t& w) {
  merge_lanes<2, 1>(v, w);
  merge_lanes<4, 2>(v, w);
  merge_lanes<8, 4>(v, w);
  merge_lanes<16, 8>(v, w);
  merge_lanes<32, 16>(v, w);
  merge_lanes<64, 32>(v, w);
}

// DIRECT: the list is the row itself (V <= kList), and there is no other launch.
template <bool BF16, bool DIRECT>
__global__ __launch_bounds__(kRowThreads) void k_sample_draw(SampleArgs p, SampleWs ws) {
  __shared__ DrawLds s;
  constexpr int PER = kList / kRowThreads;
  static_assert(kSampleMaxV / kTile <= kRowThreads, "a tile per thread");
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  // loads that depend on nothing, together (a row's draw is a chain of memory latencies)
  const RowPar r = row_par(p, t);
  RowInfo in{};
  float tile_max = -INFINITY;
  uint64_t tile_sum = 0, a[PER], f[PER];
  if constexpr (DIRECT) {
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int i = kRowThreads * q + tid;
      const float l = load_logit<BF16>(p, t, min(i, p.V - 1));
      a[q] = (uint64_t)~order_key(i < p.V ? l : -INFINITY) << 32 | (uint32_t)i;
      tile_max = fmaxf(tile_max, l);
    }
  } else {
    in = *ws.info(t);
    if (tid < ws.tiles) tile_max = ws.tmax(t)[tid], tile_sum = ws.tsum(t)[tid];
    a[0] = ws.list(t)[tid];
  }
  const double u = row_u(p, t);
  float mx = dpp_max_f(tile_max);
  if (lane == 0) s.s[tid >> 6] = mx;
  if (tid == 0) s.at = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 64; i++) mx = fmaxf(mx, s.s[i]);
  const int kind = DIRECT && mx < INFINITY && r.k < p.V && !r.greedy && mx > -INFINITY ? kTopK : row_kind(r, p.V, mx);
  auto done = [&](int token, float prob) {
    p.token[t] = token;
    if (p.prob) p.prob[t] = prob;
  };
  if (kind == kNothing) {
    if (tid == 0) done(-1, 0.f);
    return;
  }
  if (kind == kGreedy) {  // the first tile with the maximum, and its place there
    if constexpr (DIRECT) {
#pragma unroll
      for (int q = PER - 1; q >= 0; q--)
        if (entry_logit(a[q]) == mx) atomicMin(&s.at, (int)(uint32_t)a[q]);
      __syncthreads();
      if (tid == 0) done(s.at, 1.f);
      return;
    }
    if (tile_max == mx) atomicMin(&s.at, tid);
    __syncthreads();
    const int first = s.at * kTile;
    __syncthreads();
    if (tid == 0) s.at = 0x7fffffff;
    __syncthreads();
    for (int i = first + tid; i < min(first + kTile, p.V); i += kRowThreads)
      if (load_logit<BF16>(p, t, i) == mx) atomicMin(&s.at, i);
    __syncthreads();
    if (tid == 0) done(s.at, 1.f);
    return;
  }
  const int n = DIRECT ? p.V : (int)min(in.n, (uint32_t)kList + 1);
  if (kind == kTopK && n <= 64) {  // a short list by one wave: sorted, cut, and sorted again into the vocabulary's order
    if (tid >= 64) return;
    uint64_t e = lane < n ? a[0] : ~0ull, w = lane < n ? weight(entry_logit(a[0]), mx, r.rt) : 0;
    sort_lanes(e, w);
    if (lane >= r.k) w = 0;
    const uint64_t upto = wave_scan_u64(w);
    const double part = r.top_p * (double)readlane_u64(upto, 63);
    if (r.top_p < 1.0 && lane > 0 && !((double)(upto - w) < part)) w = 0;
    if (w < r.min_w) w = 0;
    uint64_t place = e << 32 | (uint32_t)lane;
    sort_lanes(place, w);
    const uint64_t sum = wave_scan_u64(w), total = readlane_u64(sum, 63);
    const uint64_t hit = __ballot(w != 0 && (double)sum > u * (double)total);
    if (hit && lane == __ffsll((long long)hit) - 1) done((int)(place >> 32), (float)((double)w / (double)total));
    return;
  }
  bool listed = kind != kOneBlock && n <= kList;
  // what is kept: the prefix of the order up to the entry `border`, as far as it has min_p
  uint64_t border = ~0ull;
  int sub[PER];
  if (listed && (DIRECT || kind != kFull)) {
    // the list in registers (what has a weight), over 512 sub-bins of its range of logits
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int q = 0; q < PER; q++) {
      const int i = kRowThreads * q + tid;
      if (!DIRECT && q > 0) a[q] = 0;
      f[q] = 0;
      if (kRowThreads * q >= n) continue;
      if (!DIRECT && q > 0) a[q] = ws.list(t)[min(i, n - 1)];
      const float l = entry_logit(a[q]);
      if (i < n) f[q] = weight(l, mx, r.rt);
      if (f[q]) lo = fminf(lo, l), hi = fmaxf(hi, l);
    }
    lo = -dpp_max_f(-lo), hi = dpp_max_f(hi);
    if (lane == 0) s.npart[tid >> 6] = __float_as_uint(lo), s.s[tid >> 6] = hi;
    s.f.w[tid] = 0, s.f.n[tid] = 0;
    __syncthreads();
    lo = INFINITY, hi = -INFINITY;
    for (int i = 0; i < kRowThreads / 64; i++) lo = fminf(lo, __uint_as_float(s.npart[i])), hi = fmaxf(hi, s.s[i]);
    const float sc = hi > lo ? fminf((float)(kSub - 1) / (hi - lo), 3e38f) : 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) {
      sub[q] = -1;
      if (f[q]) {
        sub[q] = min((int)((hi - entry_logit(a[q])) * sc), kSub - 1);
        atomicAdd(&s.f.n[sub[q]], 1u);
        atomicAdd((unsigned long long*)&s.f.w[sub[q]], (unsigned long long)f[q]);
      }
    }
    __syncthreads();
    const uint64_t own_w = s.f.w[tid];
    const uint32_t own_n = s.f.n[tid];
    uint64_t bw = own_w, W;
    uint32_t bn = own_n, Nn;
    draw_scan(s, bw, bn, W, Nn);  // this thread's sub-bin: what comes before it
    const uint32_t k = min((uint32_t)r.k, Nn);
    if (tid < ws.tiles) s.f.tile[tid] = !DIRECT && kind == kTopP ? tile_sum : 0;
    // The border by count (top-k: the k-th entry, or the last), then by weight (the first entry at which the sum reaches want, `base`
    // before the list): its sub-bin, and there, among few, the entry.
#pragma clang loop unroll(disable)
    for (int step = 0; step < 2; step++) {
      const bool by_count = step == 0;
      if (by_count ? kind != kTopK : r.top_p >= 1.0) continue;
      const uint64_t base = !DIRECT && kind == kTopP ? in.before : 0;
      double want = 0;
      if (!by_count) {
        want = r.top_p * (double)(kind == kTopK ? s.upto : DIRECT ? W : in.all);
        // the border lies above what is listed, or below
        listed = (base == 0 || (double)base < want) && (double)(base + W) >= want;
        if (!listed) break;
      }
      if (tid == 0) s.bin = kSub - 1, s.nfew = 0;
      __syncthreads();
      if (own_n) {
        const bool here = by_count ? bn < k && bn + own_n >= k
                                   : ((double)(base + bw) < want || base + bw == 0) && (double)(base + bw + own_w) >= want;
        if (here) s.bin = tid;
      }
      __syncthreads();
      const int bin = s.bin;
      if (tid == bin) s.base = base + bw, s.npart[0] = bn;
#pragma unroll
      for (int q = 0; q < PER; q++)
        if (sub[q] == bin) s.f.few[atomicAdd(&s.nfew, 1)] = a[q];
      __syncthreads();
      const int m = s.nfew;
      if (m > 64) sort_lds(s.f.few, m);
      if (tid < 64) {
        uint64_t c = s.base;
        uint32_t d = s.npart[0];
        uint64_t at = ~0ull, upto = 0;
        for (int i0 = 0; i0 < m && at == ~0ull; i0 += 64) {  // 64 entries at a time: unsorted if there are no more
          const bool live = i0 + lane < m;
          const uint64_t x = live ? s.f.few[i0 + lane] : ~0ull;
          const uint64_t w = live ? weight(entry_logit(x), mx, r.rt) : 0;
          uint64_t before = c;
          uint32_t rank = d;
          for (int j = 0; j < min(m - i0, 64); j++) {
            const uint64_t y = readlane_u64(x, j), v = readlane_u64(w, j);
            if (y < x) before += v, rank++;
            c += v;
          }
          d += min(m - i0, 64);
          const bool hit = live && (by_count ? rank == k - 1
                                             : ((double)before < want || before == 0) && (double)(before + w) >= want);
          const uint64_t who = __ballot(hit);
          if (who) {
            const int j = __ffsll((long long)who) - 1;
            at = readlane_u64(x, j), upto = readlane_u64(before + w, j);
          }
        }
        if (lane == 0) s.border = at, s.upto = upto;
      }
      __syncthreads();
      border = s.border < border ? s.border : border;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; q++)
      if (sub[q] >= 0 && a[q] <= border && f[q] >= r.min_w)
        atomicAdd((unsigned long long*)&s.f.tile[(uint32_t)a[q] / kTile], (unsigned long long)f[q]);
  } else if (listed) {
    if (tid < ws.tiles) s.f.tile[tid] = tile_sum;
  }
  __syncthreads();
  if (!listed) {
    row_sample<BF16>(s.row, p, t);
    return;
  }
  uint64_t total, W;
  uint32_t z = 0, zz;
  const uint64_t mine = tid < ws.tiles ? s.f.tile[tid] : 0;
  uint64_t before = mine;
  draw_scan(s, before, z, total, zz);
  const double want = u * (double)total;
  if (mine && (double)(before + mine) > want) atomicMin(&s.at, tid);
  __syncthreads();
  const int tile = min(s.at, ws.tiles - 1);
  if (tid == tile) s.base = before;
  __syncthreads();
  const uint64_t base = s.base;
  if (tid == 0) s.at = 0x7fffffff;
  constexpr int RUN = kTile / kRowThreads;  // neighbouring logits per thread
  const int i0 = tile * kTile + RUN * tid;
  uint64_t fx[RUN];
  before = 0;
#pragma unroll
  for (int q = 0; q < RUN; q++) {
    const int i = i0 + q;
    const float l = load_logit<BF16>(p, t, min(i, p.V - 1));
    const uint64_t e = (uint64_t)~order_key(l) << 32 | (uint32_t)i;
    const uint64_t w = weight(l, mx, r.rt);
    fx[q] = i < p.V && e <= border && w >= r.min_w ? w : 0;
    before += fx[q];
  }
  z = 0;
  draw_scan(s, before, z, W, zz);
  before += base;
  int at = 0x7fffffff;
  uint64_t fat = 0;
#pragma unroll
  for (int q = 0; q < RUN; q++) {
    before += fx[q];
    if (fx[q] && (double)before > want && at == 0x7fffffff) at = i0 + q, fat = fx[q];
  }
  if (fat) atomicMin(&s.at, at);
  __syncthreads();
  if (fat && at == s.at) done(at, (float)((double)fat / (double)total));
}

size_t sample_workspace(int T, int V) { return V <= kList ? 0 : (size_t)std::min(T, kRowsPerLaunch) * sample_ws(V).row; }

template <bool BF16>
static int launch_sample_rows(const SampleArgs& a, const SampleWs& ws, hipStream_t st) {
  // a row that fits the list: one launch (us, against the four: 4 x 4000 top-p 14.6 for 24.0, 17 x 1455 mixed 14.4 for 25.4,
  // 110 x 4079 min-p 11.6 for 15.2, 1000 x 4096 top-p 64 for 83; with 16 entries per thread for up to 8192 4 x 8192 62 for 24)
  if (a.V <= kList) {
    hipLaunchKernelGGL((k_sample_draw<BF16, true>), dim3(a.T), dim3(kRowThreads), 0, st, a, ws);
    return check_launch("sample");
  }
  const auto blocks = [&](int waves) { return (ws.tiles + waves - 1) / waves; };
  // a wave per tile where that does not fill the device; past it fewer blocks, which set up or join a histogram each (128 rows
  // of 248320: 512 / 768 / 1024 / 2048 blocks of k_sample_collect 122 / 116 / 118 / 122 us a call)
  const auto some = [&](int most) { return dim3(std::min(blocks(kSomeWaves), std::max(1, most / a.T)), a.T); };
  const dim3 some_threads(64 * kSomeWaves);
  hipLaunchKernelGGL(k_sample_max<BF16>, dim3(blocks(4), a.T), dim3(256), 0, st, a, ws);
  if (a.top_k || a.top_p) hipLaunchKernelGGL(k_sample_border<BF16>, some(512), some_threads, 0, st, a, ws);
  hipLaunchKernelGGL(k_sample_collect<BF16>, some(kCollect), some_threads, 0, st, a, ws);
  hipLaunchKernelGGL((k_sample_draw<BF16, false>), dim3(a.T), dim3(kRowThreads), 0, st, a, ws);
  return check_launch("sample");
}

int launch_sample(const void* logits, int logits_bf16, int T, int V, int ld, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const float* u, int* token, float* prob, void* mem,
                  size_t ws_bytes, hipStream_t st) {
  SampleWs ws = sample_ws(V);
  ws.base = (char*)mem;
  const size_t need = sample_workspace(T, V);
  if (need && (!mem || ws_bytes < need))
    return fail(IFD_ERR_WORKSPACE, "sample needs %zu bytes of workspace, got %zu", need, ws_bytes);
  const int step = need ? kRowsPerLaunch : 1 << 20;  // (a grid holds less than 2^32 threads)
  for (int t = 0; t < T; t += std::min(step, T - t)) {
    auto off = [&](auto* q) { return q ? q + t : q; };
    const SampleArgs a{(const char*)logits + (size_t)t * ld * (logits_bf16 ? 2 : 4), std::min(T - t, step), V, ld,
                       off(temperature), off(top_k), off(top_p), off(min_p), off(u), off(token), off(prob)};
    IFD_TRY(logits_bf16 ? launch_sample_rows<true>(a, ws, st) : launch_sample_rows<false>(a, ws, st));
  }
  return IFD_OK;
}

}  // namespace ifd
