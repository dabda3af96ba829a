// q8_sample.hip -- token ids drawn from rows of logits, with temperature, top-k,
// top-p and min-p, from given random numbers.
//
// Per row: y_i = x_i / T, w_i = exp(y_i - y_max).  Tokens are ordered by x
// descending, then by index; each filter keeps a head of that order, so the kept
// tokens are known by their sum W alone, and the drawn one is the first whose
// running sum exceeds u W.  Nothing is sorted: a histogram over bins of y of
// width 1 / 16 gives the running sums at bin borders, and only the bins that the
// three borders (k-th token, top_p of the mass, u W) fall into are looked into.
//
// Weights are held relative to their bin's middle, within 1 / 32 of 1, as whole
// numbers of 2^-40: integer sums, so the order of the atomics does not matter and
// equal inputs give equal ids; over bins they are summed in f64 in a fixed order.
// Bins reach 64 below the maximum (e^-64 of the largest weight: 2^22 such tokens
// are 2^-70 of the sum, less than a f64 sum can hold).  With the series' error they are
// within 2^-39 of exp, so an id is not the definition's where u or a border lies that close
// to a running sum.  Sums in f32 would be off by 2^-24 of the mass, as much as the step of
// a f32 u.
#include "q8_device.h"
#include "q8_launch.h"

#include <algorithm>

namespace q8 {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));   // any f32 address

constexpr int kBins = 1024;
constexpr double kBinsPerUnit = 16.0;
constexpr int kHistThreads = 512;
constexpr int kPerThread = 16;                        // logits a thread holds
constexpr int kChunk = kHistThreads * kPerThread;
constexpr int kList = 8192;                           // members of a bin kept in LDS
// A sum that meets a border exactly (equal logits, a power of two of the mass) has met
// it, whatever the last bits of the f64 sums say.  The margin covers f64 additions only, so
// both sides of a comparison are sums of the same weights: a histogram's, which are up to
// 2^-39 off in one direction, are not compared with those of exp.
constexpr double kTie = 0x1p-45;
constexpr int kMaxSlices = 64;
constexpr int kTop = 256;                             // tokens of a slice that are listed
// Members of a bin that are compared with each other (up to 256 took 8 to 11 us, a
// narrowing step before takes 3).
constexpr uint32_t kCompared = 64;

// A slice's part of its row: sums and counts of the bins below its own maximum.
// Behind them its largest tokens: all those of its first `upto` bins.
struct SampleSlice {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  double top;                                         // bin number of the maximum
  float max;                                          // -inf: no token
  int index;                                          // its lowest index
  int upto, listed;
  uint64_t list[kTop];
};

// y = x / T and the bin that holds it, as whole numbers in f64 (16 y to the nearest,
// exact); infinities have a bin of their own.
struct BinOf {
  double y, a;
};
__device__ __forceinline__ BinOf bin_of(float x, double inv_t) {
#pragma clang fp contract(off)                        // (the histogram's loop rounds alike)
  BinOf b;
  b.y = (double)x * inv_t;
  if (x == INFINITY) b.y = INFINITY;                  // (T = inf: inf * 0)
  b.a = __builtin_rint(b.y * kBinsPerUnit);
  return b;
}
// Bins below the one of the maximum; kBins: out of reach.
__device__ __forceinline__ int below(double top, double a) {
  const double d = top - a;
  return top == a ? 0 : d < (double)kBins ? (int)d : kBins;
}
// exp(y - middle of the bin) 2^40 as a whole number, from 16 times that difference, at
// most 1 / 2: the series to the 5th power is 2^-39 off at most.  The last step adds 2^52 as
// well, which leaves the integer in the low bits.
__device__ __forceinline__ uint64_t weight16(double z) {
  constexpr double h = 1.0 / kBinsPerUnit, one = 0x1p40;
  double p = one * h * h * h * h * h / 120.0;
  p = __builtin_fma(p, z, one * h * h * h * h / 24.0);
  p = __builtin_fma(p, z, one * h * h * h / 6.0);
  p = __builtin_fma(p, z, one * h * h / 2.0);
  p = __builtin_fma(p, z, one * h);
  const double w = __builtin_fma(p, z, 0x1p52 + one);
  return __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
}
__device__ __forceinline__ uint64_t weight(const BinOf &b) {
  return weight16(__builtin_isinf(b.y) ? 0.0 : b.y * kBinsPerUnit - b.a);
}

// A token's place in the order, ascending: larger values first, then lower indices.
__device__ __forceinline__ uint64_t place(float x, int i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);           // (-0 as 0)
  const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;         // ascending with x
  return (uint64_t)~key << 32 | (uint32_t)i;
}

// A value that is the same in all lanes, in scalar registers.
template <class T> __device__ __forceinline__ T uniform(T v) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    int w[W];
  } x = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int i = 0; i < W; ++i) x.w[i] = __builtin_amdgcn_readfirstlane(x.w[i]);
  return __builtin_bit_cast(T, x);
}

// Inclusive sums over a wave's lanes, in one fixed order.
template <class T> __device__ __forceinline__ T wave_sums(T v) {
  return wave_scan(v, [](T a, T b) { return a + b; });
}
// Over the block's threads; *all: the last one's.  wsum: a value a wave; the caller
// waits before it writes there again.
template <int NT, class T> __device__ __forceinline__ T block_sums(T v, T *wsum, T *all) {
  static_assert(NT / 64 <= 16, "the waves' sums are a row of lanes");
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  v = wave_sums(v);
  if (lane == 63) wsum[w] = v;
  __syncthreads();
  T s = wave_sums((lane & 15) < NT / 64 ? wsum[lane & 15] : (T)0);     // (the first row of lanes)
  struct Words {
    int w[sizeof(T) / 4];
  } x = __builtin_bit_cast(Words, s), y, z;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) {
    y.w[i] = w > 0 ? __builtin_amdgcn_readlane(x.w[i], w > 0 ? w - 1 : 0) : 0;
    z.w[i] = __builtin_amdgcn_readlane(x.w[i], NT / 64 - 1);
  }
  *all = __builtin_bit_cast(T, z);
  return __builtin_bit_cast(T, y) + v;
}

// Four times 4 logits of a row, the u-th at i + u * step, -inf from `end` on.  The loads
// are not in a branch (those of a place behind the end take the row's start), so they
// all go out together.
template <int STEP>
__device__ __forceinline__ void load16(const float *x, int64_t i, int64_t end, float (&v)[16]) {
  if (end < 4) {                                      // (uniform: a row of 1 to 3 logits)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = e < 4 && i + e < end ? x[i + e] : -INFINITY;
    return;
  }
  f32x4 y[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t at = i + u * STEP;
    y[u] = *reinterpret_cast<const f32x4_u *>(x + (at + 4 <= end ? at : 0));
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t at = i + u * STEP;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[4 * u + e] = at + 4 <= end ? y[u][e] : -INFINITY;
    if (at < end && at + 4 > end) {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (at + e < end) v[4 * u + e] = x[at + e];
    }
  }
}

struct RowSettings {
  double inv_t;
  int64_t k;
  double top_p, min_p, u;
  int greedy, pad;
};
__device__ __forceinline__ RowSettings settings(const SampleArgs &a, int64_t row) {
  const float *p = a.param + row;
  RowSettings s;
  const float t = p[0];
  s.greedy = !(t > 0.0f);
  s.inv_t = s.greedy ? 1.0 : 1.0 / (double)t;
  const int k = a.topk[row];
  s.k = k > 0 ? k : INT64_MAX;
  const float tp = p[a.rows], mp = p[2 * a.rows], u = p[3 * a.rows];
  s.top_p = tp < 1.0f ? (double)tp : 2.0;             // (NaN: off)
  s.min_p = mp > 0.0f ? (double)fminf(mp, 1.0f) : 0.0;
  s.u = u > 0.0f ? (double)fminf(u, 1.0f - 0x1p-24f) : 0.0;
  return s;
}

// ---- pass 1: the histogram of a slice, grid (slices, rows) ---------------------
// Bound: an LDS atomic and 12 f64 operations a logit (without a branch each where no lane
// needs one: no change), beside one read of the logits
// (medians: 256 rows of 151936, 156 MB, 43 us: 3.6 TB/s, half of what a plain read reaches;
// 64 rows of 128256 21 us; a row alone 9.8 us, its chain).  A block walks its slice in chunks that it holds in registers; the
// bins are a ring whose head is the slice's largest value so far, so the row's
// maximum need not be known first.
__global__ __launch_bounds__(kHistThreads, 8) void sample_hist_kernel(SampleArgs a, int64_t row0,
                                                                      int64_t slice_len) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ float wmax[kHistThreads / 64];
  __shared__ uint64_t wsum[kHistThreads / 64], wsum2[kHistThreads / 64];
  __shared__ int best, upto, listed;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.y;
  const float *x = a.x + row * a.ldx;
  SampleSlice *out = reinterpret_cast<SampleSlice *>(a.ws) + (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t i0 = blockIdx.x * slice_len, i1 = min(i0 + slice_len, a.n);
  float v[kPerThread];
  static_assert(kPerThread == 16, "load16");
  auto load = [&](int64_t c) { load16<4 * kHistThreads>(x, c + 4 * t, i1, v); };
  load(i0);
  const RowSettings s = settings(a, row);
  const bool counts = s.k < a.n;
  for (int b = t; b < kBins; b += kHistThreads) {
    mass[b] = 0;
    count[b] = 0;
  }
  float top = -INFINITY;                              // of the slice so far
  double top_bin = -INFINITY;
  int head = 0, index = INT32_MAX;
  for (int64_t c = i0; c < i1; c += kChunk) {
    if (c > i0) load(c);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) m = fmaxf(m, v[e]);            // (NaN: not taken)
    m = wave_max(m);
    if ((t & 63) == 0) wmax[t >> 6] = m;
    if (t == 0) best = INT32_MAX;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kHistThreads / 64; ++w) m = fmaxf(m, wmax[w]);
    if (m > top) {                                    // (the whole block)
      // the ring turns: bins that come in above are cleared
      const double nb = bin_of(m, s.inv_t).a;
      const double up = nb - top_bin;
      const int turn = nb == top_bin ? 0 : up < (double)kBins ? (int)up : kBins;
      for (int b = t; b < turn; b += kHistThreads) {
        const int at = (head - 1 - b) & (kBins - 1);
        mass[at] = 0;
        count[at] = 0;
      }
      head = (head - turn) & (kBins - 1);
      top = m;
      top_bin = nb;
      index = INT32_MAX;
      int mine = INT32_MAX;
#pragma unroll
      for (int q = kPerThread / 4 - 1; q >= 0; --q)
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (v[4 * q + e] == m) mine = (int)(c + 4 * (q * kHistThreads + t) + e);
      if (mine != INT32_MAX) atomicMin(&best, mine);
      __syncthreads();
      index = best;
    }
    auto add = [&](int at, uint64_t w) {
      atomicAdd(reinterpret_cast<unsigned long long *>(&mass[at]), (unsigned long long)w);
      if (counts) atomicAdd(&count[at], 1u);
    };
    // Adding 1.5 2^52 rounds to a whole number, whose low bits are the bin's; further
    // from 0 than that allows, the plain way.
    if (!s.greedy && __builtin_fabs(top_bin) < 0x1p30) {
      // The product is rounded before the addition, as bin_of rounds it: one fused operation
      // would put a logit between two bins into another one than the maximum's says.
#pragma clang fp contract(off)
      const double scale = s.inv_t * kBinsPerUnit, least = top_bin - kBins + 0.5;
      const uint32_t from = (uint32_t)(head + (int)top_bin);
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        const double z = (double)v[e] * scale, whole = z + 0x1.8p52;
        const uint64_t w = weight16(z - (whole - 0x1.8p52));
        if (z > least)                                // (not NaN; of -inf it is that or -inf)
          add((int)((from - (uint32_t)__builtin_bit_cast(uint64_t, whole)) & (kBins - 1)), w);
      }
    } else if (!s.greedy) {
#pragma unroll 1
      for (int e = 0; e < kPerThread; ++e) {
        float x = v[0];
#pragma unroll
        for (int i = 1; i < kPerThread; ++i) x = i == e ? v[i] : x;
        const BinOf b = bin_of(x, s.inv_t);
        const int d = below(top_bin, b.a);
        if (x > -INFINITY && d < kBins) add((head + d) & (kBins - 1), weight(b));
      }
    }
    __syncthreads();                                  // wmax, best, the ring's head
  }
  // A slice of one chunk lists its largest tokens from the registers: those of as many
  // bins as hold kTop (weights are within 1 / 32 of 2^40, so sums bound the counts).
  const bool lists = i1 - i0 <= kChunk && !s.greedy && top > -INFINITY &&
                     (counts || s.top_p < 1.0 || s.min_p > 0.0);
  if (t == 0) upto = listed = 0;
  if (lists) {
    const int b0 = (head + 2 * t) & (kBins - 1), b1 = (head + 2 * t + 1) & (kBins - 1);
    const uint64_t m0 = mass[b0], m1 = mass[b1];
    uint64_t every;
    const uint64_t all = block_sums<kHistThreads>(m0 + m1, wsum, &every);
    constexpr uint64_t kMost = (uint64_t)(kTop * 15 / 16) << 40;
    // (0 and set before the barrier in the sums; the bins that fit are the first ones)
    if (all <= kMost) atomicMax(&upto, 2 * t + 2);
    else if (all - m1 <= kMost) atomicMax(&upto, 2 * t + 1);
    __syncthreads();
    // by value, from a little below the bins on: more do no harm as far as there is room
    float lo = INFINITY;
    if (upto > 0) {
      const double at = (top_bin - (double)upto + 0.5) / kBinsPerUnit / s.inv_t;
      lo = __builtin_isinf(top_bin) ? INFINITY
           : at == at               ? (float)(at - __builtin_fabs(at) * 0x1p-22 - 0x1p-140)
                                    : -INFINITY;
    }
    uint32_t mine = 0;                                // which of v
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) mine |= (uint32_t)(v[e] >= lo && v[e] > -INFINITY) << e;
    const uint64_t have = __builtin_popcount(mine);
    uint64_t n;
    const uint64_t to = block_sums<kHistThreads>(have, wsum2, &n);
    const bool fits = n <= kTop;                      // (the whole block)
    if (t == 0) {
      listed = fits ? (int)n : 0;
      if (!fits) upto = 0;
    }
    uint64_t *at = out->list + (to - have);
#pragma unroll
    for (int q = 0; q < kPerThread / 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (fits && mine >> (4 * q + e) & 1)
          *at++ = place(v[4 * q + e], (int)(i0 + 4 * (q * kHistThreads + t) + e));
  }
  __syncthreads();
  if (t == 0) {
    out->top = top_bin;
    out->max = top;
    out->index = index;
    out->upto = upto;
    out->listed = listed;
  }
  if (s.greedy) return;
  for (int b = t; b < kBins; b += kHistThreads) {
    const int at = (head + b) & (kBins - 1);
    out->mass[b] = mass[at];
    if (counts) out->count[b] = count[at];
  }
}

// ---- pass 2: one block of kBins threads per row --------------------------------
// The slices' bins are added up; where the kept tokens are few they are sorted and
// the filters and the draw are one running sum, else each border's bin is looked into.
// Bound: the chain of dependent reads, searches and block-wide sums (14 us where few
// tokens are kept, a third of it fetching code for its first use), and for rows that keep many
// the second read of their logits by one CU: 12 us for 128256, with the selections behind it
// 46 us (median of 64 mixed rows; 35 where the draws are easy) to 67 us (256 rows of 151936
// with top-p, 58 at best; their read alone takes 23 us, 6.8 TB/s).

// The bin that a border falls into, the sums before it and up to it, its own.
struct BorderBin {
  uint64_t mass;
  double before, unit;                                // unit: weight of 1 in this bin
  uint32_t count, upto;
  int bin, pad;                                       // -1: none in this wave
};

struct SelectLds {
  __attribute__((aligned(16))) uint64_t mass[kBins];                               // (sorting: places; sums as f64)
  uint32_t count[kBins];
  uint64_t list[kList];                               // places of the members
  uint64_t wsum64[kBins / 64];
  double wsumd[2][kBins / 64];
  uint32_t wsum32[kBins / 64];
  BorderBin border[2][2][kBins / 64];
  uint64_t found;
  uint64_t before;                                    // sum before what was found
  uint32_t n, where;
  uint32_t key[4];
};

__device__ __forceinline__ float value_of(uint64_t place) {
  const uint32_t key = ~(uint32_t)(place >> 32);
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The row and its slices, whose heads are one a lane.
struct RowAt {
  const float *x;
  int64_t n;
  double inv_t;
  const SampleSlice *slices;
  int nslices;
  double top;                                         // lane's slice: see SampleSlice
  float max;
  int upto, listed;
};

// Values of a bin: from lo to hi.  (bin_of is monotone, so floats say exactly what f64
// would.)
struct Values {
  float lo, hi;
  __device__ __forceinline__ bool has(float x) const { return x >= lo && x <= hi; }
};
// The first float, in ascending order, of a bin from `bin` on (past: behind it); NaN-free.
// The wave halves the 2^32 patterns six times in 64 parts.
__device__ __forceinline__ uint32_t first_key(double bin, bool past, double inv_t) {
  const uint32_t least = 0x007fffffu + 1, most = 0xff800000u;          // keys of -FLT_MAX, +inf
  uint32_t at = least;                                // (the answer lies from at on)
#pragma unroll 1
  for (int sh = 26; ; sh = sh > 6 ? sh - 6 : 0) {
    const uint64_t k = (uint64_t)at + ((uint64_t)(threadIdx.x & 63) << sh);
    const uint32_t key = k < most ? (uint32_t)k : most;
    const float x = __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
    const double a = bin_of(x, inv_t).a;
    // lanes are ascending: the last one before the bin
    const uint64_t before = __builtin_amdgcn_ballot_w64(past ? a <= bin : a < bin);
    if (before == 0) return at;
    const uint64_t n = (uint64_t)at + ((uint64_t)(63 - __builtin_clzll(before)) << sh);
    if (n >= most) return most + 1;                   // (none)
    at = (uint32_t)n;
    if (sh == 0) return at + 1;
  }
}
__device__ __forceinline__ float float_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ Values values_of(uint32_t first, uint32_t behind) {
  if (first >= behind) return {INFINITY, -INFINITY};  // (no float)
  return {float_of(first), float_of(behind - 1)};
}

// Puts the tokens of the bins from `from` up to `to`, and of `also`, into LDS as far as they
// fit; their number is l.n.  From the slices' lists where those hold them all, else
// from the row.  *values1, *values2: the
// values of both.
__device__ __forceinline__ void gather(const RowAt &r, double from, double to, double also, SelectLds &l,
                                       Values *values1, Values *values2) {
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  // a border a wave
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < (also == from ? 2 : 4)) {
    const double bin = wave == 0 ? from : wave == 1 ? to : also;
    const uint32_t k = bin == INFINITY && (wave & 1) ? 0xff800001u : first_key(bin, wave & 1, r.inv_t);
    if ((threadIdx.x & 63) == 0) l.key[wave] = k;
  }
  __syncthreads();
  const Values one = values_of(uniform(l.key[0]), uniform(l.key[1]));
  const Values two = also == from ? one : values_of(uniform(l.key[2]), uniform(l.key[3]));
  *values1 = one;
  *values2 = two;
  const double least = __builtin_fmin(from, also);
  const int lane = threadIdx.x & 63;
  const bool all = __builtin_amdgcn_ballot_w64(lane < r.nslices && r.max > -INFINITY && least <= r.top &&
                                               below(r.top, least) >= r.upto) == 0;
  // a wave's candidates take their places together: `n` of this lane's
  auto places = [&](uint32_t n) {
    const uint32_t upto = wave_sums(n);
    const uint32_t sum = __builtin_amdgcn_readlane(upto, 63);
    uint32_t at = 0;
    if (sum) {
      if (lane == 0) at = atomicAdd(&l.n, sum);
      at = __builtin_amdgcn_readfirstlane(at);
    }
    return at + upto - n;
  };
  if (all) {
    constexpr int kU = 4;
    for (int e0 = 0; e0 < r.nslices * kTop; e0 += kU * kBins) {
      uint64_t p[kU];
      uint32_t mask = 0;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        // (kTop is four waves: a slice is one for the whole wave)
        const int e = e0 + u * kBins + threadIdx.x;
        const int i = min(__builtin_amdgcn_readfirstlane(e / kTop), r.nslices - 1);
        const bool on = e < r.nslices * kTop && e % kTop < __builtin_amdgcn_readlane(r.listed, i);
        p[u] = on ? r.slices[i].list[e % kTop] : UINT64_MAX;
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float x = value_of(p[u]);
        mask |= (uint32_t)(p[u] != UINT64_MAX && (one.has(x) || two.has(x))) << u;
      }
      uint32_t at = places(__builtin_popcount(mask));
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (mask >> u & 1) {
          if (at < kList) l.list[at] = p[u];
          ++at;
        }
    }
    __syncthreads();
    return;
  }
  // indices first (a lane's candidates are few of its 16), then their values
  auto is = [&](float x) { return (uint32_t)(one.has(x) || two.has(x)); };
  auto keep = [&](uint32_t i0, uint32_t mask) {
    if (__builtin_amdgcn_ballot_w64(mask != 0) == 0) return;
    uint32_t at = places(__builtin_popcount(mask));
    while (mask) {
      const int e = __builtin_ctz(mask);
      mask &= mask - 1;
      if (at < kList) l.list[at] = i0 + 4 * (e / 4) * kBins + e % 4;
      ++at;
    }
  };
  // four loads are always in flight, each sent again for the next stride when it has been
  // looked at; a place behind the end takes the row's start
  const uint32_t fours = (uint32_t)r.n & ~3u, t4 = 4 * threadIdx.x;
  if (fours > 0) {
    f32x4 y[4];
    auto load = [&](uint32_t i) {
      return *reinterpret_cast<const f32x4_u *>(r.x + (i < fours ? i : 0));
    };
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = load(t4 + 4 * u * kBins);
    for (uint32_t i0 = 0; i0 < fours; i0 += 16 * kBins) {
      uint32_t mask = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t i = i0 + t4 + 4 * u * kBins;
        uint32_t four = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) four |= is(y[u][e]) << (4 * u + e);
        mask |= i < fours ? four : 0;
        y[u] = load(i + 16 * kBins);
      }
      keep(i0 + t4, mask);
    }
  }
  const uint32_t i = fours + threadIdx.x;
  keep(i, i < (uint32_t)r.n ? is(r.x[i]) : 0);
  __syncthreads();
  const uint32_t n = min(l.n, (uint32_t)kList);
  for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 4 * kBins) {
    int j[4];
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) j[u] = i0 + u * kBins < n ? (int)l.list[i0 + u * kBins] : 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = r.x[j[u]];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * kBins < n) l.list[i0 + u * kBins] = place(v[u], j[u]);
  }
  __syncthreads();
}

// The members of a bin: visit(place) for each, from LDS where all that was gathered fits,
// else from the row.
template <class F>
__device__ __forceinline__ void members(const RowAt &r, const Values &bin, const SelectLds &l, F visit) {
  if (l.n <= kList) {
    for (uint32_t i = threadIdx.x; i < l.n; i += kBins)
      if (bin.has(value_of(l.list[i]))) visit(l.list[i]);
    return;
  }
  for (int64_t i = threadIdx.x; i < r.n; i += kBins) {
    const float z = r.x[i];
    if (bin.has(z)) visit(place(z, (int)i));
  }
}

// What a border asks for: the number `want`, or the weights' sum `rel`, reached or passed.
struct Border {
  bool by_count, passed;
  uint64_t want;
  double rel;
  __device__ __forceinline__ bool operator()(uint64_t mass, uint32_t count) const {
    return by_count ? count >= want : passed ? (double)mass > rel : (double)mass >= rel;
  }
};

// The first member of the bin, in the order, up to which the members satisfy `reached`;
// the last one where none does.  *upto: the sum of weights up to it, itself included.
// Each step narrows the places to one of kBins parts; few members of LDS are compared
// with each other.
__device__ __forceinline__ uint64_t select(const RowAt &r, const Values &bin, SelectLds &l, const Border &reached,
                                           uint64_t *upto) {
  const int t = threadIdx.x;
  // (an upper bound of the members left; where others were gathered too, or all do
  // not fit, it is not known)
  uint64_t lo = place(bin.hi, 0), hi = place(bin.lo, -1), mass0 = 0;
  uint32_t count0 = 0, left = l.n;
  __syncthreads();
  while (lo < hi) {
    if (l.n <= kList && left <= kCompared) {
      // a thread a member, against all: places and weights in l.mass
      __syncthreads();
      if (t == 0) l.where = 0;
      __syncthreads();
      members(r, bin, l, [&](uint64_t p) {
        if (p < lo || p > hi) return;
        const uint32_t i = atomicAdd(&l.where, 1u);
        l.mass[2 * i] = p;
        l.mass[2 * i + 1] = weight(bin_of(value_of(p), r.inv_t));
      });
      __syncthreads();
      left = l.where;
      bool is = false;
      uint64_t p = 0, m = mass0;
      if (t < (int)left) {
        p = l.mass[2 * t];
        const uint64_t w = l.mass[2 * t + 1];
        uint32_t c = count0;
#pragma unroll 8
        for (uint32_t j = 0; j < left; ++j) {
          const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&l.mass[2 * j]);
          const bool first = o.x < p;
          m += first ? o.y : 0;
          c += first;
        }
        is = reached(m + w, c + 1) && !reached(m, c);
        if (c - count0 == left - 1) {                 // the last one, unless another is it
          l.found = p;
          l.before = m;
        }
      }
      __syncthreads();
      if (is) {
        l.found = p;
        l.before = m;
      }
      __syncthreads();
      lo = hi = l.found;
      mass0 = l.before;
      break;
    }
    const int bits = 64 - __builtin_clzll(hi - lo);   // places lo .. lo + 2^bits - 1
    const int sh = bits > 10 ? bits - 10 : 0;
    l.mass[t] = 0;
    l.count[t] = 0;
    if (t == 0) l.where = 0;
    __syncthreads();
    members(r, bin, l, [&](uint64_t p) {
      if (p < lo || p > hi) return;
      const uint32_t s = (uint32_t)((p - lo) >> sh);
      atomicAdd(reinterpret_cast<unsigned long long *>(&l.mass[s]),
                (unsigned long long)weight(bin_of(value_of(p), r.inv_t)));
      atomicAdd(&l.count[s], 1u);
    });
    __syncthreads();
    const uint64_t m = l.mass[t];
    const uint32_t c = l.count[t];
    uint64_t every;
    uint32_t number;
    const uint64_t mi = mass0 + block_sums<kBins>(m, l.wsum64, &every);
    const uint32_t ci = count0 + block_sums<kBins>(c, l.wsum32, &number);
    const bool on = c > 0 && reached(mi, ci);
    const bool on_before = c > 0 && reached(mi - m, ci - c);
    // the first part that reaches it; the last one that holds anything otherwise
    const bool any = __syncthreads_or(on);
    if (any ? on && !on_before : c > 0) atomicMax(&l.where, (uint32_t)t);
    __syncthreads();
    const uint32_t at = l.where;
    if ((uint32_t)t == at) {
      l.found = mi - m;
      l.before = (uint64_t)(ci - c);
    }
    __syncthreads();
    mass0 = l.found;
    count0 = (uint32_t)l.before;
    left = l.count[at];
    const uint64_t nlo = lo + ((uint64_t)at << sh);
    hi = min(hi, nlo + (((uint64_t)1 << sh) - 1));
    lo = nlo;
    __syncthreads();
    if (sh > 0 && left == 1) {                        // one member: find it
      members(r, bin, l, [&](uint64_t p) {
        if (p >= lo && p <= hi) l.found = p;
      });
      __syncthreads();
      lo = hi = l.found;
      __syncthreads();
    }
  }
  *upto = mass0 + weight(bin_of(value_of(lo), r.inv_t));
  return lo;
}

// The n values of `list`, one a thread, in ascending order, UINT64_MAX behind them.  Few
// are placed by their rank among all (60 of them 0.5 us, 3 by exchanges); of more, lanes
// of a wave exchange in registers, waves through `via`.
__device__ __forceinline__ uint64_t sorted(const uint64_t *list, uint32_t n, uint64_t *via) {
  const int t = threadIdx.x;
  uint64_t v = (uint32_t)t < n ? list[t] : UINT64_MAX;
  if (n <= kBins / 4) {
    if ((uint32_t)t < n) {
      uint32_t at = 0;
#pragma unroll 8
      for (uint32_t i = 0; i < n; ++i) at += list[i] < v;              // (places are not equal)
      via[at] = v;
    }
    __syncthreads();
    return (uint32_t)t < n ? via[t] : UINT64_MAX;
  }
  const uint32_t wave = __builtin_amdgcn_readfirstlane(t & ~63);
  for (uint32_t k = 2; k < 2 * n; k *= 2) {           // (places are not equal; pads are)
    for (uint32_t j = k / 2; j > 0; j /= 2) {
      uint64_t o;
      if (wave >= 2 * n) {                            // (pads alone)
        if (j >= 64) {
          __syncthreads();
          __syncthreads();
        }
        continue;
      }
      if (j < 64) {
        o = __shfl_xor(v, (int)j);
      } else {
        __syncthreads();
        via[t] = v;
        __syncthreads();
        o = via[t ^ j];
      }
      const bool up = (t & k) == 0, low = (t & j) == 0;
      v = up == low ? min(v, o) : max(v, o);
    }
  }
  __syncthreads();
  return v;
}

__global__ __launch_bounds__(kBins) void sample_draw_kernel(SampleArgs a, int64_t row0, int slices) {
  __shared__ SelectLds l;
  const int t = threadIdx.x, lane = t & 63;
  const int64_t row = row0 + blockIdx.x;
  const SampleSlice *sl = reinterpret_cast<const SampleSlice *>(a.ws) + (int64_t)blockIdx.x * slices;
  static_assert(kMaxSlices <= 64, "a slice a lane");
  const SampleSlice &mine = sl[min(lane, slices - 1)];
  const RowSettings s = uniform(settings(a, row));    // (vector registers are short)
  const RowAt r = {a.x + row * a.ldx, a.n, s.inv_t, sl, slices, mine.top, mine.max, mine.upto, mine.listed};
  int index = mine.index;
  const float top = wave_max(r.max);                  // the row's maximum
  const uint64_t tops = __builtin_amdgcn_ballot_w64(r.max == top);
  const double top_bin = uniform(__shfl(r.top, __builtin_ctzll(tops)));
  if (top == -INFINITY || s.greedy) {                 // (the whole block)
    if (r.max != top) index = INT32_MAX;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) index = min(index, __shfl_xor(index, d));
    if (t == 0) {
      a.ids[row] = top == -INFINITY ? -1 : index;
      if (a.logp) a.logp[row] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    return;
  }
  const bool counts = s.k < a.n;
  // this thread's bin, t below the maximum's
  uint64_t m = 0;
  uint32_t c = 0;
  const int down = r.max == -INFINITY ? kBins : below(top_bin, r.top);
  for (int i0 = 0; i0 < slices; i0 += 8) {
    uint64_t mi[8];
    uint32_t ci[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u, slices - 1), shift = __builtin_amdgcn_readlane(down, i);
      const bool on = i0 + u < slices && t >= shift;
      mi[u] = on ? sl[i].mass[t - shift] : 0;
      ci[u] = on && counts ? sl[i].count[t - shift] : 0;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      m += mi[u];
      c += ci[u];
    }
  }
  // (without a count: about as many, weights are within 1 / 32 of 2^40)
  if (!counts) c = (uint32_t)((m + ((uint64_t)1 << 39)) >> 40);
  const double ymax = uniform(bin_of(top, s.inv_t).y);
  // (y of the maximum from its bin's middle on, exact)
  const double rest = uniform(__builtin_isinf(ymax) ? 0.0 : ymax - top_bin / kBinsPerUnit);
  const double unit = exp(-(double)t / kBinsPerUnit - rest) * 0x1p-40;  // weight of 1 in this bin
  const double here = (double)m * unit;
  double mass_all;
  uint32_t count_all;
  const double upto = block_sums<kBins>(here, l.wsumd[0], &mass_all);     // this bin included
  const uint32_t cupto = block_sums<kBins>(c, l.wsum32, &count_all);
  const double total = uniform(mass_all);
  const uint32_t tokens = uniform(count_all);
  // the bin that a border falls into: the first one that reaches it; the last one with
  // tokens where rounding leaves none.  (Two places in turn: a barrier lies between two
  // uses of the same.)
  const uint64_t some = __builtin_amdgcn_ballot_w64(m > 0);
  int turn = 0;
  auto border = [&](bool on) {
    const uint64_t who = __builtin_amdgcn_ballot_w64(m > 0 && on);
    const int first = who ? __builtin_ctzll(who) : -1, final = some ? 63 - __builtin_clzll(some) : -1;
    BorderBin *to = l.border[turn][0] + (t >> 6);
    if (lane == 0) to[0].bin = to[kBins / 64].bin = -1;
#pragma unroll
    for (int z = 0; z < 2; ++z)
      if (lane == (z ? final : first)) {
        BorderBin &o = to[z * (kBins / 64)];
        o.mass = m;
        o.before = upto - here;
        o.unit = unit;
        o.count = c;
        o.upto = cupto;
        o.bin = t;
      }
    __syncthreads();
    // lane z: wave z's first, wave z - 16's last
    const int has = lane < 2 * (kBins / 64) && l.border[turn][0][lane & 31].bin >= 0;
    const uint64_t w = __builtin_amdgcn_ballot_w64(has);
    const int at = (w & 0xffff) ? __builtin_ctzll(w) : 63 - __builtin_clzll(w);
    const BorderBin f = uniform(l.border[turn][0][at]);
    turn ^= 1;
    return f;
  };
  auto bin_at = [&](int b) { return uniform(b == 0 ? top_bin : top_bin - (double)b); };
  const bool by_k = counts && s.k < (int64_t)tokens;
  // the last bin of min_p: weights from min_p on
  int last = kBins - 1;
  if (s.min_p > 0.0 && !__builtin_isinf(ymax))
    last = min(last, below(top_bin, __builtin_rint((ymax + log(s.min_p)) * kBinsPerUnit)));

  // Few kept tokens: gathered and sorted.  Many: the bin of the k-th token, of top_p, of
  // min_p and of the draw in turn, each where its setting is on.
  enum { FEW, BY_K, BY_MASS, BY_WEIGHT, DRAW };
  int b = last;
  // (top_p goes by the sum of all k)
  if (by_k || s.top_p < 1.0) {
    const double least = fmax(s.top_p, 0.0) * total * (1.0 - kTie);
    const int at = border(by_k ? (int64_t)cupto >= s.k : upto >= least).bin;
    b = by_k ? at : min(b, at);
  }
  // a bin's running sums
  __shared__ double e_upto, e_few;
  __shared__ uint32_t e_count;
  if (t == b) {
    e_count = cupto;
    e_few = upto;
  }
  if (t == last) e_upto = upto;
  __syncthreads();
  double W = total;
  double have = NAN, also = NAN;                      // the bins in LDS
  Values values1, values2;
  // (estimates of counts are within 1 / 32)
  for (int stage = e_count <= kBins * 15 / 16 ? FEW : BY_K; stage <= DRAW; ++stage) {
    if ((stage == BY_K && !by_k) || (stage == BY_MASS && !(s.top_p < 1.0)) ||
        (stage == BY_WEIGHT && !(s.min_p > 0.0 && last < kBins - 1)))
      continue;
    double more = NAN;
    const double want = uniform(stage == BY_MASS ? fmax(s.top_p, 0.0) * W * (1.0 - kTie) : s.u * W * (1.0 + kTie));
    BorderBin f = {};
    if (stage != FEW)
      f = border(stage == BY_K        ? (int64_t)cupto >= s.k
                 : stage == BY_MASS   ? upto >= want
                 : stage == BY_WEIGHT ? t == last
                                      : upto > want);
    if (stage == BY_MASS) {
      // with it the bin that the draw falls into, by what is kept at least, where
      // both fit into LDS
      const BorderBin draw = border(upto > s.u * f.before * (1.0 + kTie));
      const uint64_t both = f.mass + (draw.bin == f.bin ? 0 : draw.mass);
      if ((both >> 40) + (both >> 45) < kList) more = bin_at(draw.bin);
    }
    if (stage == BY_WEIGHT && f.bin != last) {        // (no token there)
      if (e_upto > 0.0) W = uniform(fmin(W, e_upto));
      continue;
    }
    const double before = f.before, u = f.unit;
    const double bin = bin_at(stage == FEW ? b : f.bin);
    if (stage == FEW || !(bin == have || bin == also)) {
      gather(r, bin, stage == FEW ? INFINITY : bin, stage == FEW || more != more ? bin : more, l, &values1,
             &values2);
      have = stage == FEW ? NAN : bin;
      also = more;
    }
    if (stage == FEW) {
      const uint32_t n = l.n;                         // (1 at least: the maximum)
      if (n > kBins) continue;
      const uint64_t p = sorted(l.list, n, l.mass);
      const bool in = (uint32_t)t < n;
      double y = 0.0, w = 0.0;
      if (in) {
        y = bin_of(value_of(p), s.inv_t).y;
        w = __builtin_isinf(ymax) ? 1.0 : exp(y - ymax);
      }
      double every;
      const double sum = block_sums<kBins>(w, l.wsumd[1], &every);
      double *sums = reinterpret_cast<double *>(l.mass);
      sums[t] = sum;
      __syncthreads();
      // top_p's sum: of the first k, or of all that were gathered and of the bins behind
      // them (the histogram's: off by 2^-39 of what is not here, and by some last bits of
      // the whole where nothing is, which kTie covers)
      const double S = by_k ? sums[min((int64_t)n, s.k) - 1] : sums[n - 1] + (total - e_few);
      const bool keep = in && t < s.k && (t == 0 || ((s.top_p >= 1.0 || sum - w < s.top_p * S * (1.0 - kTie)) &&
                                                     w >= s.min_p));
      const int kept = __syncthreads_count(keep);     // (a head of the order)
      W = sums[kept - 1];
      const int at = min(__syncthreads_count(in && sum <= s.u * W * (1.0 + kTie)), kept - 1);
      if (t == at) {
        a.ids[row] = (int)(uint32_t)p;
        if (a.logp) a.logp[row] = (float)((__builtin_isinf(ymax) ? 0.0 : y - ymax) - log(W));
      }
      return;
    }
    const Values in_bin = bin == have ? values1 : values2;
    if (stage == BY_WEIGHT) {
      if (t == 0) l.found = 0;
      __syncthreads();
      uint64_t part = 0;
      members(r, in_bin, l, [&](uint64_t p) {
        const BinOf q = bin_of(value_of(p), s.inv_t);
        if (exp(q.y - ymax) >= s.min_p) part += weight(q);
      });
      if (part) atomicAdd(reinterpret_cast<unsigned long long *>(&l.found), (unsigned long long)part);
      __syncthreads();
      const double kept = before + (double)l.found * u;
      if (kept > 0.0) W = uniform(fmin(W, kept));
      __syncthreads();
      continue;
    }
    const Border reached = {stage == BY_K, stage == DRAW, (uint64_t)s.k - (f.upto - f.count), (want - before) / u};
    uint64_t J;
    const uint64_t p = select(r, in_bin, l, reached, &J);
    if (stage != DRAW) {
      W = uniform(fmin(W, before + (double)J * u));
    } else if (t == 0) {
      a.ids[row] = (int)(uint32_t)p;
      const double y = bin_of(value_of(p), s.inv_t).y;
      if (a.logp) a.logp[row] = (float)((__builtin_isinf(ymax) ? 0.0 : y - ymax) - log(W));
    }
  }
}

}  // namespace

// Slices of a row: enough blocks for the chip (four of 512 threads a CU), none
// shorter than a chunk (256 rows of 151936 with top-p: 127 us with 1024 blocks, 132 with
// 512, 131 with 2048; 64 rows of 128256 73, 72, 73).
constexpr int64_t kBlocks = 1024;
static int64_t sample_slices(int64_t rows, int64_t n) {
  const int64_t most = std::min<int64_t>(kMaxSlices, (n + kChunk - 1) / kChunk);
  return std::max<int64_t>(1, std::min(most, (kBlocks + rows - 1) / rows));
}

hipError_t launch_sample(const SampleArgs &a, int64_t ws_bytes, hipStream_t st) {
  int64_t slices = sample_slices(a.rows, a.n);
  const int64_t len = ((a.n + slices - 1) / slices + 3) / 4 * 4;
  slices = (a.n + len - 1) / len;
  // (rows are at most 65535 a launch, a grid's y)
  const int64_t most = std::min<int64_t>(65535, ws_bytes / (slices * (int64_t)sizeof(SampleSlice)));
  for (int64_t r = 0; r < a.rows; r += most) {
    const int64_t rows = std::min(most, a.rows - r);
    hipLaunchKernelGGL(sample_hist_kernel, dim3((unsigned)slices, (unsigned)rows), dim3(kHistThreads), 0, st,
                       a, r, len);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_draw_kernel, dim3((unsigned)rows), dim3(kBins), 0, st, a, r, (int)slices);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace q8
