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
// Weights are held relative to their bin's lower edge, in [1, e^(1/16)), as whole
// numbers of 2^-40: integer sums, so the order of the atomics does not matter and
// equal inputs give equal ids; over bins they are summed in f64 in a fixed order.
// Bins reach 64 below the maximum (e^-64 of the largest weight: 2^22 such tokens
// are 2^-70 of the sum, less than a f64 sum can hold).  Sums in f32 would be off
// by 2^-24 of the mass, as much as the step of a f32 u.
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
constexpr int kList = 4096;                           // members of a bin kept in LDS

// A slice's part of its row: sums and counts of the bins below its own maximum.
struct SampleSlice {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  double top;                                         // bin number of the maximum
  float max;                                          // -inf: no token
  int index;                                          // its lowest index
};

// y = x / T and the bin that holds it, as whole numbers in f64 (floor(16 y), exact);
// infinities have a bin of their own.
struct BinOf {
  double y, a;
};
__device__ __forceinline__ BinOf bin_of(float x, double inv_t) {
  BinOf b;
  b.y = (double)x * inv_t;
  if (x == INFINITY) b.y = INFINITY;                  // (T = inf: inf * 0)
  b.a = __builtin_floor(b.y * kBinsPerUnit);
  return b;
}
// Bins below the one of the maximum; kBins: out of reach.
__device__ __forceinline__ int below(double top, double a) {
  const double d = top - a;
  return top == a ? 0 : d < (double)kBins ? (int)d : kBins;
}
// exp(y - edge) 2^40 as a whole number.  The argument is in [0, 1/16): the series
// to the 8th power is below 2^-54 off.  Adding 2^52 leaves the integer in the low
// bits.
__device__ __forceinline__ uint64_t weight(const BinOf &b) {
  const double r = __builtin_isinf(b.y) ? 0.0 : __builtin_fma(b.a, -1.0 / kBinsPerUnit, b.y);
  double p = 1.0 / 40320.0;
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const double w = __builtin_fma(p, 0x1p40, 0x1p52);
  return __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
}

struct RowSettings {
  bool greedy;
  double inv_t;
  int64_t k;
  double top_p, min_p, u;
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
// Bound: HBM (one read of the logits), beside 15 f64 operations and an LDS atomic
// a logit.  A block walks its slice in chunks that it holds in registers; the
// bins are a ring whose head is the slice's largest value so far, so the row's
// maximum need not be known first.
__global__ __launch_bounds__(kHistThreads) void sample_hist_kernel(SampleArgs a, int64_t row0,
                                                                   int64_t slice_len) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ float wmax[kHistThreads / 64];
  __shared__ int best;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.y;
  const float *x = a.x + row * a.ldx;
  SampleSlice *out = reinterpret_cast<SampleSlice *>(a.ws) + (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const RowSettings s = settings(a, row);
  const bool counts = s.k < a.n;
  const int64_t i0 = blockIdx.x * slice_len, i1 = min(i0 + slice_len, a.n);
  for (int b = t; b < kBins; b += kHistThreads) {
    mass[b] = 0;
    count[b] = 0;
  }
  float top = -INFINITY;                              // of the slice so far
  double top_bin = -INFINITY;
  int head = 0, index = INT32_MAX;
  for (int64_t c = i0; c < i1; c += kChunk) {
    float v[kPerThread];
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < kPerThread / 4; ++q) {
      const int64_t i = c + 4 * (q * kHistThreads + t);
      if (i + 4 <= i1) {
        const f32x4 y = *reinterpret_cast<const f32x4_u *>(x + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = y[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = i + e < i1 ? x[i + e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, v[4 * q + e]);          // (NaN: not taken)
    }
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
    if (!s.greedy) {
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        if (!(v[e] > -INFINITY)) continue;
        const BinOf b = bin_of(v[e], s.inv_t);
        const int d = below(top_bin, b.a);
        if (d >= kBins) continue;
        const int at = (head + d) & (kBins - 1);
        atomicAdd(reinterpret_cast<unsigned long long *>(&mass[at]), (unsigned long long)weight(b));
        if (counts) atomicAdd(&count[at], 1u);
      }
    }
    __syncthreads();                                  // wmax, best, the ring's head
  }
  if (t == 0) {
    out->top = top_bin;
    out->max = top;
    out->index = index;
  }
  if (s.greedy) return;
  for (int b = t; b < kBins; b += kHistThreads) {
    const int at = (head + b) & (kBins - 1);
    out->mass[b] = mass[at];
    out->count[b] = count[at];
  }
}

// ---- pass 2: one block of kBins threads per row --------------------------------
// A token's place in the order, ascending: larger values first, then lower indices.
__device__ __forceinline__ uint64_t place(float x, int i) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);           // (-0 as 0)
  const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;         // ascending with x
  return (uint64_t)~key << 32 | (uint32_t)i;
}

// Inclusive sums over the block's threads, in one fixed order.
template <class T> __device__ __forceinline__ T block_sums(T v, T *wsum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) wsum[w] = v;
  __syncthreads();
  T base = 0;
  for (int x = 0; x < w; ++x) base += wsum[x];
  __syncthreads();
  return base + v;
}

struct SelectLds {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t list[kList];                               // places of a bin's members
  uint64_t wsum64[kBins / 64];
  double wsumd[kBins / 64];
  uint32_t wsum32[kBins / 64];
  uint64_t lo, hi, found;
  uint64_t before;                                    // sum before what was found
  double dsum;
  uint32_t n, where;
};

__device__ __forceinline__ float value_of(uint64_t place) {
  const uint32_t key = ~(uint32_t)(place >> 32);
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The row's members of the bin `bin`: visit(place) for each.  From the list where
// they fit, else from the row.
template <class F>
__device__ __forceinline__ void members(const SampleArgs &a, const float *x, double inv_t, double bin,
                                        const SelectLds &l, bool listed, F visit) {
  if (listed) {
    for (uint32_t i = threadIdx.x; i < l.n; i += kBins) visit(l.list[i]);
    return;
  }
  for (int64_t i0 = 0; i0 < a.n; i0 += 4 * kBins) {
    const int64_t i = i0 + 4 * threadIdx.x;
    float v[4];
    if (i + 4 <= a.n) {
      const f32x4 y = *reinterpret_cast<const f32x4_u *>(x + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = y[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < a.n ? x[i + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] > -INFINITY && bin_of(v[e], inv_t).a == bin) visit(place(v[e], (int)(i + e)));
  }
}

// Puts the members of `bin` into the list; whether they fit.
__device__ __forceinline__ bool gather(const SampleArgs &a, const float *x, double inv_t, double bin,
                                       SelectLds &l) {
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  members(a, x, inv_t, bin, l, false, [&](uint64_t p) {
    const uint32_t i = atomicAdd(&l.n, 1u);
    if (i < kList) l.list[i] = p;
  });
  __syncthreads();
  return l.n <= kList;
}

// The first member of the bin, in the order, up to which the sum of weights (or,
// BY_COUNT, the number) satisfies `reached`; the last one where none does.  *upto:
// the sum of weights up to it, itself included.  Each step narrows the places to one
// of kBins parts.
template <bool BY_COUNT, class F>
__device__ __forceinline__ uint64_t select(const SampleArgs &a, const float *x, double inv_t, double bin,
                                           SelectLds &l, bool listed, F reached, uint64_t *upto) {
  const int t = threadIdx.x;
  if (t == 0) {
    l.lo = UINT64_MAX;
    l.hi = 0;
  }
  __syncthreads();
  {
    uint64_t lo = UINT64_MAX, hi = 0;
    members(a, x, inv_t, bin, l, listed, [&](uint64_t p) {
      lo = min(lo, p);
      hi = max(hi, p);
    });
    if (lo <= hi) {
      atomicMin(reinterpret_cast<unsigned long long *>(&l.lo), (unsigned long long)lo);
      atomicMax(reinterpret_cast<unsigned long long *>(&l.hi), (unsigned long long)hi);
    }
  }
  __syncthreads();
  uint64_t lo = l.lo, hi = l.hi, mass0 = 0;
  uint32_t count0 = 0;
  while (lo < hi) {
    const int bits = 64 - __builtin_clzll(hi - lo);   // places lo .. lo + 2^bits - 1
    const int sh = bits > 10 ? bits - 10 : 0;
    l.mass[t] = 0;
    l.count[t] = 0;
    if (t == 0) l.where = 0;
    __syncthreads();
    members(a, x, inv_t, bin, l, listed, [&](uint64_t p) {
      if (p < lo || p > hi) return;
      const uint32_t s = (uint32_t)((p - lo) >> sh);
      atomicAdd(reinterpret_cast<unsigned long long *>(&l.mass[s]),
                (unsigned long long)weight(bin_of(value_of(p), inv_t)));
      atomicAdd(&l.count[s], 1u);
    });
    __syncthreads();
    const uint64_t m = l.mass[t];
    const uint32_t c = l.count[t];
    const uint64_t mi = mass0 + block_sums(m, l.wsum64);
    const uint32_t ci = count0 + block_sums(c, l.wsum32);
    const bool on = c > 0 && reached(BY_COUNT ? (uint64_t)ci : mi);
    const bool on_before = c > 0 && reached(BY_COUNT ? (uint64_t)(ci - c) : mi - m);
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
    const uint64_t nlo = lo + ((uint64_t)at << sh);
    hi = min(hi, nlo + (((uint64_t)1 << sh) - 1));
    lo = nlo;
    if (sh > 0 && l.count[at] == 1) {                 // one member: find it
      __syncthreads();
      members(a, x, inv_t, bin, l, listed, [&](uint64_t p) {
        if (p >= lo && p <= hi) l.found = p;
      });
      __syncthreads();
      lo = hi = l.found;
    }
    __syncthreads();
  }
  *upto = mass0 + weight(bin_of(value_of(lo), inv_t));
  return lo;
}

__global__ __launch_bounds__(kBins) void sample_draw_kernel(SampleArgs a, int64_t row0, int slices) {
  __shared__ SelectLds l;
  const int t = threadIdx.x;
  const int64_t row = row0 + blockIdx.x;
  const float *x = a.x + row * a.ldx;
  const SampleSlice *sl = reinterpret_cast<const SampleSlice *>(a.ws) + (int64_t)blockIdx.x * slices;
  const RowSettings s = settings(a, row);
  // the row's maximum
  float top = -INFINITY;
  double top_bin = -INFINITY;
  int index = INT32_MAX;
  for (int i = 0; i < slices; ++i) {
    if (sl[i].max > top) {
      top = sl[i].max;
      top_bin = sl[i].top;
      index = sl[i].index;
    } else if (sl[i].max == top) {
      index = min(index, sl[i].index);
    }
  }
  if (top == -INFINITY || s.greedy) {                 // (the whole block)
    if (t == 0) {
      a.ids[row] = top == -INFINITY ? -1 : index;
      if (a.logp) a.logp[row] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    return;
  }
  // this thread's bin, t below the maximum's
  uint64_t m = 0;
  uint32_t c = 0;
  for (int i = 0; i < slices; ++i) {
    if (sl[i].max == -INFINITY) continue;
    const int shift = below(top_bin, sl[i].top);
    if (t >= shift) {
      m += sl[i].mass[t - shift];
      c += sl[i].count[t - shift];
    }
  }
  const double ymax = bin_of(top, s.inv_t).y;
  const double rest = __builtin_isinf(ymax) ? 0.0 : ymax - top_bin / kBinsPerUnit;    // exact
  const double unit = exp(-(double)t / kBinsPerUnit - rest) * 0x1p-40;  // weight of 1 in this bin
  const double mine = (double)m * unit;
  const double upto = block_sums(mine, l.wsumd);      // this bin included
  const uint32_t cupto = block_sums(c, l.wsum32);
  // the bin that a border falls into: the first one that reaches it, `upto` and
  // `unit` of which go around; the last one with tokens where rounding leaves none
  __shared__ double e_before, e_unit;
  auto border = [&](bool on) {
    const bool any = __syncthreads_or(on && m > 0);
    if (t == 0) l.where = any ? kBins : 0;
    __syncthreads();
    if (m > 0) {
      if (any) {
        if (on) atomicMin(&l.where, (uint32_t)t);
      } else {
        atomicMax(&l.where, (uint32_t)t);
      }
    }
    __syncthreads();
    const int b = (int)l.where;
    if (t == b) {
      e_before = upto - mine;
      e_unit = unit;
    }
    __syncthreads();
    return b;
  };
  auto bin_at = [&](int b) { return b == 0 ? top_bin : top_bin - (double)b; };

  if (t == kBins - 1) {
    l.dsum = upto;
    l.found = cupto;
  }
  __syncthreads();
  double W = l.dsum;
  const uint32_t tokens = (uint32_t)l.found;
  __syncthreads();
  int have = -1;                                      // the bin in the list
  bool listed = false;
  auto look = [&](int b) {
    if (have != b) listed = gather(a, x, s.inv_t, bin_at(b), l);
    have = b;
  };
  uint64_t J;
  if (s.k < (int64_t)tokens) {
    const int b = border((int64_t)cupto >= s.k);
    if (t == b) l.before = cupto - c;
    __syncthreads();
    const uint64_t want = (uint64_t)s.k - l.before;
    const double before = e_before, u = e_unit;
    look(b);
    select<true>(a, x, s.inv_t, bin_at(b), l, listed, [&](uint64_t n) { return n >= want; }, &J);
    W = before + (double)J * u;
  }
  if (s.top_p < 1.0) {
    const double want = fmax(s.top_p, 0.0) * W;
    const int b = border(upto >= want);
    const double before = e_before, u = e_unit, rel = (want - before) / u;
    look(b);
    select<false>(a, x, s.inv_t, bin_at(b), l, listed, [&](uint64_t n) { return (double)n >= rel; }, &J);
    W = fmin(W, before + (double)J * u);
  }
  if (s.min_p > 0.0) {
    // tokens of weight min_p and more: whole bins above the border's
    const double z = log(s.min_p);                    // y - ymax from which on
    const double edge = __builtin_isinf(ymax) ? top_bin : __builtin_floor((ymax + z) * kBinsPerUnit);
    const int d = below(top_bin, edge);
    if (d < kBins) {
      if (t == d) {
        e_before = upto - mine;
        e_unit = unit;
        l.dsum = (double)m;
      }
      __syncthreads();
      const double before = e_before, u = e_unit;
      if (l.dsum > 0.0) look(d);
      __syncthreads();
      if (t == 0) l.found = 0;
      __syncthreads();
      if (l.dsum > 0.0) {
        uint64_t part = 0;
        members(a, x, s.inv_t, bin_at(d), l, listed, [&](uint64_t p) {
          const BinOf q = bin_of(value_of(p), s.inv_t);
          if (__builtin_isinf(ymax) || exp(q.y - ymax) >= s.min_p) part += weight(q);
        });
        if (part) atomicAdd(reinterpret_cast<unsigned long long *>(&l.found), (unsigned long long)part);
      }
      __syncthreads();
      const double kept = before + (double)l.found * u;
      if (kept > 0.0) W = fmin(W, kept);
      __syncthreads();
    }
  }
  const double want = s.u * W;
  const int b = border(upto > want);
  const double before = e_before, u = e_unit, rel = (want - before) / u;
  look(b);
  const uint64_t p = select<false>(a, x, s.inv_t, bin_at(b), l, listed,
                                   [&](uint64_t n) { return (double)n > rel; }, &J);
  if (t == 0) {
    a.ids[row] = (int)(uint32_t)p;
    const double y = bin_of(value_of(p), s.inv_t).y;
    if (a.logp) a.logp[row] = (float)((__builtin_isinf(ymax) ? 0.0 : y - ymax) - log(W));
  }
}

}  // namespace

// Slices of a row: enough blocks for the chip (two of 512 threads a CU), none
// shorter than a chunk.
static int64_t sample_slices(int64_t rows, int64_t n) {
  const int64_t most = (n + kChunk - 1) / kChunk;
  return std::max<int64_t>(1, std::min(most, (512 + rows - 1) / rows));
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
