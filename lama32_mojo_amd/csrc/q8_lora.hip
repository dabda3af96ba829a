// q8_lora.hip -- low-rank adapters of many requests at once, beside a projection
// that they share: y[r] = base[r] + s B (A x[r]) with the A, B and s of row r's
// sequence.
//
// Rows are taken by adapter: the sequences' adapters and row counts are summed in
// LDS by every block, so a tile is up to TR rows of one adapter, wherever they lie,
// and an adapter's weights are read once per tile.  Two launches: A x over parts of
// K (`lora_shrink_kernel`), then B times the sum of the parts (`lora_expand_kernel`).
//
// Products run on v_mfma_f32_16x16x32_bf16.  x and A x enter as three bf16 terms
// whose sum is the f32 value, bf16 weights as they are and f32 weights as three
// terms too (the six products above 2^-24 of the largest), so nothing is rounded to
// fewer bits than f32.
// Bound: HBM, by the adapters' weights for token steps and by base and y (and x)
// for prompts.
#include "q8_device.h"
#include "q8_launch.h"
#include "q8_ragged.h"

#include <algorithm>

namespace q8 {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));   // any f32 address

constexpr int kThreads = 256;
constexpr int kRankTiles = 4;                         // 16-rank tiles of a shrink block

// x as three bf16 terms (truncations, exact), eight values.
__device__ __forceinline__ void split3x8(const float (&x)[8], u32x4 (&o)[3]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float t[2][3];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = x[2 * u + e];
      t[e][0] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u);
      const float r = v - t[e][0];
      t[e][1] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) & 0xffff0000u);
      t[e][2] = r - t[e][1];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) o[k][u] = pk_hi16(t[0][k], t[1][k]);
  }
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight weights as terms; c += W x over them, the smallest products first.
template <bool F32> struct Weights8 {
  u32x4 t[F32 ? 3 : 1];
  __device__ __forceinline__ void load(const uint8_t *w, int64_t elem) {
    if constexpr (F32) {
      const float *p = reinterpret_cast<const float *>(w) + elem;
      const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
      const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      split3x8(x, t);
    } else {
      t[0] = *reinterpret_cast<const u32x4 *>(w + 2 * elem);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < (F32 ? 3 : 1); ++k) t[k] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ f32x4 times(const u32x4 (&x)[3], f32x4 c) const {
    if constexpr (F32) {
      c = mfma(t[2], x[0], c);
      c = mfma(t[0], x[2], c);
      c = mfma(t[1], x[1], c);
      c = mfma(t[1], x[0], c);
      c = mfma(t[0], x[1], c);
      return mfma(t[0], x[0], c);
    } else {
      c = mfma(t[0], x[2], c);
      c = mfma(t[0], x[1], c);
      return mfma(t[0], x[0], c);
    }
  }
};

__device__ __forceinline__ int rank8(int rank, int max_rank) {
  return rank > 0 ? (min(rank, max_rank) + 7) & ~7 : 0;
}

// Inclusive sum over the block's threads; *total the whole one.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *wsum, uint32_t *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) wsum[w] = v;
  __syncthreads();
  uint32_t base = 0, all = 0;
#pragma unroll
  for (int x = 0; x < kThreads / 64; ++x) {
    base += x < w ? wsum[x] : 0;
    all += wsum[x];
  }
  __syncthreads();
  *total = all;
  return base + v;
}

// The rows of tile `tile`: their adapter (nadapters: none) and numbers, in LDS.
// False for a tile behind the last one.  Counts are unsigned, so that arrays that
// hold nonsense wrap and every row number stays one of its sequence's, below `rows`.
template <int TR>
__device__ __forceinline__ bool lora_tile(const LoraArgs &a, uint32_t tile, uint32_t *count, uint32_t *wsum,
                                          int *found, int *rows) {
  const int t = threadIdx.x, na = (int)a.nadapters, nseq = (int)a.nseq;
  for (int i = t; i <= na; i += kThreads) count[i] = 0;
  if (t == 0) found[0] = -1;
  __syncthreads();
  auto of = [&](int i, int *first) {
    const int r0 = clamp_i(a.cu[i], 0, a.rows), r1 = clamp_i(a.cu[i + 1], 0, a.rows);
    *first = r0;
    return (uint32_t)max(r1 - r0, 0);
  };
  auto who = [&](int i) {
    const int id = a.id[i];
    return id >= 0 && id < na && a.rank[id] > 0 ? id : na;
  };
  for (int i = t; i < nseq; i += kThreads) {
    int first;
    const uint32_t n = of(i, &first);
    if (n) atomicAdd(&count[who(i)], n);
  }
  __syncthreads();
  // the adapter that holds the tile
  const int per = (na + 1 + kThreads - 1) / kThreads;
  uint32_t mine = 0, all;
  for (int e = 0; e < per; ++e) {
    const int i = t * per + e;
    if (i <= na && !(i == na && a.in_place)) mine += (count[i] + TR - 1) / TR;
  }
  uint32_t at = block_scan(mine, wsum, &all) - mine;
  if (tile >= at && tile - at < mine) {
    for (int e = 0; e < per; ++e) {
      const int i = t * per + e;
      const uint32_t tiles = i <= na ? (count[i] + TR - 1) / TR : 0;
      if (tile - at < tiles) {
        found[0] = i;
        found[1] = (int)(tile - at) * TR;            // the tile's first place among the adapter's rows
        found[2] = (int)min((uint32_t)TR, count[i] - (tile - at) * TR);
        break;
      }
      at += tiles;
    }
  }
  if (t < TR) rows[t] = 0;
  __syncthreads();
  if (found[0] < 0) return false;
  const uint32_t p0 = (uint32_t)found[1];
  uint32_t base = 0;
  for (int i0 = 0; i0 < nseq; i0 += kThreads) {
    const int i = i0 + t;
    int first = 0;
    uint32_t n = 0;
    if (i < nseq && who(i) == found[0]) n = of(i, &first);
    const uint32_t end = base + block_scan(n, wsum, &all), from = end - n;
    if (n)
      for (int k = 0; k < TR; ++k)
        if (p0 + k - from < n) rows[k] = first + (int)(p0 + k - from);
    base += all;
    if (base - p0 >= (uint32_t)TR && base >= p0) break;
  }
  __syncthreads();
  return true;
}

// A tile's record: adapter, number of rows, the rows; behind the records of all
// tiles the parts of A x, [tile][part of K][row][rank].
template <int TR> constexpr int record_ints() { return TR + 4; }
template <int TR> __device__ __forceinline__ int *record_at(const LoraArgs &a, int tile) {
  return reinterpret_cast<int *>(a.ws) + (int64_t)tile * record_ints<TR>();
}
template <int TR>
__device__ __forceinline__ float *part_at(const LoraArgs &a, int tile, int split) {
  return a.ws + (int64_t)a.tiles * record_ints<TR>() +
         ((int64_t)tile * a.splits + split) * TR * a.ranks;
}

// A x of a tile over one part of K: grid (tiles, parts of K, groups of kRankTiles
// rank tiles).  RT = 1: 16 rows, the waves take K steps in turn and meet in LDS; RT =
// 4: 64 rows, 16 a wave.
template <bool F32, int RT>
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraArgs a) {
  constexpr int TR = 16 * RT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ uint32_t wsum[kThreads / 64];
  __shared__ int found[3], rows[TR];
  __shared__ f32x4 meet[RT == 1 ? 3 : 1][kRankTiles][64];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int split = blockIdx.y;
  if (!lora_tile<TR>(a, a.tile0 + blockIdx.x, reinterpret_cast<uint32_t *>(lds), wsum, found, rows)) {
    if (t == 0 && split == 0 && blockIdx.z == 0) record_at<TR>(a, blockIdx.x)[1] = 0;
    return;
  }
  const int ad = found[0], n = found[2];
  if (split == 0 && blockIdx.z == 0) {
    int *rec = record_at<TR>(a, blockIdx.x);
    if (t == 0) {
      rec[0] = ad;
      rec[1] = n;
    }
    if (t < TR) rec[4 + t] = rows[t];
  }
  if (ad == a.nadapters) return;
  const int rp = rank8(a.rank[ad], a.max_rank), ranks = a.parts * rp;
  const int q0 = blockIdx.z * kRankTiles;             // this block's first rank tile
  const int nq = min(kRankTiles, (ranks + 15) / 16 - q0);
  if (nq <= 0) return;
  const int64_t m = a.m;
  const int64_t per = ((m + a.splits - 1) / a.splits + 31) / 32 * 32;
  const int64_t k0 = split * per, k1 = min(k0 + per, m);
  const uint8_t *A = a.A + (int64_t)ad * a.a_stride * (F32 ? 4 : 2);
  const float *x = a.x + (int64_t)rows[(RT == 1 ? 0 : 16 * w) + col] * a.ldx + 8 * g4;
  int64_t wrow[kRankTiles];
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q)
    wrow[q] = (int64_t)min(16 * (q0 + q) + col, ranks - 1) * m + 8 * g4;
  f32x4 acc[kRankTiles];
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q) acc[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (RT == 1 || 16 * w < n) {
    for (int64_t k = k0 + (RT == 1 ? 32 * w : 0); k < k1; k += RT == 1 ? 128 : 32) {
      const bool in = k + 8 * g4 < k1;                // (m is a multiple of 8)
      const int64_t kk = in ? k : -8 * g4;            // (row's start: any valid one)
      const f32x4 xa = *reinterpret_cast<const f32x4_u *>(x + kk);
      const f32x4 xb = *reinterpret_cast<const f32x4_u *>(x + kk + 4);
      float xs[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        xs[e] = in ? xa[e] : 0.0f;
        xs[4 + e] = in ? xb[e] : 0.0f;
      }
      u32x4 xt[3];
      split3x8(xs, xt);
#pragma unroll
      for (int q = 0; q < kRankTiles; ++q) {
        if (q >= nq) continue;
        Weights8<F32> wt;
        wt.load(A, wrow[q] + kk);
        if (!in) wt.zero();
        acc[q] = wt.times(xt, acc[q]);
      }
    }
  }
  if (RT == 1) {
    if (w > 0) {
#pragma unroll
      for (int q = 0; q < kRankTiles; ++q) meet[w - 1][q][lane] = acc[q];
    }
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int z = 0; z < 3; ++z)
#pragma unroll
      for (int q = 0; q < kRankTiles; ++q) acc[q] += meet[z][q][lane];
  }
  // lane: ranks 16 q + 4 g4 .. of row col
  const int row = (RT == 1 ? 0 : 16 * w) + col;
  if (row >= n) return;
  float *out = part_at<TR>(a, blockIdx.x, split) + (int64_t)row * a.ranks + 16 * q0 + 4 * g4;
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q)
    if (q < nq) *reinterpret_cast<f32x4 *>(out + 16 * q) = acc[q];
}

// y = base + B (s A x) of a tile and up to `cols` columns of one of the stacked
// projections: grid (tiles, column blocks).  The block adds the parts of A x and keeps
// them in LDS as three bf16 terms; an MFMA step takes four (term, eight ranks) pairs, so
// ranks of 8 and 16 fill it too.  16 columns at a time, four of a row in a lane.
template <bool F32, int RT>
__global__ __launch_bounds__(kThreads) void lora_expand_kernel(LoraArgs a, int cols) {
  constexpr int TR = 16 * RT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int *rec = record_at<TR>(a, blockIdx.x);
  const int ad = rec[0], n = rec[1];
  if (n <= 0) return;
  // the part and its columns
  int p = 0, b = blockIdx.y, first = 0;
  while (p < a.parts - 1 && b >= (a.width[p] + cols - 1) / cols) {
    b -= (a.width[p] + cols - 1) / cols;
    first += a.width[p++];
  }
  const int c0 = b * cols, c1 = min(c0 + cols, a.width[p]);
  if (ad == a.nadapters) {                            // no adapter: base as it is
    for (int r = 0; r < n; ++r) {
      const int64_t o = (int64_t)rec[4 + r] * a.ldy + first;
      for (int c = c0 + t; c < c1; c += kThreads) a.y[o + c] = a.base[o + c];
    }
    return;
  }
  const int rp = rank8(a.rank[ad], a.max_rank);
  const int ld = rp + 8;                              // bf16 of an LDS row
  uint16_t *xs = reinterpret_cast<uint16_t *>(lds);   // [3][TR][ld]
  const float s = a.scale[ad];
  for (int i = t; i < TR * (rp / 8); i += kThreads) {
    const int r = i / (rp / 8), j = 8 * (i % (rp / 8));
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (r < n) {
      for (int z = 0; z < a.splits; ++z) {
        const float *q = part_at<TR>(a, blockIdx.x, z) + (int64_t)r * a.ranks + p * rp + j;
        const f32x4 u0 = *reinterpret_cast<const f32x4 *>(q), u1 = *reinterpret_cast<const f32x4 *>(q + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += u0[e];
          v[4 + e] += u1[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= s;
    }
    u32x4 o[3];
    split3x8(v, o);
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<u32x4 *>(xs + ((int64_t)k * TR + r) * ld + j) = o[k];
  }
  __syncthreads();
  const uint8_t *B = a.B + (int64_t)ad * a.b_stride * (F32 ? 4 : 2);
  const int chunks = rp / 8;
  const int pairs = (F32 ? 6 : 3) * chunks, steps = (pairs + 3) / 4;
  int64_t yrow[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) yrow[u] = (int64_t)rec[4 + 16 * u + col] * a.ldy + first;
  for (int c = c0 + 16 * w; c < c1; c += 16 * (kThreads / 64)) {
    const int64_t brow = (int64_t)(first + min(c + col, c1 - 1)) * rp;
    const int cc = c + 4 * g4, left = c1 - cc;        // this lane's columns
    f32x4 acc[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (16 * u + col < n) {
        const float *q = a.base + yrow[u] + cc;
        if (left >= 4) acc[u] = *reinterpret_cast<const f32x4_u *>(q);
        else
          for (int e = 0; e < 3; ++e)
            if (e < left) acc[u][e] = q[e];
      }
    }
    f32x4 d[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) d[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int z = 0; z < steps; ++z) {
      // pair: the smallest products first
      const int pair = 4 * z + g4;
      const bool in = pair < pairs;
      const int kind = in ? pair / chunks : 0, j = in ? 8 * (pair % chunks) : 0;
      // terms of x and of the weights: f32 (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
      const int xt = F32 ? (0x021010 >> (4 * (5 - kind))) & 3 : 2 - kind;
      Weights8<F32> wt;
      wt.load(B, brow + j);
      u32x4 wv = wt.t[0];
      if constexpr (F32) {
        const int wk = (0x201100 >> (4 * (5 - kind))) & 3;
        wv = wk == 0 ? wt.t[0] : wk == 1 ? wt.t[1] : wt.t[2];
      }
      if (!in) wv = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        u32x4 xv = *reinterpret_cast<const u32x4 *>(xs + ((int64_t)xt * TR + 16 * u + col) * ld + j);
        if (!in) xv = u32x4{0, 0, 0, 0};
        d[u] = mfma(wv, xv, d[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      if (16 * u + col >= n) continue;
      acc[u] += d[u];
      float *q = a.y + yrow[u] + cc;
      if (left >= 4) *reinterpret_cast<f32x4_u *>(q) = acc[u];
      else
        for (int e = 0; e < 3; ++e)
          if (e < left) q[e] = acc[u][e];
    }
  }
}

template <bool F32, int RT>
hipError_t launch_lora_t(LoraArgs a, int64_t ws_floats, hipStream_t st) {
  constexpr int TR = 16 * RT;
  const int64_t all = a.rows / TR + std::min(std::min(a.nseq, a.nadapters + 1), a.rows);
  a.ranks = (a.parts * a.max_rank + 15) / 16 * 16;
  const int rank_groups = (a.ranks / 16 + kRankTiles - 1) / kRankTiles;
  // parts of K: two blocks a CU, each with four steps of 32 a wave at least; few
  // for large tiles, whose parts are added by every column block
  const int64_t step = RT == 1 ? 512 : 1024;
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + all - 1) / all, (a.m + step - 1) / step));
  if (RT > 1) a.splits = std::min(a.splits, 4);
  const int64_t per = record_ints<TR>() + (int64_t)a.splits * TR * a.ranks;
  const int64_t most = std::min<int64_t>(ws_floats / per, 65535);
  if (most < 1) return hipErrorInvalidValue;
  const int cols = RT == 1 ? 512 : 2048;
  int blocks = 0;
  for (int p = 0; p < a.parts; ++p) blocks += (a.width[p] + cols - 1) / cols;
  const size_t lds0 = (size_t)(a.nadapters + 1) * 4, lds1 = (size_t)3 * TR * (a.max_rank + 8) * 2;
  for (int64_t t0 = 0; t0 < all; t0 += most) {
    a.tile0 = (int)t0;
    a.tiles = (int)std::min(most, all - t0);
    hipLaunchKernelGGL((lora_shrink_kernel<F32, RT>),
                       dim3((unsigned)a.tiles, (unsigned)a.splits, (unsigned)rank_groups), dim3(kThreads), lds0,
                       st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((lora_expand_kernel<F32, RT>), dim3((unsigned)a.tiles, (unsigned)blocks), dim3(kThreads),
                       lds1, st, a, cols);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_lora(const LoraArgs &a, int64_t ws_floats, hipStream_t st) {
  // tiles of 64 rows where an adapter has as many on average
  const int64_t groups = std::min(a.nseq, a.nadapters);
  const bool wide = a.rows >= 64 * std::max<int64_t>(groups, 1) && a.max_rank <= 128;
  if (a.f32) return wide ? launch_lora_t<true, 4>(a, ws_floats, st) : launch_lora_t<true, 1>(a, ws_floats, st);
  return wide ? launch_lora_t<false, 4>(a, ws_floats, st) : launch_lora_t<false, 1>(a, ws_floats, st);
}

}  // namespace q8
