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
#include <type_traits>

namespace q8 {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));   // any f32 address

constexpr int kThreads = 256;
// Columns of a block, 64-row tiles (4130 rows x 28672 columns 261 us, 512 262, 128 284; 512
// rows x 14336 columns 23.6, 512 25.9, 128 26.1).
constexpr int kCols = 256;
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

// Eight weights as loaded, and their terms; times(): c += W x, the smallest products
// first.
template <bool F32> struct Weights8 {
  u32x4 raw[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t *w, int64_t elem) {
    const u32x4 *p = reinterpret_cast<const u32x4 *>(w + (F32 ? 4 : 2) * elem);
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) raw[i] = p[i];
  }
  __device__ __forceinline__ void terms(bool in, u32x4 (&t)[F32 ? 3 : 1]) const {
    if constexpr (F32) {
      const f32x4 a = __builtin_bit_cast(f32x4, raw[0]), b = __builtin_bit_cast(f32x4, raw[1]);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = !in ? 0.0f : e < 4 ? a[e] : b[e - 4];
      split3x8(x, t);
    } else {
      t[0] = in ? raw[0] : u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ f32x4 times(bool in, const u32x4 (&x)[3], f32x4 c) const {
    u32x4 t[F32 ? 3 : 1];
    terms(in, t);
    if constexpr (F32) {
      c = mfma(t[2], x[0], c);
      c = mfma(t[0], x[2], c);
      c = mfma(t[1], x[1], c);
      c = mfma(t[1], x[0], c);
      c = mfma(t[0], x[1], c);
    } else {
      c = mfma(t[0], x[2], c);
      c = mfma(t[0], x[1], c);
    }
    return mfma(t[0], x[0], c);
  }
};

__device__ __forceinline__ int rank8(int rank, int max_rank) {
  return rank > 0 ? (min(rank, max_rank) + 7) & ~7 : 0;
}

// Inclusive sum over the block's threads; *total the whole one.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *wsum, uint32_t *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = wave_scan(v, [](uint32_t a, uint32_t b) { return a + b; });
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
    return id >= 0 && id < na ? id : na;
  };
  const int rank0 = t < na ? a.rank[t] : 0;           // (in flight beside the search)
  // (this thread's first sequence stays in registers)
  int first0 = 0, who0 = -1;
  uint32_t n0 = 0;
  if (t < nseq) {
    who0 = who(t);
    n0 = of(t, &first0);
  }
  for (int i = t; i < nseq; i += kThreads) {
    int first = first0;
    const uint32_t n = i == t ? n0 : of(i, &first);
    if (n) atomicAdd(&count[i == t ? who0 : who(i)], n);
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
  if (t == found[0]) found[3] = rank0;
  else if (t == 0 && found[0] >= kThreads && found[0] < na) found[3] = a.rank[found[0]];
  const uint32_t p0 = (uint32_t)found[1];
  uint32_t base = 0;
  for (int i0 = 0; i0 < nseq; i0 += kThreads) {
    const int i = i0 + t;
    int first = 0;
    uint32_t n = 0;
    if (i0 == 0) {
      first = first0;
      n = who0 == found[0] ? n0 : 0;
    } else if (i < nseq && who(i) == found[0]) {
      n = of(i, &first);
    }
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

// A tile's record: adapter, number of rows, rank, the rows; behind the records of all
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

// A x of 16 rows of a tile over one part of K: grid (tiles, parts of K, groups of
// kRankTiles rank tiles x the tile's 16-row parts).  The waves take K steps in turn and
// meet in LDS.  (A wave to each 16 rows of 64 and all of its part of K took 51 us where
// this takes 45: five adapters of rank 16 to 64 over 4130 rows of 4096, two projections.)
// Bound: for prompts the matrix work and the weights' way through L1, 6 KB a wave and
// step for 12 MFMAs; for token steps the chain cu -> adapter -> weights -> meeting (64
// requests over 24 adapters 12 us, 1 request 5).
template <bool F32, int RT>
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraArgs a) {
  constexpr int TR = 16 * RT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ uint32_t wsum[kThreads / 64];
  __shared__ int found[4], rows[TR];
  __shared__ f32x4 meet[kThreads / 64 - 1][kRankTiles][64];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int split = blockIdx.y, row0 = 16 * (blockIdx.z % RT);
  if (!lora_tile<TR>(a, a.tile0 + blockIdx.x, reinterpret_cast<uint32_t *>(lds), wsum, found, rows)) {
    if (t == 0 && split == 0 && blockIdx.z == 0) record_at<TR>(a, blockIdx.x)[1] = 0;
    return;
  }
  const int ad = found[0], n = found[2], rank = ad < a.nadapters ? found[3] : 0;
  if (split == 0 && blockIdx.z == 0) {
    int *rec = record_at<TR>(a, blockIdx.x);
    if (t == 0) {
      rec[0] = ad;
      rec[1] = n;
      rec[2] = rank;
    }
    if (t < TR) rec[4 + t] = rows[t];
  }
  if (rank <= 0) return;
  const int rp = rank8(rank, a.max_rank), ranks = a.parts * rp;
  const int q0 = blockIdx.z / RT * kRankTiles;        // this block's first rank tile
  const int nq = min(kRankTiles, (ranks + 15) / 16 - q0);
  if (nq <= 0 || row0 >= n) return;
  const int64_t m = a.m;
  const int64_t per = ((m + a.splits - 1) / a.splits + 31) / 32 * 32;
  const int64_t k0 = split * per, k1 = min(k0 + per, m);
  const uint8_t *A = a.A + (int64_t)ad * a.a_stride * (F32 ? 4 : 2);
  const float *x = a.x + (int64_t)rows[row0 + col] * a.ldx + 8 * g4;
  int64_t wrow[kRankTiles];
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q)
    wrow[q] = (int64_t)min(16 * (q0 + q) + col, ranks - 1) * m + 8 * g4;
  f32x4 acc[kRankTiles];
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q) acc[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // U steps of 32 at a time, all their loads first; the last ones with a test for each
  // lane's eight (m is a multiple of 8; those behind k1 load the row's start)
  constexpr int U = F32 ? 1 : 4, STEP = 32 * (kThreads / 64);
  auto steps = [&](int64_t k, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    f32x4 xa[U], xb[U];
    Weights8<F32> wt[U][kRankTiles];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t ku = k + u * STEP;
      in[u] = WHOLE || ku + 8 * g4 < k1;
      const int64_t kk = in[u] ? ku : -8 * g4;
      xa[u] = *reinterpret_cast<const f32x4_u *>(x + kk);
      xb[u] = *reinterpret_cast<const f32x4_u *>(x + kk + 4);
#pragma unroll
      for (int q = 0; q < kRankTiles; ++q)
        if (q < nq) wt[u][q].load(A, wrow[q] + kk);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float xs[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        xs[e] = in[u] ? xa[u][e] : 0.0f;
        xs[4 + e] = in[u] ? xb[u][e] : 0.0f;
      }
      u32x4 xt[3];
      split3x8(xs, xt);
#pragma unroll
      for (int q = 0; q < kRankTiles; ++q)
        if (q < nq) acc[q] = wt[u][q].times(in[u], xt, acc[q]);
    }
  };
  int64_t k = k0 + 32 * w;
  for (; k + (U - 1) * STEP + 32 <= k1; k += U * STEP) steps(k, std::true_type{});
  if (k < k1) steps(k, std::false_type{});
  if (w > 0) {
#pragma unroll
    for (int q = 0; q < kRankTiles; ++q) meet[w - 1][q][lane] = acc[q];
  }
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int z = 0; z < kThreads / 64 - 1; ++z)
#pragma unroll
    for (int q = 0; q < kRankTiles; ++q) acc[q] += meet[z][q][lane];
  // lane: ranks 16 q + 4 g4 .. of row col
  const int row = row0 + col;
  if (row >= n) return;
  float *out = part_at<TR>(a, blockIdx.x, split) + (int64_t)row * a.ranks + 16 * q0 + 4 * g4;
#pragma unroll
  for (int q = 0; q < kRankTiles; ++q)
    if (q < nq) *reinterpret_cast<f32x4 *>(out + 16 * q) = acc[q];
}

// y = base + B (s A x) of a tile and up to `cols` columns of one of the stacked
// projections: grid (tiles, column blocks).  The block adds the parts of A x and keeps
// them in LDS as three bf16 terms.  A lane loads the weights of eight ranks of a column
// once for all products of terms; ranks of 8 and 16 leave room in an MFMA step (32
// ranks), which then takes four or two products.  A wave takes 32 columns at a time;
// base and the first weights are loaded ahead of the LDS work.  The accumulators hold
// 16 rows x 64 B; they are turned in LDS to 8 rows x 128 B, whole lines (4126 rows x 28672
// columns read and written 233 -> 195 us by that alone).
// Rows lie a multiple of 4 KB apart, as a rule, which is one channel of the L2 for all
// of them: blocks begin at different columns, so that they do not go from channel to
// channel together.
template <bool F32, int RT>
__global__ __launch_bounds__(kThreads, 3) void lora_expand_kernel(LoraArgs a, int cols) {
  constexpr int TR = 16 * RT, CT = 2, WC = 16 * CT, BC = WC * (kThreads / 64);
  constexpr int KINDS = F32 ? 6 : 3;                  // products of terms
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ __attribute__((aligned(16))) float turn[kThreads / 64][16][WC + 4];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int col = lane & 15, g4 = lane >> 4;
  const int *rec = record_at<TR>(a, blockIdx.x);
  const int ad = rec[0], n = rec[1], rp = rank8(rec[2], a.max_rank);
  if (n <= 0 || (rp == 0 && a.in_place)) return;
  // the part and its columns
  int p = 0, b = blockIdx.y, first = 0;
  while (p < a.parts - 1 && b >= (a.width[p] + cols - 1) / cols) {
    b -= (a.width[p] + cols - 1) / cols;
    first += a.width[p++];
  }
  const int c0 = b * cols, c1 = min(c0 + cols, a.width[p]);
  if (rp == 0) {                                      // no adapter: base as it is
    const int q = (c1 - c0 + 3) / 4, all = n * q;
    for (int i0 = t; i0 < all; i0 += 4 * kThreads) {
      f32x4 v[4];
      int64_t o[4];
      int left[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * kThreads, all - 1), r = i / q, c = c0 + 4 * (i - r * q);
        left[u] = i0 + u * kThreads < all ? c1 - c : 0;
        o[u] = (int64_t)rec[4 + r] * a.ldy + first + c;
        if (left[u] >= 4) v[u] = *reinterpret_cast<const f32x4_u *>(a.base + o[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (left[u] >= 4) *reinterpret_cast<f32x4_u *>(a.y + o[u]) = v[u];
        else
          for (int e = 0; e < left[u]; ++e) a.y[o[u] + e] = a.base[o[u] + e];
      }
    }
    return;
  }
  const int ld = rp + 8;                              // bf16 of an LDS row
  uint16_t *xs = reinterpret_cast<uint16_t *>(lds);   // [3][TR][ld]
  const uint8_t *B = a.B + (int64_t)ad * a.b_stride * (F32 ? 4 : 2);
  // eights of ranks, groups of four of them (a lane's: 4 q + g4 % side), products a step
  const int chunks = rp / 8, groups = (chunks + 3) / 4;
  const int shift = chunks > 2 ? 2 : chunks - 1, side = 1 << shift;    // 1, 2 or 4
  const int steps = ((KINDS << shift) + 3) / 4;
  // this lane's rows, 8 h + lane / 8 of each 16, and columns 4 (lane % 8) .. of each 32
  const int rl = lane >> 3, cl = 4 * (lane & 7);
  int yrow[RT][2];
#pragma unroll
  for (int u = 0; u < RT; ++u)
#pragma unroll
    for (int h = 0; h < 2; ++h) yrow[u][h] = rec[4 + 16 * u + 8 * h + rl];
  auto row_at = [&](int u, int h) { return (int64_t)yrow[u][h] * a.ldy + first; };

  f32x4 base[RT][2];
  Weights8<F32> wt[CT];
  auto load_weights = [&](int c, int q) {
    const int j = 8 * min(4 * q + (g4 & (side - 1)), chunks - 1);
#pragma unroll
    for (int v = 0; v < CT; ++v) wt[v].load(B, (int64_t)(first + min(c + 16 * v + col, c1 - 1)) * rp + j);
  };
  auto load = [&](int c) {
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = c1 - c - cl;
        base[u][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (16 * u + 8 * h + rl < n) {
          const float *q = a.base + row_at(u, h) + c + cl;
          if (left >= 4) base[u][h] = *reinterpret_cast<const f32x4_u *>(q);
          else
            for (int e = 0; e < 3; ++e)
              if (e < left) base[u][h][e] = q[e];
        }
      }
    load_weights(c, 0);
  };
  const int its = (c1 - c0 + BC - 1) / BC;
  int it = (int)((blockIdx.x + blockIdx.y) % (unsigned)its);
  auto column = [&](int i) { return c0 + BC * i + WC * w; };
  load(column(it));

  const float s = a.scale[ad];
  for (int i = t; i < TR * chunks; i += kThreads) {
    const int r = i / chunks, j = 8 * (i - r * chunks);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (r < n) {
      const float *q = part_at<TR>(a, blockIdx.x, 0) + (int64_t)r * a.ranks + p * rp + j;
      const int64_t next = (int64_t)TR * a.ranks;
      for (int z0 = 0; z0 < a.splits; z0 += 4) {
        f32x4 u[4][2];
#pragma unroll
        for (int z = 0; z < 4; ++z)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            u[z][h] = *reinterpret_cast<const f32x4 *>(q + min(z0 + z, a.splits - 1) * next + 4 * h);
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (z0 + z < a.splits) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += u[z][e / 4][e % 4];
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

  for (int done = 0; done < its; ++done) {
    const int c = column(it);
    f32x4 d[RT][CT];
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int v = 0; v < CT; ++v) d[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int q = 0; q < groups; ++q) {
      const int chunk = 4 * q + (g4 & (side - 1));
      u32x4 tm[CT][F32 ? 3 : 1];
#pragma unroll
      for (int v = 0; v < CT; ++v) wt[v].terms(chunk < chunks, tm[v]);
      if (q + 1 < groups) load_weights(c, q + 1);
      // terms of x and of the weights, the smallest products first; f32:
      // (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
#pragma unroll
      for (int z = 0; z < KINDS; ++z) {
        if (z >= steps) continue;
        const int kind = (z << (2 - shift)) + (g4 >> shift);
        const bool in = kind < KINDS && chunk < chunks;
        const int xt = !in ? 0 : F32 ? 0x021010 >> (4 * (5 - kind)) & 3 : 2 - kind;
        const int wk = in && F32 ? 0x201100 >> (4 * (5 - kind)) & 3 : 0;
        u32x4 wv[CT];
#pragma unroll
        for (int v = 0; v < CT; ++v) {
          wv[v] = tm[v][0];
          if constexpr (F32) wv[v] = wk == 0 ? tm[v][0] : wk == 1 ? tm[v][1] : tm[v][2];
        }
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          u32x4 xv = *reinterpret_cast<const u32x4 *>(xs + (xt * TR + 16 * u + col) * ld + 8 * (in ? chunk : 0));
          if (!in) xv = u32x4{0, 0, 0, 0};
#pragma unroll
          for (int v = 0; v < CT; ++v) d[u][v] = mfma(wv[v], xv, d[u][v]);
        }
      }
    }
    f32x4 out[RT][2];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      // (one wave's own LDS, whose operations go in order)
#pragma unroll
      for (int v = 0; v < CT; ++v) *reinterpret_cast<f32x4 *>(&turn[w][col][16 * v + 4 * g4]) = d[u][v];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int h = 0; h < 2; ++h)
        out[u][h] = *reinterpret_cast<const f32x4 *>(&turn[w][8 * h + rl][cl]) + base[u][h];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    it = it + 1 < its ? it + 1 : 0;
    if (done + 1 < its) load(column(it));
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = c1 - c - cl;
        if (16 * u + 8 * h + rl >= n) continue;
        float *q = a.y + row_at(u, h) + c + cl;
        if (left >= 4) *reinterpret_cast<f32x4_u *>(q) = out[u][h];
        else
          for (int e = 0; e < 3; ++e)
            if (e < left) q[e] = out[u][h][e];
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
  const int64_t mine = all * RT;
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + mine - 1) / mine, (a.m + 511) / 512));
  if (RT > 1) a.splits = std::min(a.splits, 4);
  const int64_t per = record_ints<TR>() + (int64_t)a.splits * TR * a.ranks;
  const int64_t most = std::min<int64_t>(ws_floats / per, 65535);
  if (most < 1) return hipErrorInvalidValue;
  // (blocks are a grid's y)
  int cols = RT == 1 ? 128 : kCols, blocks = 0;
  for (;; cols *= 2) {
    blocks = 0;
    for (int p = 0; p < a.parts; ++p) blocks += (a.width[p] + cols - 1) / cols;
    if (blocks <= 65535) break;
  }
  const size_t lds0 = (size_t)(a.nadapters + 1) * 4, lds1 = (size_t)3 * TR * (a.max_rank + 8) * 2;
  for (int64_t t0 = 0; t0 < all; t0 += most) {
    a.tile0 = (int)t0;
    a.tiles = (int)std::min(most, all - t0);
    hipLaunchKernelGGL((lora_shrink_kernel<F32, RT>),
                       dim3((unsigned)a.tiles, (unsigned)a.splits, (unsigned)(rank_groups * RT)), dim3(kThreads), lds0,
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
  // Tiles of 64 rows where an adapter has 256 on average (f32: 64): fewer reads of its
  // weights and fewer terms of f32 ones, but fewer blocks (us in tiles of 64 / 16: four
  // adapters of 4096 x 14336, rank 64, with 128 rows each 43 / 36, 192 43 / 45, 256 60
  // / 63, 384 71 / 92; of 4096 x 4096, rank 16, 256 24 / 23, 512 31 / 34; f32, rank 64,
  // 32 rows 46 / 43, 64 51 / 69, 256 118 / 212; rank 16, 64 23 / 21, 128 24 / 26).
  const int64_t groups = std::min(a.nseq, a.nadapters);
  const bool wide = a.rows >= (a.f32 ? 64 : 256) * std::max<int64_t>(groups, 1) && a.max_rank <= 128;
  if (a.f32) return wide ? launch_lora_t<true, 4>(a, ws_floats, st) : launch_lora_t<true, 1>(a, ws_floats, st);
  return wide ? launch_lora_t<false, 4>(a, ws_floats, st) : launch_lora_t<false, 1>(a, ws_floats, st);
}

}  // namespace q8
