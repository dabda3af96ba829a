// q8_packed.hip -- causal attention over the prompts of several sequences,
// packed row after row.
//
// Row r of sequence i attends the rows cu[i] .. r of the same sequence, query
// head h reading KV head h / grp.  One block of 4 waves serves one KV head and
// rows_per_block(grp) consecutive rows of a sequence with all heads of the
// group: 128 columns, a column being one (row, query head).  K and V tiles of
// 64 keys are staged in LDS once for all of them (V transposed), each wave
// forms S^T = K Q^T and O^T += V^T P^T for its 32 columns with
// v_mfma_f32_32x32x16_f16 and keeps an online softmax.
//
// f32 q (and the probabilities beside them) enter as binary16 hi + lo pairs:
// q scaled per column by a power of two (largest |q| in [2^14, 2^15)), p by
// 2^14, so the pair carries a value to 2^-22 and to 2^-40 of the column's
// largest; K and V are binary16 already, so products are exact and the sums,
// f32, have f32-level error.  bf16 q fits one binary16 after the scaling, and
// p is rounded to one (2^-12 of itself, a sixteenth of the bf16 output's own
// rounding): half the matrix work.  (Of 16282 rows the error is 1.66e-3 of float64,
// with f32 probabilities 1.65e-3; one output in ten is the neighbouring bf16 value
// of the one that those give.)  Columns where those terms hold too little of
// the small dims of q (kFarDim) are formed in f32.
// Bound: MFMA (4 hd flops per (row, head, key seen), twice issued for f32) with
// the softmax's VALU work and the LDS traffic beside it; of 16001 rows in bf16
// (2.1 ms, 1000 TFLOP/s) the staging of the tiles costs 0.5 ms and the LDS reads of
// the operands 0.4.  Blocks of 4 waves, two to a CU, raise their priority in the
// matrix phases, so one block's softmax falls beside the other's products (8
// ragged f32 prompts 361 -> 349 us).
//
// Lane layout of the 32x32x16 MFMA (lane l, h = l / 32): A element i is
// A[l % 32][8h + i], B element i is B[8h + i][l % 32], accumulator element v is
// D[8(v / 4) + 4h + v % 4][l % 32].  The keys of a P^T column held by a lane
// follow the accumulator layout, so V^T stores each 16-key chunk permuted (key
// 8a + 4h + b at 8h + 4a + b).
#include "q8_device.h"
#include "q8_launch.h"
#include "q8_ragged.h"

namespace q8 {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
constexpr int kBK = 64;                // keys per staged tile
constexpr float kPScale = 16384.0f;    // 2^14 on p in binary16
// Rows per sequence from which heads of 128 take 8 waves a block, which halves the
// loads and LDS writes a column costs (one sequence of 8192 rows, 32 / 8 heads:
// f32 1014 -> 968 us, bf16 634 -> 572; of 2048 rows 96 -> 104 and 64 -> 67, for
// the tiles are twice as tall and fewer; 8 sequences of 700 rows, bf16, 64 ->
// 73).  Heads of 64 gain nothing (579 -> 595).
constexpr int kWideRows = 4096;
// Sequences up to which the row tiles are served longest first.
constexpr int kSorted = 16;

// Small dims of q: the terms' 2^-25 (at largest values in [2^14, 2^15)) is up to 2^-19
// of a dim 20 binary exponents below its column's largest, and bf16 (8 bits) is
// exact in them down to 31 below.  Dims that lie further below (one f32 column of
// normal values in 4000) make an error of the score of at most sqrt(HD) 2^-39
// max|q| max|k| (max|q| as the power of two below it), and of 6.6e-6, 6 times the
// mean square, where that product reaches 2^20: no binary16 k takes a largest q
// below 32 there.  From 32 on a wave with such a column looks its keys through, and
// columns past 2^20 are formed in f32: beside dims that are 2^23 to 2^126 times
// the others, and 0 in K, 1e-5 to 1 -> 8e-7 of float64.  (If every wave looked:
// 8088 ragged f32 rows 357 -> 452 us; with largest q below 32 none does.)
template <bool BF16> constexpr int kFarDim = BF16 ? 31 : 20;

// Rows of a block of nw waves, 32 columns each.
__host__ __device__ inline int rows_per_block(int grp, int nw) { return 32 * nw / grp; }

template <bool BF16> struct QType { typedef float T; };
template <> struct QType<true> { typedef __bf16 T; };

// Eight consecutive q values as f32.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    x[c] = a[c];
    x[4 + c] = b[c];
  }
}
__device__ __forceinline__ void load8(const __bf16 *p, float (&x)[8]) {
  const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    x[2 * c] = bf16_bits_to_f32(w[c] & 0xffffu);
    x[2 * c + 1] = bf16_bits_to_f32(w[c] >> 16);
  }
}
__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
__device__ __forceinline__ void store4(__bf16 *p, f32x4 v) {
  *reinterpret_cast<u32x2 *>(p) =
      u32x2{bf16_rne(v.x) | bf16_rne(v.y) << 16, bf16_rne(v.z) | bf16_rne(v.w) << 16};
}

// The largest |k| of the keys 0 .. nk-1, by one wave.
template <int HD>
__device__ __forceinline__ float largest(const __half *__restrict__ kc, int64_t kvdim, int nk, int lane) {
  constexpr int LPK = HD / 8, KPW = 64 / LPK;            // lanes of a key, keys of a load
  uint32_t mx = 0;
  for (int j0 = lane / LPK; j0 < nk; j0 += 8 * KPW) {
    u32x4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      x[u] = *reinterpret_cast<const u32x4 *>(kc + (int64_t)min(j0 + u * KPW, nk - 1) * kvdim + lane % LPK * 8);
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = max(mx, max(x[u][v] & 0x7fffu, x[u][v] >> 16 & 0x7fffu));
  }
  return wave_max((float)__builtin_bit_cast(_Float16, (uint16_t)mx));
}

// One (row, head) over its keys 0 .. nk-1 by one wave in f32, reading no other
// key: the output's dims lane (and lane + 64).
template <int HD, class T>
__device__ __forceinline__ void row_f32(const T *__restrict__ q, const __half *__restrict__ kc,
                                        const __half *__restrict__ vc, int64_t kvdim, int nk,
                                        int lane, float (&o)[HD / 64]) {
  const float cs = 1.44269504088896341f / sqrtf((float)HD);
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) o[e] = 0.0f;
  for (int j0 = 0; j0 < nk; j0 += 64) {
    const int n = min(64, nk - j0);
    float sc = -INFINITY;
    if (lane < n) {
      const __half *kr = kc + (int64_t)(j0 + lane) * kvdim;
      sc = 0.0f;
#pragma unroll 4
      for (int d = 0; d < HD; ++d) sc = __builtin_fmaf((float)q[d], __half2float(kr[d]), sc);
      sc *= cs;
    }
    const float mn = fmaxf(m, wave_max(sc));
    const float ms = mn == -INFINITY ? 0.0f : mn;   // (nothing but scores of -inf so far)
    const float alpha = exp2f(m - ms);
    const float p = lane < n ? exp2f(sc - ms) : 0.0f;
    l = __builtin_fmaf(l, alpha, wave_sum(p));
    m = mn;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) o[e] *= alpha;
    for (int t = 0; t < n; ++t) {
      const float pt =
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), t));
      const __half *vr = vc + (int64_t)(j0 + t) * kvdim + lane;
#pragma unroll
      for (int e = 0; e < HD / 64; ++e)
        o[e] = __builtin_fmaf(pt, __half2float(vr[64 * e]), o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < HD / 64; ++e) o[e] /= l;
}

// The row tile of block b of nb: tile `tile` of the sequence with the rows r0 ..
// r1-1 (none: tile < 0 or past the rows).  Up to 16 sequences: all tiles in
// descending order of their place in their sequence, which is the order of
// their key runs, so the longest start first whatever the sequences' order: tile
// k (and with it a sequence) of block b is the last k for which more than b
// tiles have a place from k on, searched by the lanes side by side (8 sequences
// of 700 rows, 32 / 8 heads of 64, 56.4 -> 51.5 us; 3000 rows between 600 and 40,
// of 128, 164 -> 160).  More sequences: the last ones' last tiles first, since the
// search grows with them and such tiles are short (61 sequences of 100 rows 33.6
// us, sorted 41.5).
struct PackedTile {
  int r0, r1;
  int64_t tile;
};
__device__ __forceinline__ PackedTile packed_tile(const int *__restrict__ cu, int nseq, int64_t rows,
                                                  int PB, int nb, int b) {
  const int lane = threadIdx.x & 63;
  if (nseq <= kSorted) {
    const int x = min(lane, nseq - 1);
    const int c0 = clamp_i(cu[x], 0, rows), c1 = clamp_i(cu[x + 1], 0, rows);
    const int tiles = lane < nseq && c1 > c0 ? (c1 - c0 + PB - 1) / PB : 0;
    int k0 = 0, step = nb, from = 0;             // k lies in [k0, k0 + step)
    do {
      step = (step + 63) / 64;
      const int k = k0 + lane * step;
      int c = 0;                                 // tiles with a place from k on
      for (int i = 0; i < nseq; ++i) c += max(__builtin_amdgcn_readlane(tiles, i) - k, 0);
      const uint64_t m = __builtin_amdgcn_ballot_w64(c > b);
      if (m == 0) return {0, 0, -1};
      const int z = 63 - __builtin_clzll(m);
      k0 += z * step;
      from = __builtin_amdgcn_readlane(c, z);
    } while (step > 1);
    const uint64_t m = __builtin_amdgcn_ballot_w64(tiles > k0);
    const int r = b - (from - (int)__builtin_popcountll(m));   // of the sequences that have a tile k0
    const int mine = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                                    __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    const uint64_t at = __builtin_amdgcn_ballot_w64((m >> lane & 1) && mine == r);
    const int i = at ? __builtin_ctzll(at) : 0;
    return {__builtin_amdgcn_readlane(c0, i), __builtin_amdgcn_readlane(c1, i), at ? k0 : -1};
  }
  b = nb - 1 - b;
  int i0 = 0, n = nseq;                          // the last i with seq_first_block(cu[i], i) <= b
  while (n > 1) {
    const int step = (n + 63) / 64, x = i0 + lane * step;
    const bool le = lane * step < n &&
                    seq_first_block(clamp_i(cu[x < nseq ? x : nseq - 1], 0, rows), x, PB, 1) <= b;
    const uint64_t m = __builtin_amdgcn_ballot_w64(le);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    n = min(n - k * step, step);
    i0 += k * step;
  }
  const int r0 = clamp_i(cu[i0], 0, rows);
  return {r0, clamp_i(cu[i0 + 1], 0, rows), b - seq_first_block(r0, i0, PB, 1)};
}

// Grid seq_blocks(rows, nseq, rows_per_block, 1) x nkv, the KV heads of a tile
// side by side (8 of them: one per XCD, whose L2 then holds that head).
template <int HD, bool BF16, int NW>
__global__ __launch_bounds__(64 * NW, 2) void packed_attn_kernel(PackedAttnArgs a) {
  typedef typename QType<BF16>::T T;
  constexpr int KS = HD / 16;                    // 16-dim steps of a score tile
  constexpr int DT = HD / 32;                    // 32-dim tiles of the output
  constexpr int KST = HD + 8;                    // K row stride in LDS (halves)
  constexpr int VST = kBK + 8;                   // V^T row stride in LDS (halves)
  constexpr int NTH = 64 * NW;                   // threads
  constexpr int KCH = (kBK * (HD / 8) + NTH - 1) / NTH;        // 16-byte K chunks per thread
  constexpr int VALL = (kBK / 2) * (HD / 8);     // V key pairs x 8 dims
  constexpr int VCH = (VALL + NTH - 1) / NTH;
  constexpr int NT = BF16 ? 1 : 2;               // binary16 terms of q and p
  constexpr int NB = NW == 8 ? 2 : 1;            // staged tiles
  __shared__ __attribute__((aligned(16))) _Float16 ks_[NB][kBK * KST];
  __shared__ __attribute__((aligned(16))) _Float16 vt_[NB][HD * VST];
  const int g = blockIdx.x % a.nkv, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = lane & 31, hf = lane >> 5;
  const int grp = a.nheads / a.nkv, PB = rows_per_block(grp, NW), nseq = (int)a.nseq;
  const PackedTile pt = packed_tile(a.cu, nseq, a.rows, PB, (int)(gridDim.x / a.nkv), (int)(blockIdx.x / a.nkv));
  const int r0 = pt.r0, r1 = pt.r1;
  const int64_t tile = pt.tile;
  if (tile < 0 || tile * PB >= r1 - r0) return;  // (the whole block)
  const int n = r1 - r0, row0 = (int)tile * PB;  // rows and keys count within the sequence
  const int nkeys = min(row0 + PB, n);
  const int ntiles = (nkeys + kBK - 1) / kBK;
  const int64_t kvdim = (int64_t)a.nkv * HD;
  const __half *kc = a.kc + (int64_t)r0 * kvdim + g * HD, *vc = a.vc + (int64_t)r0 * kvdim + g * HD;

  // this lane's column: row i, query head; columns past the rows read the
  // last one and store nothing
  const int ci = w * 32 + col, cr = ci / grp;
  const bool live = cr < PB && row0 + cr < n;
  const int i = min(row0 + min(cr, PB - 1), n - 1);
  const int head = g * grp + ci % grp;
  const int kend = i + 1;
  // keys that the wave's first and last columns see
  const int wfirst = min(row0 + min(w * 32 / grp, PB - 1), n - 1) + 1;
  const int wlast = min(row0 + min((w * 32 + 31) / grp, PB - 1), n - 1) + 1;
  const bool wlive = w * 32 / grp < PB && row0 + w * 32 / grp < n;

  half8 qf[NT][KS];
  float cs, klim;                                // |k| up to which the terms of q do
  {
    const T *qr = static_cast<const T *>(a.q) + (int64_t)(r0 + i) * a.ldq + (int64_t)head * HD + 8 * hf;
    float qv[KS][8], mx = 0.0f;
    uint32_t mn = ~0u;                           // (2 |q| as bits) - 1: zeros are largest
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      load8(qr + 16 * k, qv[k]);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        mx = fmaxf(mx, fabsf(qv[k][c]));
        mn = min(mn, (__builtin_bit_cast(uint32_t, qv[k][c]) << 1) - 1u);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    mn = min(mn, (uint32_t)__shfl_xor((int)mn, 32));
    const int ex = (int)((__builtin_bit_cast(uint32_t, mx) >> 23) & 255u) - 127;
    klim = (int)(mn >> 24) + kFarDim<BF16> < ex + 127 ? __builtin_ldexpf(1.0f, 20 - ex) : INFINITY;
    const int e = min(max(14 - ex, -126), 126);
    const float qsc = __builtin_ldexpf(1.0f, e);
    cs = __builtin_ldexpf(1.44269504088896341f / sqrtf((float)HD), -e);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float x = qv[k][c] * qsc;
        qf[0][k][c] = (_Float16)x;
        if constexpr (NT == 2) qf[1][k][c] = (_Float16)(x - (float)qf[0][k][c]);
      }
  }

  // staging: registers hold the next tile while the current one is used
  u32x4 kreg[KCH], vreg[VCH][2];
  auto load_tile = [&](int kt) {
    const int k0 = kt * kBK, nk = min(kBK, nkeys - k0);
    // keys past the block's read as zero
    const uint32_t nbytes = (uint32_t)(((nk - 1) * kvdim + HD) * 2);
    const rsrc_t rk = make_rsrc(kc + k0 * kvdim, nbytes), rv = make_rsrc(vc + k0 * kvdim, nbytes);
    const uint32_t kvd = (uint32_t)kvdim;
#pragma unroll
    for (int u = 0; u < KCH; ++u) {
      const uint32_t c = threadIdx.x + NTH * u, key = c / (HD / 8), dg = c % (HD / 8);
      kreg[u] = bload16(rk, (key * kvd + dg * 8) * 2);
    }
#pragma unroll
    for (int u = 0; u < VCH; ++u) {
      const uint32_t c = threadIdx.x + NTH * u, kp = c % (kBK / 2), dg = c / (kBK / 2);
      const uint32_t off = c < VALL ? (2 * kp * kvd + dg * 8) * 2 : kOutOfRange;
      vreg[u][0] = bload16(rv, off);
      vreg[u][1] = bload16(rv, off + kvd * 2);
    }
  };
  auto store_tile = [&](int buf) {
    _Float16 *ks = ks_[buf], *vt = vt_[buf];
#pragma unroll
    for (int u = 0; u < KCH; ++u) {
      const int c = threadIdx.x + NTH * u, key = c / (HD / 8), dg = c % (HD / 8);
      *reinterpret_cast<u32x4 *>(&ks[key * KST + dg * 8]) = kreg[u];
    }
#pragma unroll
    for (int u = 0; u < VCH; ++u) {
      const int c = threadIdx.x + NTH * u, kp = c % (kBK / 2), dg = c / (kBK / 2);
      if (VALL % NTH && c >= VALL) continue;
      const int key = 2 * kp, r = key & 15;
      const int at = (key & ~15) + 8 * ((r >> 2) & 1) + 4 * (r >> 3) + (r & 3);
#pragma unroll
      for (int d2 = 0; d2 < 4; ++d2) {
        // dims 8dg + 2d2 and +1: (key, key + 1) pairs as one 32-bit word each
        const uint32_t x = vreg[u][0][d2], y = vreg[u][1][d2];
        *reinterpret_cast<uint32_t *>(&vt[(dg * 8 + 2 * d2) * VST + at]) =
            __builtin_amdgcn_perm(y, x, 0x05040100u);
        *reinterpret_cast<uint32_t *>(&vt[(dg * 8 + 2 * d2 + 1) * VST + at]) =
            __builtin_amdgcn_perm(y, x, 0x07060302u);
      }
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[t][v] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  load_tile(0);
  if (NB == 2) {
    store_tile(0);
    if (ntiles > 1) load_tile(1);
  }
  for (int kt = 0; kt < ntiles; ++kt) {
    const _Float16 *ks = ks_[kt % NB], *vt = vt_[kt % NB];
    __syncthreads();                             // every wave is done with the last tile
    if (NB == 2) {                               // (and this one is staged)
      if (kt + 1 < ntiles) {
        store_tile((kt + 1) % NB);
        if (kt + 2 < ntiles) load_tile(kt + 2);
      }
    } else {
      store_tile(0);
      __syncthreads();
      if (kt + 1 < ntiles) load_tile(kt + 1);
    }
    const int k0 = kt * kBK;
    if (!wlive || k0 >= wlast) continue;         // past every row of this wave
    if (NB == 1) __builtin_amdgcn_s_setprio(1);
    f32x16 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[t][v] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const half8 x = *reinterpret_cast<const half8 *>(&ks[(32 * t + col) * KST + 16 * k + 8 * hf]);
#pragma unroll
        for (int z = 0; z < NT; ++z)
          sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qf[z][k], sc[t], 0, 0, 0);
      }
    }
    if (NB == 1) __builtin_amdgcn_s_setprio(0);
    // m is the running maximum of the scores in the log2 domain rounded to an
    // integer: p = exp2(s cs - m) takes one FMA, and alpha is a power of two
    // that is 1 for most tiles
    if (k0 + kBK > wfirst) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = k0 + 32 * t + 8 * (v >> 2) + 4 * hf + (v & 3);
          sc[t][v] = key < kend ? sc[t][v] : -INFINITY;
        }
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) tmax = fmaxf(tmax, sc[t][v]);
    tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
    // (key 0 is visible to every column, so m is -inf only for scores of -inf:
    // then p is NaN, as the formula has it)
    const float mn = fmaxf(m, __builtin_rintf(tmax * cs));
    const float alpha = __builtin_amdgcn_exp2f(m - mn), mp = BF16 ? mn - 14.0f : mn;
    m = mn;
    float ps = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][v], cs, -mp));
        sc[t][v] = p;
        ps += p;
      }
    l = __builtin_fmaf(l, alpha, ps);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] *= alpha;
    }
    if (NB == 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        half8 pf[NT];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float p = sc[t][8 * j + c];
          pf[0][c] = (_Float16)(BF16 ? p : p * kPScale);
          if constexpr (NT == 2) pf[1][c] = (_Float16)__builtin_fmaf(p, kPScale, -(float)pf[0][c]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const half8 x =
              *reinterpret_cast<const half8 *>(&vt[(32 * d + col) * VST + 32 * t + 16 * j + 8 * hf]);
#pragma unroll
          for (int z = 0; z < NT; ++z)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pf[z], o[d], 0, 0, 0);
        }
      }
    if (NB == 1) __builtin_amdgcn_s_setprio(0);
  }
  l += __shfl_xor(l, 32);
  // The MFMAs multiply every key of a tile into every column: 0 times an
  // infinite or NaN v of a key that the column's row must not see is NaN, and
  // so is an infinity times the halves of a pair.  A sum that once was not
  // finite stays so; these columns are formed again from their own keys, in f32.
  float chk = 0.0f * l;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) chk = __builtin_fmaf(o[t][v], 0.0f, chk);
  chk += __shfl_xor(chk, 32);
  bool bad = chk != 0.0f;
  if (__builtin_amdgcn_ballot_w64(live && klim < 65536.0f)) bad |= largest<HD>(kc, kvdim, wlast, lane) > klim;
  T *out = static_cast<T *>(a.out);
  const int64_t qdim = (int64_t)a.nheads * HD;
  if (live && !bad) {
    const float il = 1.0f / (BF16 ? l : l * kPScale);
    T *orow = out + (int64_t)(r0 + i) * qdim + (int64_t)head * HD + 4 * hf;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int vb = 0; vb < 4; ++vb) {
        f32x4 r;
#pragma unroll
        for (int c = 0; c < 4; ++c) r[c] = o[d][4 * vb + c] * il;
        store4(orow + 32 * d + 8 * vb, r);
      }
  }
  for (uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(live && bad); left; left &= left - 1) {
    const int x = w * 32 + __builtin_ctz(left);
    const int xi = row0 + x / grp, xh = g * grp + x % grp;
    float y[HD / 64];
    row_f32<HD>(static_cast<const T *>(a.q) + (int64_t)(r0 + xi) * a.ldq + (int64_t)xh * HD, kc, vc,
                kvdim, xi + 1, lane, y);
    T *orow = out + (int64_t)(r0 + xi) * qdim + (int64_t)xh * HD + lane;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) orow[64 * e] = (T)y[e];
  }
}

template <int HD, int NW>
hipError_t launch_packed_t(const PackedAttnArgs &a, hipStream_t st) {
  const int64_t nb = seq_blocks(a.rows, a.nseq, rows_per_block(a.nheads / a.nkv, NW), 1);
  const dim3 grid((unsigned)(nb * a.nkv));
  if (a.bf16)
    hipLaunchKernelGGL((packed_attn_kernel<HD, true, NW>), grid, dim3(64 * NW), 0, st, a);
  else
    hipLaunchKernelGGL((packed_attn_kernel<HD, false, NW>), grid, dim3(64 * NW), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_packed(const PackedAttnArgs &a, hipStream_t st) {
  if (a.head_dim == 64) return launch_packed_t<64, 4>(a, st);
  return a.rows >= kWideRows * a.nseq ? launch_packed_t<128, 8>(a, st) : launch_packed_t<128, 4>(a, st);
}

}  // namespace q8
