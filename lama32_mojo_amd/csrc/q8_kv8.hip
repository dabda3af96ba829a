// q8_kv8.hip -- the 8-bit paged cache of several sequences: append (RoPE at
// each row's own position, quantisation) and the attention that reads it.
//
// A page holds `page` tokens of one layer (kv8_page_bytes): K codes as rows
// [token][dim] and V codes as columns [dim][token], each head's contiguous, and
// one f32 scale per KV head for K and for V.  The value of a code is
// code * scale.  K and V are laid out as the two matrix products of the
// attention read them, so codes go from memory to the MFMA operands in
// registers, with no transposition and no LDS.
#include "q8_device.h"
#include "q8_launch.h"
#include "q8_ragged.h"

#include <algorithm>

namespace q8 {
namespace {

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));   // any f32 address

// The sequence of block b: the last i with seq_first_block(cu[i], i) <= b.
// The whole wave searches, 64 candidates a step.
__device__ __forceinline__ int find_seq(const int *__restrict__ cu, int nseq, int64_t rows,
                                        int64_t b, int tile, int spare) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = nseq;                     // the answer lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) / 64;         // candidates lo, lo + step, ...
    const int i = lo + lane * step;
    const bool le = lane * step < n &&
                    seq_first_block(clamp_i(cu[i < nseq ? i : nseq - 1], 0, rows), i, tile, spare) <= b;
    const uint64_t m = __builtin_amdgcn_ballot_w64(le);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    n = n - k * step < step ? n - k * step : step;
    lo += k * step;
  }
  return lo;
}

// cos and sin of pos * inv to f64 accuracy: the angle as an exact f64
// product (24 x 31 bits), less the nearest multiple of pi / 2 (pi / 2 in three
// parts, the first two of 33 bits, so that their products with the count are
// exact), then the Taylor series on [-pi/4, pi/4], whose first left-out terms
// are below 2^-54.  f32 angles of far positions are off by up to 2^-8 rad at
// 10^5 tokens; here the rotated key is rounded once, so equal inputs give
// equal codes on every path.
__device__ __forceinline__ void sincos_pos(int pos, float inv, double &sn, double &cs) {
  const double a = (double)pos * (double)inv;
  const double k = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-k, 0x1.921fb544p+0, a);
  r = __builtin_fma(-k, 0x1.0b4611a6p-34, r);
  r = __builtin_fma(-k, 0x1.3198a2e037073p-69, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0;                       // -1/15!
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  double c = 1.0 / 20922789888000.0;                       // 1/16!
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int q = (int)((int64_t)k & 3);
  const double ss = (q & 1) ? c : s, cc = (q & 1) ? s : c;
  sn = (q & 2) ? -ss : ss;
  cs = (q == 1 || q == 2) ? -cc : cc;
}

// ---- append --------------------------------------------------------------------
// One block of 256 threads per (page that a sequence's new rows touch, KV
// head), grid (seq_blocks(rows, nseq, page, 2), nkv).  It rotates the head's
// keys and its query heads, takes the largest |k| and |v| of the new rows,
// settles the page's two scales (s1 = max(s0, amax / 127); s0 counts where old
// tokens lie in the page), re-rounds the old tokens' codes where the scale
// grew, and writes the new codes.  A thread holds (token, dims 4j .. 4j+3 and
// their partners half a head on) items, so the rotation needs no exchange and
// the values stay in registers between the two passes.
// Bound: HBM for prompts (q read and written, k and v read, codes written),
// the chain of dependent loads for a token per sequence.

// rint(x / s), half to even, as if divided exactly: c = rint(x * (1/s)) is off
// by one at most, next to a border; x - c s is exact (a multiple of ulp(s) below
// 2^24 of them), so its side of s / 2 settles it.
__device__ __forceinline__ float code_of(float x, float s, float inv) {
  float c = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-c, s, x), h = 0.5f * s;
  const bool odd = ((int)c & 1) != 0;
  c += (r > h || (r == h && odd)) ? 1.0f : (r < -h || (r == -h && odd)) ? -1.0f : 0.0f;
  return __builtin_fminf(__builtin_fmaxf(c, -127.0f), 127.0f);
}

template <int HD, int P>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  constexpr int half = HD / 2;
  constexpr int IPT = HD / 8;                 // items per token
  constexpr int TPP = 256 / IPT;              // tokens per pass
  constexpr int NP = (P + TPP - 1) / TPP;     // passes
  constexpr int VST = P + 4;                  // bytes of a V column in LDS
  __shared__ __attribute__((aligned(16))) uint8_t vt[HD * VST];
  __shared__ uint32_t red[2][4];
  const Kv8Args &c = a.c;
  const int t = threadIdx.x, g = blockIdx.y, grp = c.nheads / c.nkv;
  const int nseq = (int)c.nseq;
  const int i = find_seq(c.cu, nseq, c.rows, blockIdx.x, P, 2);
  const int r0 = clamp_i(c.cu[i], 0, c.rows), r1 = clamp_i(c.cu[i + 1], 0, c.rows);
  const int len = clamp_i(c.len[i], 0, (int64_t)1 << 30);
  const int64_t b = (int64_t)blockIdx.x - seq_first_block(r0, i, P, 2);
  const int64_t pg = len / P + b;             // page of the sequence
  const int64_t p0 = pg * P;                  // its first position
  const int64_t ta = p0 > len ? p0 : len, tz = min(p0 + P, (int64_t)len + (r1 - r0));
  if (b < 0 || ta >= tz) return;              // (the whole block)
  const int e = (int)(ta - p0), z = (int)(tz - p0);   // new tokens of the page: [e, z)
  const int row0 = r0 + (int)(p0 - len);      // row of the page's token 0
  int id = pg < c.maxpages ? c.tab[(int64_t)i * c.maxpages + pg] : -1;
  id = page_or_none(id, (int)c.npages);
  const int64_t kvdim = (int64_t)c.nkv * HD;

  float kx[NP][8], vx[NP][8];
  uint32_t kmax = 0, vmax = 0;                // |.| as bits: NaN above infinity above all
  const int j = t % IPT;                      // dims 4j .. and half + 4j ..
  float freq[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) freq[u] = a.inv[4 * j + u];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int tok = p * TPP + t / IPT;
#pragma unroll
    for (int u = 0; u < 8; ++u) kx[p][u] = vx[p][u] = 0.0f;
    if (tok < e || tok >= z) continue;
    const int64_t row = row0 + tok;
    const float *kr = a.k + row * a.ldk + g * HD + 4 * j, *vr = a.v + row * a.ldk + g * HD + 4 * j;
    const f32x4 k0 = *reinterpret_cast<const f32x4_u *>(kr);
    const f32x4 k1 = *reinterpret_cast<const f32x4_u *>(kr + half);
    const f32x4 v0 = *reinterpret_cast<const f32x4_u *>(vr);
    const f32x4 v1 = *reinterpret_cast<const f32x4_u *>(vr + half);
    float cs[4], sn[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      double s, co;
      sincos_pos((int)p0 + tok, freq[u], s, co);
      cs[u] = (float)co;
      sn[u] = (float)s;
      kx[p][u] = (float)__builtin_fma((double)k0[u], co, -((double)k1[u] * s));
      kx[p][4 + u] = (float)__builtin_fma((double)k1[u], co, (double)k0[u] * s);
      vx[p][u] = v0[u];
      vx[p][4 + u] = v1[u];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      kmax = max(kmax, __builtin_bit_cast(uint32_t, kx[p][u]) & 0x7fffffffu);
      vmax = max(vmax, __builtin_bit_cast(uint32_t, vx[p][u]) & 0x7fffffffu);
    }
    if (a.krow) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4), aligned(2)));
      const int64_t o = row * kvdim + g * HD + 4 * j;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half4 y, x;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          y[u] = (_Float16)kx[p][4 * h + u];
          x[u] = (_Float16)vx[p][4 * h + u];
        }
        *reinterpret_cast<half4 *>(a.krow + o + h * half) = y;
        *reinterpret_cast<half4 *>(a.vrow + o + h * half) = x;
      }
    }
    for (int hh = 0; hh < grp; ++hh) {
      const int64_t o = (int64_t)(g * grp + hh) * HD + 4 * j;
      const float *qr = a.q + row * a.ldq + o;
      const f32x4 q0 = *reinterpret_cast<const f32x4_u *>(qr);
      const f32x4 q1 = *reinterpret_cast<const f32x4_u *>(qr + half);
      f32x4 y0, y1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        y0[u] = __builtin_fmaf(q0[u], cs[u], -(q1[u] * sn[u]));
        y1[u] = __builtin_fmaf(q1[u], cs[u], q0[u] * sn[u]);
      }
      float *qo = a.qr + row * a.ldr + o;
      *reinterpret_cast<f32x4_u *>(qo) = y0;
      *reinterpret_cast<f32x4_u *>(qo + half) = y1;
    }
  }
  if (id < 0) return;                         // no page: nothing is stored (the whole block)
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    kmax = max(kmax, (uint32_t)__shfl_xor((int)kmax, d));
    vmax = max(vmax, (uint32_t)__shfl_xor((int)vmax, d));
  }
  if ((t & 63) == 0) {
    red[0][t >> 6] = kmax;
    red[1][t >> 6] = vmax;
  }
  __syncthreads();
  uint8_t *page = c.pages + (int64_t)id * kv8_page_bytes(P, c.nkv, HD);
  float *scale = reinterpret_cast<float *>(page + kv8_scales_at(P, c.nkv, HD));
  float s0[2], s1[2], inv[2];
  bool fine[2], grew[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t mx = max(max(red[x][0], red[x][1]), max(red[x][2], red[x][3]));
    const float am = __builtin_bit_cast(float, mx) / 127.0f;
    s0[x] = e > 0 ? scale[x * c.nkv + g] : 0.0f;
    s1[x] = am > s0[x] || am != am ? am : s0[x];          // (a NaN s0 stays)
    fine[x] = __builtin_isfinite(s1[x]);
    if (!fine[x]) s1[x] = __builtin_nanf("");
    grew[x] = e > 0 && fine[x] && s1[x] > s0[x];
    // 1 / s1 and x - c s1 keep their bits while s1 is well inside the normal
    // range; below, the codes are formed from the f64 quotient
    inv[x] = 1.0f / s1[x];
  }
  __syncthreads();                            // every thread has read s0
  if (t < 2) scale[t * c.nkv + g] = s1[t];
  uint8_t *kc = page + (int64_t)g * P * HD, *vc = page + (int64_t)(c.nkv + g) * P * HD;
  auto code = [&](float x, int w) -> uint32_t {
    if (!fine[w] || s1[w] == 0.0f) return 0;
    const float q = s1[w] > 0x1p-100f
                        ? code_of(x, s1[w], inv[w])
                        : (float)fmin(fmax(rint((double)x / (double)s1[w]), -127.0), 127.0);
    return (uint32_t)(int)q & 255u;
  };
  // the old tokens' codes at a larger scale
  auto again = [&](uint8_t *at, int w) {
    const double d = (double)(int8_t)*at * (double)s0[w] / (double)s1[w];
    *at = (uint8_t)(int8_t)(int)rint(d);
  };
  if (grew[0])
    for (int n = t; n < e * HD; n += 256) again(kc + n, 0);
  if (grew[1])
    for (int n = t; n < e * HD; n += 256) again(vc + (n / e) * P + n % e, 1);
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int tok = p * TPP + t / IPT;
    if (tok < e || tok >= z) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        w |= code(kx[p][4 * h + u], 0) << (8 * u);
        vt[(h * half + 4 * j + u) * VST + tok] = (uint8_t)code(vx[p][4 * h + u], 1);
      }
      *reinterpret_cast<uint32_t *>(kc + tok * HD + h * half + 4 * j) = w;
    }
  }
  __syncthreads();
  if (e == 0 && z == P) {                     // a whole page: 4 tokens a store
    for (int n = t; n < HD * P / 4; n += 256) {
      const int d = n / (P / 4), x = 4 * (n % (P / 4));
      *reinterpret_cast<uint32_t *>(vc + d * P + x) =
          *reinterpret_cast<const uint32_t *>(&vt[d * VST + x]);
    }
  } else {
    const int m = z - e;
    for (int n = t; n < HD * m; n += 256) {
      const int d = n / m, x = e + n % m;
      vc[d * P + x] = vt[d * VST + x];
    }
  }
}

// ---- attention -------------------------------------------------------------------
// out[column] = sum_t p_t vs[page(t)] vcode_t / sum_t p_t over the keys t that
// the column's row sees, p_t = exp(ks[page(t)] (q . kcode_t) / sqrt(HD) - max),
// a column being one (row, query head) of a KV head's group.
//
// Bound: HBM (2 HD bytes a key and KV head), as long as a tile's columns are
// few.  The units of work (64 keys of one sequence's row tile) of all sequences
// are laid end to end and cut into equal runs, one per block of a KV head, so
// ragged contexts leave no block behind; a run that ends inside a row tile
// leaves a record for kv8_merge_kernel.  Within a run the block's four waves
// take the units in turn, each with its own online softmax, and meet in LDS.
//
// A wave holds a unit's codes in registers: S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32_bf16, the codes as bf16 (exact), q and p as three bf16
// terms each whose sum is the f32 value, so products are exact and scores and
// sums carry f32-level error whatever the sizes of q's dims or the scales; the
// scales are applied to scores and probabilities in f32.  Lane layout (lane l,
// g4 = l / 16): A element i is A[l % 16][8 g4 + i], B element i is
// B[8 g4 + i][l % 16], accumulator element i is D[4 g4 + i][l % 16].  Which key
// is row r of score tile tt, and which dim is element (step, g4, i), is free;
// taking key 16 (r / 4) + 4 tt + r % 4 makes the four accumulators of a lane
// hold 16 consecutive keys of its column, the ones its V operand loads as one
// 16-byte run of a V column, and taking dim 64 h + 16 g4 + 8 e + i for step
// 2 h + e makes its K operands two halves of one 16-byte run of a K row.
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

// x as three bf16 terms (truncations, exact): the upper halves of h, m, l.
__device__ __forceinline__ void split3(float x, float &h, float &m, float &l) {
  h = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u);
  const float r = x - h;
  m = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r) & 0xffff0000u);
  l = r - m;
}
__device__ __forceinline__ void split3x8(const float (&x)[8], u32x4 (&o)[3]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    float a0, a1, a2, b0, b1, b2;
    split3(x[2 * u], a0, a1, a2);
    split3(x[2 * u + 1], b0, b1, b2);
    o[0][u] = pk_hi16(a0, b0);
    o[1][u] = pk_hi16(a1, b1);
    o[2][u] = pk_hi16(a2, b2);
  }
}

// Prefix sums of the sequences' units in LDS (pre[0] = 0 .. pre[nseq]); all
// 256 threads.
__device__ __forceinline__ int kv8_plan(const Kv8Args &c, int cols, int *pre, int *wsum) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, nseq = (int)c.nseq;
  const int grp = c.nheads / c.nkv;
  int base = 0;
  if (t == 0) pre[0] = 0;
  for (int i0 = 0; i0 < nseq; i0 += 256) {
    const int i = i0 + t;
    int u = 0;
    if (i < nseq) {
      const Kv8Seq s = kv8_seq(c.cu[i], c.cu[i + 1], c.len[i], c.rows, c.maxpages * c.page, grp, cols);
      u = kv8_units_of(s);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(u, d);
      if (lane >= d) u = kv8_add(u, o);
    }
    if (lane == 63) wsum[w] = u;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      u = kv8_add(u, x < w ? wsum[x] : 0);
      all = kv8_add(all, wsum[x]);
    }
    if (i < nseq) pre[i + 1] = kv8_add(base, u);
    base = kv8_add(base, all);
    __syncthreads();
  }
  return base;
}

// The sequence that holds unit u: the last i with pre[i] <= u.
__device__ __forceinline__ int kv8_seq_of(const int *pre, int nseq, int u) {
  int lo = 0, hi = nseq;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= u) lo = m;
    else hi = m;
  }
  return lo;
}

constexpr int kKv8Least = 4;              // units a block serves at least: one per wave

// Record of a block and KV head: o[NC][HD] unnormalised, m[NC], l[NC]; slot 0
// for a run that begins inside a row tile, slot 1 for one that ends inside.
template <int HD, int NC> constexpr int kv8_record() { return NC * (HD + 2); }

template <int HD, int MT>
__global__ __launch_bounds__(256, 2) void kv8_attn_kernel(Kv8AttnArgs a) {
  constexpr int KS = HD / 32, DT = HD / 16, HH = HD / 64, NC = 16 * MT;
  constexpr int OST = HD + 4;             // floats of a column's sums in LDS
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  // q fragments [term][step][tile][lane], then (at the end of a segment) the
  // sums of two waves; behind them the prefix sums
  u32x4 *qf = reinterpret_cast<u32x4 *>(lds);
  float *ob = reinterpret_cast<float *>(lds);
  constexpr int kQBytes = 3 * KS * MT * 64 * 16, kOBytes = 2 * NC * OST * 4;
  int *pre = reinterpret_cast<int *>(lds + (kQBytes > kOBytes ? kQBytes : kOBytes));
  __shared__ int wsum[4];
  __shared__ float wm[4][NC], wl[4][NC];
  const Kv8Args &c = a.c;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, col = lane & 15, g4 = lane >> 4;
  const int g = blockIdx.y, grp = c.nheads / c.nkv, nseq = (int)c.nseq, P = c.page;
  const int64_t cap = c.maxpages * P;
  const int64_t pbytes = kv8_page_bytes(P, c.nkv, HD);
  const int64_t scales_at = kv8_scales_at(P, c.nkv, HD);
  const int64_t k_at = (int64_t)g * P * HD, v_at = (int64_t)(c.nkv + g) * P * HD;
  const float qscale = 1.44269504088896341f / sqrtf((float)HD);

  const int units = kv8_plan(c, NC, pre, wsum);
  const int per = kv8_units_per_block(units, gridDim.x, kKv8Least);
  int u = blockIdx.x * per;
  const int uend = min(u + per, units);
  while (u < uend) {
    const int i = kv8_seq_of(pre, nseq, u);
    const Kv8Seq sq = kv8_seq(c.cu[i], c.cu[i + 1], c.len[i], c.rows, cap, grp, NC);
    const int local = u - pre[i], rt = local / sq.key_units, t0 = local % sq.key_units;
    const int t1 = min(sq.key_units, t0 + (uend - u));
    u += t1 - t0;
    const int row0 = clamp_i(c.cu[i], 0, c.rows);
    const int *tab = c.tab + (int64_t)i * c.maxpages;
    const int ctx = (int)min((int64_t)sq.old + sq.n, cap);

    // ---- q of the tile's columns, scaled, as three bf16 terms
    __syncthreads();                      // the last segment's sums are read
    for (int n = t; n < NC * (HD / 8); n += 256) {
      const int cc = n / (HD / 8), d8 = n % (HD / 8);
      const int lin = rt * NC + cc, j = lin / grp;
      float x[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) x[v] = 0.0f;
      if (j < sq.n) {
        const float *q = a.q + (int64_t)(row0 + j) * a.ldq + (int64_t)(g * grp + lin % grp) * HD + 8 * d8;
        const f32x4 x0 = *reinterpret_cast<const f32x4_u *>(q);
        const f32x4 x1 = *reinterpret_cast<const f32x4_u *>(q + 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          x[v] = x0[v] * qscale;
          x[4 + v] = x1[v] * qscale;
        }
      }
      u32x4 f[3];
      split3x8(x, f);
      const int h = d8 >> 3, gg = (d8 & 7) >> 1, e = d8 & 1;
#pragma unroll
      for (int k = 0; k < 3; ++k)
        qf[((k * KS + 2 * h + e) * MT + cc / 16) * 64 + gg * 16 + cc % 16] = f[k];
    }
    // keys each of this lane's columns sees: 0 .. kend-1 (0: no such column)
    int kend[MT];
    int kmin = INT32_MAX;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int j = (rt * NC + 16 * mt + col) / grp;
      kend[mt] = j < sq.n ? (int)min((int64_t)sq.old + j + 1, cap) : 0;
      if (j < sq.n) kmin = min(kmin, kend[mt]);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) kmin = min(kmin, __shfl_xor(kmin, d));
    __syncthreads();

    // ---- the wave's units
    u32x4 kr[4][HH], vr[DT];
    float ks = 0.0f, vs = 0.0f;
    // page of the 16 keys from key0 on (reads page 0 where there is none)
    auto page_at = [&](int key0) -> int {
      return key0 < ctx ? page_or_none(tab[key0 / P], (int)c.npages) : 0;
    };
    auto load_k = [&](int kt) {
      const int key0 = kt * kKv8Unit + 16 * (col >> 2);
      const int id = page_at(key0);
      const uint8_t *p = c.pages + (id < 0 ? 0 : id) * pbytes + k_at +
                         (int64_t)(key0 % P + (col & 3)) * HD + 16 * g4;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int h = 0; h < HH; ++h)
          kr[tt][h] = *reinterpret_cast<const u32x4 *>(p + 4 * tt * HD + 64 * h);
    };
    auto load_v = [&](int kt) {
      const int key0 = kt * kKv8Unit + 16 * g4;
      const int id = page_at(key0);
      const uint8_t *base = c.pages + (id < 0 ? 0 : id) * pbytes;
      const float *sc = reinterpret_cast<const float *>(base + scales_at);
      ks = id < 0 ? __builtin_nanf("") : sc[g];
      vs = id < 0 ? __builtin_nanf("") : sc[c.nkv + g];
      const uint8_t *p = base + v_at + (int64_t)col * P + key0 % P;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        vr[d] = *reinterpret_cast<const u32x4 *>(p + (int64_t)16 * d * P);
    };
    f32x4 o[DT][MT];
    float m[MT], l[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = -INFINITY;
      l[mt] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][mt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int kt = t0 + w;
    if (kt < t1) {
      load_k(kt);
      load_v(kt);
    }
    for (; kt < t1; kt += 4) {
      f32x4 s[4][MT];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[tt][mt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < HH; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          bf16x8_t ka[4];
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) ka[tt] = codes_to_bf16(kr[tt][h][2 * e], kr[tt][h][2 * e + 1]);
#pragma unroll
          for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const bf16x8_t b =
                  __builtin_bit_cast(bf16x8_t, qf[((k * KS + 2 * h + e) * MT + mt) * 64 + lane]);
#pragma unroll
              for (int tt = 0; tt < 4; ++tt)
                s[tt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[tt], b, s[tt][mt], 0, 0, 0);
            }
        }
      const float ksc = ks, vsc = vs;
      if (kt + 4 < t1) load_k(kt + 4);
      const int key0 = kt * kKv8Unit + 16 * g4;
      const bool masked = kt * kKv8Unit + kKv8Unit > kmin;
      u32x4 pf[2][MT][3];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float tmax = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float x = s[tt][mt][v] * ksc;
            if (masked) x = key0 + 4 * tt + v < kend[mt] ? x : -INFINITY;
            s[tt][mt][v] = x;
            tmax = fmaxf(tmax, x);
          }
        tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
        // the maximum rounded to an integer: alpha is a power of two, and 1
        // for most units
        const float mnew = fmaxf(m[mt], __builtin_rintf(tmax));
        const float ms = mnew == -INFINITY ? 0.0f : mnew;
        const float alpha = __builtin_amdgcn_exp2f(m[mt] - ms);
        m[mt] = mnew;
        float ps = 0.0f;
        float pv[2][8];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float p = __builtin_amdgcn_exp2f(s[tt][mt][v] - ms);
            ps += p;
            // (a page of NaN scale counts for the rows that see one of its keys)
            float x = p * vsc;
            if (masked) x = key0 + 4 * tt + v < kend[mt] ? x : 0.0f;
            pv[tt >> 1][4 * (tt & 1) + v] = x;
          }
        l[mt] = __builtin_fmaf(l[mt], alpha, ps);
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][mt] *= alpha;
        }
        split3x8(pv[0], pf[0][mt]);
        split3x8(pv[1], pf[1][mt]);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bf16x8_t va = codes_to_bf16(vr[d][2 * e], vr[d][2 * e + 1]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int k = 0; k < 3; ++k)
              o[d][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  va, __builtin_bit_cast(bf16x8_t, pf[e][mt][k]), o[d][mt], 0, 0, 0);
        }
      if (kt + 4 < t1) load_v(kt + 4);
    }

    // ---- the four waves meet
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      l[mt] += __shfl_xor(l[mt], 16);
      l[mt] += __shfl_xor(l[mt], 32);
      if (g4 == 0) {
        wm[w][16 * mt + col] = m[mt];
        wl[w][16 * mt + col] = l[mt];
      }
    }
    __syncthreads();                      // (and q's fragments are done with)
    float mall[MT], lall[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int cc = 16 * mt + col;
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 4; ++x) mx = fmaxf(mx, wm[x][cc]);
      const float ms = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        sum = __builtin_fmaf(wl[x][cc], __builtin_amdgcn_exp2f(wm[x][cc] - ms), sum);
      mall[mt] = mx;
      lall[mt] = sum;
      const float f = __builtin_amdgcn_exp2f(m[mt] - ms);
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d][mt] *= f;
    }
    auto put = [&](float *dst) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<f32x4 *>(dst + (16 * mt + col) * OST + 16 * d + 4 * g4) = o[d][mt];
    };
    auto take = [&](const float *src) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d][mt] += *reinterpret_cast<const f32x4 *>(src + (16 * mt + col) * OST + 16 * d + 4 * g4);
    };
    // (a wave without units adds zeros; its order in the sum is fixed)
    if (w >= 2) put(ob + (w - 2) * NC * OST);
    __syncthreads();
    if (w < 2) take(ob + w * NC * OST);
    __syncthreads();
    if (w == 1) put(ob);
    __syncthreads();
    if (w == 0) {
      take(ob);
      const bool whole = t0 == 0 && t1 == sq.key_units;
      float *rec = a.ws + (((int64_t)blockIdx.x * c.nkv + g) * 2 + (t0 == 0)) * kv8_record<HD, NC>();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int cc = 16 * mt + col, lin = rt * NC + cc, j = lin / grp;
        if (whole) {
          if (j >= sq.n) continue;
          const float il = 1.0f / lall[mt];
          float *out = a.out + ((int64_t)(row0 + j) * c.nheads + g * grp + lin % grp) * HD + 4 * g4;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4_u *>(out + 16 * d) = o[d][mt] * il;
        } else {
#pragma unroll
          for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4 *>(rec + cc * HD + 16 * d + 4 * g4) = o[d][mt];
          if (g4 == 0) {
            rec[NC * HD + cc] = mall[mt];
            rec[NC * HD + NC + cc] = lall[mt];
          }
        }
      }
    }
  }
}

// Joins the records of the row tiles that several blocks served: grid
// (rows, nkv), the block's threads over the group's heads x HD / 4 dims.
template <int HD, int MT>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8AttnArgs a, int nblocks) {
  constexpr int NC = 16 * MT;
  extern __shared__ __attribute__((aligned(16))) int pre[];
  __shared__ int wsum[4];
  const Kv8Args &c = a.c;
  const int g = blockIdx.y, grp = c.nheads / c.nkv, nseq = (int)c.nseq;
  const int row = blockIdx.x;
  const int units = kv8_plan(c, NC, pre, wsum);
  const int per = kv8_units_per_block(units, nblocks, kKv8Least);
  __syncthreads();
  // the sequence of this row
  int lo = 0, hi = nseq;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (c.cu[m] <= row) lo = m;
    else hi = m;
  }
  const Kv8Seq sq = kv8_seq(c.cu[lo], c.cu[lo + 1], c.len[lo], c.rows, c.maxpages * c.page, grp, NC);
  const int j = row - clamp_i(c.cu[lo], 0, c.rows);
  if (j < 0 || j >= sq.n) return;             // behind the last sequence
  for (int n = threadIdx.x; n < grp * (HD / 4); n += 256) {
    const int hh = n / (HD / 4), d = 4 * (n % (HD / 4));
    const int lin = j * grp + hh, rt = lin / NC, cc = lin % NC;
    const int64_t ua = pre[lo] + (int64_t)rt * sq.key_units;
    const int b0 = clamp_i(ua / per, 0, nblocks - 1);
    const int b1 = clamp_i((ua + sq.key_units - 1) / per, 0, nblocks - 1);
    if (b0 == b1) continue;                   // written whole
    auto rec = [&](int b) {
      return a.ws + (((int64_t)b * c.nkv + g) * 2 + (b == b0)) * kv8_record<HD, NC>();
    };
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int z0 = b0; z0 <= b1; z0 += 8) {
      float zm[8], zl[8];
      f32x4 zo[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float *r = rec(z0 + x <= b1 ? z0 + x : b1);
        zm[x] = r[NC * HD + cc];
        zl[x] = r[NC * HD + NC + cc];
        zo[x] = *reinterpret_cast<const f32x4 *>(r + cc * HD + d);
      }
      float mx = m;
#pragma unroll
      for (int x = 0; x < 8; ++x) mx = fmaxf(mx, z0 + x <= b1 ? zm[x] : -INFINITY);
      const float ms = mx == -INFINITY ? 0.0f : mx;
      const float f0 = __builtin_amdgcn_exp2f(m - ms);
      l *= f0;
      o *= f0;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float f = z0 + x <= b1 ? __builtin_amdgcn_exp2f(zm[x] - ms) : 0.0f;
        if (z0 + x > b1) continue;
        l = __builtin_fmaf(f, zl[x], l);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = __builtin_fmaf(f, zo[x][v], o[v]);
      }
      m = mx;
    }
    const float il = 1.0f / l;
    *reinterpret_cast<f32x4_u *>(a.out + ((int64_t)row * c.nheads + g * grp + hh) * HD + d) = o * il;
  }
}

template <int HD, int MT>
hipError_t launch_kv8_attn_t(const Kv8AttnArgs &a, hipStream_t st) {
  constexpr int NC = 16 * MT, KS = HD / 32, OST = HD + 4;
  constexpr int kQBytes = 3 * KS * MT * 64 * 16, kOBytes = 2 * NC * OST * 4;
  const Kv8Args &c = a.c;
  const int grp = c.nheads / c.nkv;
  // two blocks per CU over all KV heads, as far as the work (by its bound)
  // and the records' space reach
  const int64_t units = (c.rows * grp / NC + c.nseq) * ((c.maxpages * c.page + kKv8Unit - 1) / kKv8Unit);
  int64_t nb = (512 + c.nkv - 1) / c.nkv;
  nb = std::min(nb, (units + kKv8Least - 1) / kKv8Least);
  nb = std::min(nb, a.ws_floats / (2 * (int64_t)c.nkv * kv8_record<HD, NC>()));
  if (nb < 1) nb = 1;
  const size_t plan = (size_t)(c.nseq + 1) * 4;
  const size_t lds = (size_t)std::max(kQBytes, kOBytes) + plan;
  hipLaunchKernelGGL((kv8_attn_kernel<HD, MT>), dim3((unsigned)nb, (unsigned)c.nkv), dim3(256), lds,
                     st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || nb == 1) return e;
  hipLaunchKernelGGL((kv8_merge_kernel<HD, MT>), dim3((unsigned)c.rows, (unsigned)c.nkv), dim3(256),
                     plan, st, a, (int)nb);
  return hipGetLastError();
}

template <int HD>
hipError_t launch_append_t(const Kv8AppendArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)seq_blocks(a.c.rows, a.c.nseq, a.c.page, 2), (unsigned)a.c.nkv);
  switch (a.c.page) {
    case 16: hipLaunchKernelGGL((kv8_append_kernel<HD, 16>), grid, dim3(256), 0, st, a); break;
    case 32: hipLaunchKernelGGL((kv8_append_kernel<HD, 32>), grid, dim3(256), 0, st, a); break;
    case 64: hipLaunchKernelGGL((kv8_append_kernel<HD, 64>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((kv8_append_kernel<HD, 128>), grid, dim3(256), 0, st, a); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_append(const Kv8AppendArgs &a, hipStream_t st) {
  return a.c.head_dim == 64 ? launch_append_t<64>(a, st) : launch_append_t<128>(a, st);
}

hipError_t launch_kv8_attention(const Kv8AttnArgs &a, hipStream_t st) {
  // one 16-column tile where a sequence's rows fill no more on average
  const bool one = a.c.rows * (a.c.nheads / a.c.nkv) <= 16 * a.c.nseq;
  if (a.c.head_dim == 64)
    return one ? launch_kv8_attn_t<64, 1>(a, st) : launch_kv8_attn_t<64, 2>(a, st);
  return one ? launch_kv8_attn_t<128, 1>(a, st) : launch_kv8_attn_t<128, 2>(a, st);
}

}  // namespace q8
