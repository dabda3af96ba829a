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

// The sequence of block b: the last i with seq_first_block(cu[i], i) <= b, with
// its rows and length.  The whole wave searches, 64 candidates a step, and reads
// the candidates' rows and lengths along, so up to 64 sequences take one round
// trip.
struct SeqAt {
  int i, r0, r1, len;
};
__device__ __forceinline__ SeqAt find_seq(const int *__restrict__ cu, const int *__restrict__ len,
                                          int nseq, int64_t rows, int64_t b, int tile, int spare) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = nseq;                     // the answer lies in [lo, lo + n)
  for (;;) {
    const int step = (n + 63) / 64;         // candidates lo, lo + step, ...
    const int i = min(lo + lane * step, nseq - 1);
    const int c0 = clamp_i(cu[i], 0, rows), c1 = clamp_i(cu[i + 1], 0, rows), ln = len[i];
    const bool le = lane * step < n && seq_first_block(c0, i, tile, spare) <= b;
    const uint64_t m = __builtin_amdgcn_ballot_w64(le);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    n = min(n - k * step, step);
    lo += k * step;
    if (n <= 1)
      return {lo, __builtin_amdgcn_readlane(c0, k), __builtin_amdgcn_readlane(c1, k),
              __builtin_amdgcn_readlane(ln, k)};
  }
}

// cos and sin of pos * inv to f64 accuracy: the angle as an exact f64
// product (24 x 29 bits), less the nearest multiple of pi / 2 (pi / 2 in three
// parts, the first two of 33 bits, so that their products with counts below 2^20
// are exact), then the Taylor series on [-pi/4, pi/4], whose first left-out terms
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
// settles the page's two scales (s1 = max(s0, amax * f32(1 / 127)), a product by
// definition: the quotient is another number in 1 of 20 cases, and codes beside a
// border are others by it; s0 counts where old tokens lie in the page), re-rounds
// the old tokens' codes where the scale grew, and writes the new codes.  Keys,
// whose codes must not depend on the path, are rotated in f64 and rounded once;
// q takes cos and sin rounded to f32 and f32 products (3.5e-8 of float64; rounded
// once 2.5e-8, for f64 products of every head of the group).  A thread holds
// (token, dims 4j .. 4j+3 and their partners half a head on) items, so the
// rotation needs no exchange and the values stay in registers between the passes.
// Bound: HBM for prompts (q read and written, k and v read, codes written),
// the chain of dependent loads for a token per sequence.

// rint(x / s), half to even, as if divided exactly, of four values, as bytes:
// c = rint(x * (1/s)) is off by one at most, next to a border; x - c s is exact
// (a multiple of ulp(s) below 2^24 of them), so its side of s / 2 settles it.
// s from 2^-100 on; below, the f64 quotient is far enough from any border that
// it does not hit.
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float s, float inv) {
  float c[4];
  if (s <= 0x1p-100f) {
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = s == 0.0f ? 0.0f : (float)rint((double)x[u] / (double)s);
  } else {
    const float h = 0.5f * s;
    float r[4], worst = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      c[u] = __builtin_rintf(x[u] * inv);
      r[u] = __builtin_fmaf(-c[u], s, x[u]);
      worst = fmaxf(worst, fabsf(r[u]));
    }
    if (worst >= h) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool odd = ((int)c[u] & 1) != 0;
        c[u] += (r[u] > h || (r[u] == h && odd)) ? 1.0f : (r[u] < -h || (r[u] == -h && odd)) ? -1.0f : 0.0f;
      }
    }
  }
  uint32_t w = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    w |= ((uint32_t)(int)__builtin_amdgcn_fmed3f(c[u], -127.0f, 127.0f) & 255u) << (8 * u);
  return w;
}

template <int HD, int P>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  constexpr int half = HD / 2;
  constexpr int IPT = HD / 8;                 // items per token
  constexpr int TPP = 256 / IPT;              // tokens per pass
  constexpr int NP = (P + TPP - 1) / TPP;     // passes
  constexpr int VST = P + 16;                 // bytes of a V column in LDS
  __shared__ __attribute__((aligned(16))) uint8_t vt[HD * VST];
  __shared__ uint32_t red[2][4];
  const Kv8Args &c = a.c;
  const int t = threadIdx.x, g = blockIdx.y, grp = c.nheads / c.nkv;
  const int nseq = (int)c.nseq;
  const SeqAt sq = find_seq(c.cu, c.len, nseq, c.rows, blockIdx.x, P, 2);
  const int i = sq.i, r0 = sq.r0, r1 = sq.r1, len = clamp_i(sq.len, 0, (int64_t)1 << 30);
  const int64_t b = (int64_t)blockIdx.x - seq_first_block(r0, i, P, 2);
  const int64_t pg = len / P + b;             // page of the sequence
  const int64_t p0 = pg * P;                  // its first position
  const int64_t ta = p0 > len ? p0 : len, tz = min(p0 + P, (int64_t)len + (r1 - r0));
  if (b < 0 || ta >= tz) return;              // (the whole block)
  const int e = (int)(ta - p0), z = (int)(tz - p0);   // new tokens of the page: [e, z)
  const int row0 = r0 + (int)(p0 - len);      // row of the page's token 0
  int id = pg < c.maxpages ? c.tab[(int64_t)i * c.maxpages + pg] : -1;
  id = page_or_none(id, (int)c.npages);
  uint8_t *page = c.pages + (int64_t)(id < 0 ? 0 : id) * kv8_page_bytes(P, c.nkv, HD);
  float *scale = reinterpret_cast<float *>(page + kv8_scales_at(P, c.nkv, HD));
  const float old0 = scale[g], old1 = scale[c.nkv + g];
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
  float s0[2], s1[2], inv[2];
  bool fine[2], grew[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t mx = max(max(red[x][0], red[x][1]), max(red[x][2], red[x][3]));
    const float am = __builtin_bit_cast(float, mx) * (1.0f / 127.0f);
    s0[x] = e > 0 ? (x ? old1 : old0) : 0.0f;
    s1[x] = am > s0[x] || am != am ? am : s0[x];          // (a NaN s0 stays)
    fine[x] = __builtin_isfinite(s1[x]);
    if (!fine[x]) s1[x] = __builtin_nanf("");
    grew[x] = e > 0 && fine[x] && s1[x] > s0[x];
    inv[x] = 1.0f / s1[x];
  }
  if (t < 2) scale[t * c.nkv + g] = s1[t];
  uint8_t *kc = page + (int64_t)g * P * HD, *vc = page + (int64_t)(c.nkv + g) * P * HD;
  // The old codes that stay around new ones in a V run of 16 tokens, or that
  // change: all loads go out together.
  constexpr int KI = (HD * P / 16 + 255) / 256;          // 16-byte runs per thread
  constexpr int RPC = P / 16;                            // runs of a V column
  u32x4 kold[KI], vold[KI];
#pragma unroll
  for (int u = 0; u < KI; ++u) {
    const int n = t + 256 * u, x = 16 * (n % RPC);
    if (grew[0] && n < e * (HD / 16)) kold[u] = *reinterpret_cast<const u32x4 *>(kc + 16 * n);
    if (n < HD * RPC && x < z && (x < e ? x + 16 > e || grew[1] : x + 16 > z))
      vold[u] = *reinterpret_cast<const u32x4 *>(vc + 16 * n);
  }
  // An old token's code at a larger scale: rint(c s0 / s1).  The f32 quotient is
  // within 127 2^-22 of it; next to a border the remainder decides, exact in f64
  // (c s0 and q s1 have 31 bits).
  float ratio[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) ratio[x] = grew[x] ? s0[x] / s1[x] : 1.0f;
  auto again = [&](uint32_t byte, int w) -> uint32_t {
    const float c = (float)(int8_t)byte, y = c * ratio[w];
    float q = __builtin_rintf(y);
    if (__builtin_fabsf(__builtin_fabsf(y - q) - 0.5f) < 1e-4f) {
      const double r = __builtin_fma(-(double)q, (double)s1[w], (double)c * (double)s0[w]);
      const double h = 0.5 * (double)s1[w];
      const bool odd = ((int)q & 1) != 0;
      q += (r > h || (r == h && odd)) ? 1.0f : (r < -h || (r == -h && odd)) ? -1.0f : 0.0f;
    }
    return (uint32_t)(int)q & 255u;
  };
  auto again4 = [&](uint32_t x, int w) -> uint32_t {
    return again(x & 255u, w) | again(x >> 8 & 255u, w) << 8 | again(x >> 16 & 255u, w) << 16 |
           again(x >> 24, w) << 24;
  };
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int tok = p * TPP + t / IPT;
    if (tok < e || tok >= z) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float k4[4] = {kx[p][4 * h], kx[p][4 * h + 1], kx[p][4 * h + 2], kx[p][4 * h + 3]};
      const float v4[4] = {vx[p][4 * h], vx[p][4 * h + 1], vx[p][4 * h + 2], vx[p][4 * h + 3]};
      const uint32_t kw = fine[0] ? codes4(k4, s1[0], inv[0]) : 0;
      const uint32_t vw = fine[1] ? codes4(v4, s1[1], inv[1]) : 0;
      *reinterpret_cast<uint32_t *>(kc + tok * HD + h * half + 4 * j) = kw;
#pragma unroll
      for (int u = 0; u < 4; ++u) vt[(h * half + 4 * j + u) * VST + tok] = (uint8_t)(vw >> (8 * u));
    }
  }
  if (grew[0]) {
#pragma unroll
    for (int u = 0; u < KI; ++u) {
      const int n = t + 256 * u;
      if (n >= e * (HD / 16)) continue;
#pragma unroll
      for (int x = 0; x < 4; ++x) kold[u][x] = again4(kold[u][x], 0);
      *reinterpret_cast<u32x4 *>(kc + 16 * n) = kold[u];
    }
  }
  __syncthreads();
  // V runs that hold a new token or an old one whose code changes; a run is one
  // thread's, which keeps what is around them
#pragma unroll
  for (int u = 0; u < KI; ++u) {
    const int n = t + 256 * u, x = 16 * (n % RPC);
    if (n >= HD * RPC || x >= z || (x + 16 <= e && !grew[1])) continue;
    u32x4 y = *reinterpret_cast<const u32x4 *>(&vt[(n / RPC) * VST + x]);
    if (x < e || x + 16 > z) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // bytes of tokens before e and from z on
        const int lo = min(max(e - x - 4 * i, 0), 4), hi = min(max(z - x - 4 * i, 0), 4);
        const uint32_t om = (uint32_t)((1ull << (8 * lo)) - 1);
        const uint32_t zm = ~(uint32_t)((1ull << (8 * hi)) - 1);
        const uint32_t o = grew[1] && lo > 0 ? again4(vold[u][i], 1) : vold[u][i];
        y[i] = (y[i] & ~(om | zm)) | (o & om) | (vold[u][i] & zm);
      }
    }
    *reinterpret_cast<u32x4 *>(vc + 16 * n) = y;
  }
}

// ---- attention -------------------------------------------------------------------
// out[column] = sum_t p_t vs[page(t)] vcode_t / sum_t p_t over the keys t that
// the column's row sees, p_t = exp(ks[page(t)] (q . kcode_t) / sqrt(HD) - max),
// a column being one (row, query head) of a KV head's group.
//
// Bound: HBM (2 HD bytes a key and KV head), as long as a tile's columns are
// few.  The units of work (64 keys of one sequence's row tile) of all sequences
// are laid end to end and cut into equal runs, one per wave of a KV head, so
// ragged contexts leave no wave behind (a row tile of 16 MT columns: one per MT
// waves, which go through the same keys side by side).  A wave streams its run through
// registers without a barrier: page ids are read two units ahead, codes one,
// across the ends of row tiles, so the loads never wait for a sum to be
// written.  A run that ends inside a row tile leaves a record for
// kv8_merge_kernel.  A few short tables take a block of 8 waves per row tile
// instead (WHOLE), which meet in LDS, and no merge.
//
// Scores: S^T = K Q^T on v_mfma_i32_16x16x64_i8 with the codes as they are and
// q as four signed base-256 digits of 2^30 q / 2^e (2^e the power of two above
// the column's largest |q|): exact integer sums, joined in f32, so q is carried
// to 2^-31 of the column's largest and nothing is lost in the sum.  That is an
// error of the score: the dims' roundings add up to at most sqrt(HD) 2^(e-31) of
// the largest |k|, and to 2^(e-31) / sqrt(3) of it in the mean square (6 times
// that is 6.6e-6 where 2^e |k| reaches 2^12).  Beyond 2^12, where dims that are
// many times the others meet codes near 0, a unit's scores are formed with q as
// three bf16 terms, which carry every dim as f32 does (beside dims 2^14 to 2^126
// times the others 3e-5 to 1 -> 6e-7 of float64; all units formed so: 64 sequences
// 67 -> 85 us, 4 contexts of up to 131000 tokens 122 -> 152).  Outputs:
// O^T += V^T P^T on v_mfma_f32_16x16x32_bf16, the codes as bf16 (exact) and
// p vs as three bf16 terms whose sum is the f32 value, whatever the scales.
// (Codes as bf16 in both products cost 192 more conversions of a unit's 700
// VALU operations, and 16 more matrix instructions.)
// Lane layout (lane l, g4 = l / 16), n = 16 (i8) or 8 (bf16) elements: A element
// i is A[l % 16][n g4 + i], B element i is B[n g4 + i][l % 16], accumulator
// element i is D[4 g4 + i][l % 16].  Which key is row r of score tile tt, and
// which dims are the elements of a step, is free: key 16 (r / 4) + 4 tt + r % 4
// makes the accumulators of a lane hold 16 consecutive keys of its column, the
// ones its V operand loads as one 16-byte run of a V column, and dims 64 h + 16
// g4 + i make its K operand one 16-byte run of a K row.
typedef int i32x4 __attribute__((ext_vector_type(4)));

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

// Four values' base-256 digits: byte i of digit k's word is digit k of x[i]
// (k = 3 the highest; digits 0 to 2 in [-128, 127]).
__device__ __forceinline__ void digits4(const float (&x)[4], uint32_t (&o)[4]) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = ((uint32_t)(int)__builtin_rintf(x[i]) + 0x00808080u) ^ 0x00808080u;
  const uint32_t a = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u);   // bytes 0, 1 of y0, y1
  const uint32_t b = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(y[1], y[0], 0x07030602u);   // bytes 2, 3
  const uint32_t d = __builtin_amdgcn_perm(y[3], y[2], 0x07030602u);
  o[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// The scale of a unit's integer scores, 2^(e - 30) ks log2(e) / sqrt(HD), up to
// which 2^e 127 ks <= 2^12.
template <int HD> __device__ __forceinline__ float kv8_exact_up_to() {
  return 1.44269504088896341f / sqrtf((float)HD) * (0x1p-18f / 127.0f);
}

// The four digits of a column's q (this lane's dims of it, x); returns the scale of the
// integer scores, 2^(e - 30) qscale, or NaN where q is not finite.
template <int HD>
__device__ __forceinline__ float kv8_digits(const float (&x)[HD / 64][16], float qscale,
                                            u32x4 (&qd)[4][HD / 64]) {
  constexpr int HH = HD / 64;
  uint32_t bits = 0;                      // |q| as bits: NaN and infinity above all
#pragma unroll
  for (int h = 0; h < HH; ++h)
#pragma unroll
    for (int v = 0; v < 16; ++v)
      bits = max(bits, __builtin_bit_cast(uint32_t, x[h][v]) & 0x7fffffffu);
  bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16));
  bits = max(bits, (uint32_t)__shfl_xor((int)bits, 32));
  const bool fine = bits < 0x7f800000u;
  const int e = max((int)(bits >> 23) - 126, -90);     // |q| < 2^e
  const float up = __builtin_ldexpf(1.0f, 30 - e);
#pragma unroll
  for (int h = 0; h < HH; ++h)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float y[4];
      uint32_t d[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) y[z] = fine ? x[h][4 * v + z] * up : 0.0f;
      digits4(y, d);
#pragma unroll
      for (int k = 0; k < 4; ++k) qd[k][h][v] = d[k];
    }
  return fine ? __builtin_ldexpf(qscale, e - 30) : __builtin_nanf("");
}

// The plan of a call in LDS: the prefix sums of the sequences' units (WHOLE: row
// tiles), pre[0] = 0 .. pre[nseq], and their first rows, row counts and cached
// tokens; all NT threads.
struct Kv8Plan {
  int *pre, *row0, *n, *old, *k0;
};

// What q8_kv8_share found: the group of each sequence (-1: none), the tokens that it
// takes from the group and the place of its first row in the list of rows; the groups'
// leaders, tokens and places of their rows; the list.  Read as if it could hold anything.
struct Kv8ShareAt {
  const int *group, *tok, *pos, *lead, *gtok, *gcu, *row;
  int groups;
};
Q8_HD int kv8_most_groups(int64_t nseq, int64_t rows) {
  const int64_t n = (nseq < rows ? nseq : rows) / 2;
  return (int)(n < kKv8ShareGroups ? n : kKv8ShareGroups);
}
__device__ __forceinline__ Kv8ShareAt kv8_share_at(const Kv8Args &c, const int *p) {
  const int64_t n = c.nseq;
  return {p + 1,         p + 1 + n,     p + 1 + 2 * n, p + 1 + 3 * n,
          p + 1 + 4 * n, p + 1 + 5 * n, p + 2 + 6 * n, clamp_i(p[0], 0, kv8_most_groups(n, c.rows))};
}
// Shared tokens as read: whole pages of what the table can hold.
__device__ __forceinline__ int kv8_tokens(const Kv8Args &c, int tok) {
  return clamp_i(tok, 0, c.maxpages * c.page) & ~(c.page - 1);
}
// Tokens of sequence i that its group's part of the attention covers (kept: the groups
// that have one).
__device__ __forceinline__ int kv8_shared_tokens(const Kv8Args &c, const Kv8ShareAt &sh, int i, uint64_t kept) {
  const int g = sh.group[i], tok = sh.tok[i];
  return g >= 0 && g < sh.groups && (kept >> g & 1) ? kv8_tokens(c, tok) : 0;
}
static_assert(kKv8ShareGroups <= 64, "a group a bit, a group a lane");

// What of a sequence a launch goes through: all its keys, or the ones behind the
// shared tokens.
enum { KV8_ALL = 0, KV8_OWN = 1 };

template <bool WHOLE, int NT, int PART>
__device__ __forceinline__ int kv8_plan(const Kv8Args &c, const int *share, uint64_t kept, int cols,
                                        const Kv8Plan &pl, int *wsum) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, nseq = (int)c.nseq;
  const int grp = c.nheads / c.nkv;
  int base = 0;
  if (t == 0) pl.pre[0] = 0;
  for (int i0 = 0; i0 < nseq; i0 += NT) {
    const int i = i0 + t;
    int u = 0;
    if (i < nseq) {
      const int a = c.cu[i];
      Kv8Seq s = kv8_seq(a, c.cu[i + 1], c.len[i], c.rows, c.maxpages * c.page, grp, cols);
      if (PART == KV8_OWN) {
        const int k0 = kv8_shared_tokens(c, kv8_share_at(c, share), i, kept);
        kv8_from(s, k0, c.maxpages * c.page);
        pl.k0[i] = k0;
      }
      u = WHOLE ? s.row_tiles : kv8_units_of(s);
      pl.row0[i] = clamp_i(a, 0, c.rows);
      pl.n[i] = s.n;
      pl.old[i] = s.old;
    }
    u = wave_scan(u, [](int a, int b) { return kv8_add(a, b); });
    if (lane == 63) wsum[w] = u;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int x = 0; x < NT / 64; ++x) {
      u = kv8_add(u, x < w ? wsum[x] : 0);
      all = kv8_add(all, wsum[x]);
    }
    if (i < nseq) pl.pre[i + 1] = kv8_add(base, u);
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

// Tables of up to this many units, and no more blocks of 8 waves than CUs (one fits a
// CU), take a block per row tile: the merge launch costs 4 us, a second round of
// blocks more (us whole / split: 1 sequence of 500 tokens, heads of 128 in groups
// of 4, 11.4 / 13.3, of 900 15.4 / 13.5; 32 of 700, 256 blocks, 14.7 / 22.8, 34 of
// 700, 272 blocks, 26.1 / 23.5; heads of 64 in groups of 16, 32 of 250 7.7 / 13.1,
// 48 17.1 / 14.4).
constexpr int kKv8WholeUnits = 12;
constexpr int kKv8WholeBlocks = 256;
constexpr int kKv8Waves = 4;              // waves of a block (WHOLE: 8)
constexpr int kKv8ShareCols = 16 * kKv8Waves;   // columns of a row tile of the shared tokens
constexpr int kKv8PlanSeq = 1024;         // sequences of a launch (16 KB of LDS for the plan)

// Record of a run and KV head: o[NC][HD] unnormalised, m[NC], l[NC] (of the
// columns that exist); slot 0 for a run that begins inside a row tile, slot 1
// for one that ends inside.
template <int HD, int NC> constexpr int kv8_record() { return NC * (HD + 2); }
// The prefix sums, behind the records of the call's runs.
template <int HD, int NC>
__device__ __forceinline__ int *kv8_plan_at(const Kv8AttnArgs &a, int runs) {
  return reinterpret_cast<int *>(a.ws + (int64_t)runs * a.c.nkv * 2 * kv8_record<HD, NC>());
}

// A place in a run of units: unit u of row tile rt of sequence i, its keys kt,
// the row tile's units of the run ending at t1.
struct Kv8Place {
  int u, i, rt, kt, t0, t1, units;       // units: the row tile's
  int ctx;                               // keys its last row sees
  int k0;                                // the first unit's first key
};

// The groups' part, a group a lane (whole waves): a block goes through `per` units at most
// of one row tile of a group, cut so that about `target` blocks have work.  The blocks of
// group g are base .. base + tiles * cuts - 1, its tiles' cuts one after the other.
// A call with a limit (kv8_share_room) keeps to `limit` blocks: fewer cuts where it must, and
// where row tiles alone are more, the first groups that fit.  Of its groups it takes those
// that save work: a row alone costs a wave a unit, a row tile kKv8Waves.  (32 KV heads of 128,
// two layers, us with groups / each sequence for itself, behind 400 and 2000 tokens: one group
// of 160 171 / 217, 205 / 728; 20 groups of 8 190 / 199, 343 / 603; 40 of 4 taken 253 / 203,
// 647 / 631, left out 233, 660; 64 of 2 taken 299 / 178, 798 / 549, left out 196, 566.)
// The others have no part (n = 0).
struct Kv8Groups {
  int lead, tokens, row0, n, units, cuts, base;
  int per, blocks;                       // the same in all lanes
  uint64_t kept;
};
__device__ __forceinline__ Kv8Groups kv8_groups(const Kv8Args &c, const Kv8ShareAt &sh, int target, int limit) {
  const int lane = threadIdx.x & 63, at = clamp_i(lane, 0, c.nseq - 1);
  Kv8Groups g;
  g.lead = clamp_i(sh.lead[at], 0, c.nseq - 1);
  g.tokens = kv8_tokens(c, sh.gtok[at]);
  g.row0 = clamp_i(sh.gcu[at], 0, c.rows);
  const int end = clamp_i(sh.gcu[at + 1], 0, c.rows);
  g.n = lane < sh.groups && end > g.row0 ? end - g.row0 : 0;
  g.units = (g.tokens + kKv8Unit - 1) / kKv8Unit;
  int64_t tiles = ((int64_t)g.n * (c.nheads / c.nkv) + kKv8ShareCols - 1) / kKv8ShareCols;
  if (limit < kKv8MaxUnits && g.n <= kKv8Waves * tiles) g.n = tiles = 0;
  const int64_t work = tiles * g.units;
  auto add = [](int a, int b) { return kv8_add(a, b); };
  const int all = __builtin_amdgcn_readlane(wave_scan(work < kKv8MaxUnits ? (int)work : kKv8MaxUnits, add), 63);
  int u;
  auto cut = [&](int target) {
    g.per = kv8_units_per_block(all, target, 1);
    g.cuts = (g.units + g.per - 1) / g.per;
    const int64_t blocks = tiles * g.cuts;
    const int mine = blocks < kKv8MaxUnits ? (int)blocks : kKv8MaxUnits;
    u = wave_scan(mine, add);
    g.base = u - mine;
    g.blocks = __builtin_amdgcn_readlane(u, 63);
  };
  cut(target);
  g.kept = ~(uint64_t)0;
  if (limit < kKv8MaxUnits) {
    if (g.blocks > limit)
      cut(kv8_fewer_blocks(limit, __builtin_amdgcn_readlane(
          wave_scan(tiles < kKv8MaxUnits ? (int)tiles : kKv8MaxUnits, add), 63)));
    if (u > limit) g.n = 0;              // (u ascends over the lanes)
    g.kept = __builtin_amdgcn_ballot_w64(g.n > 0);
    g.blocks = g.kept ? __builtin_amdgcn_readlane(u, 63 - __builtin_clzll(g.kept)) : 0;
  }
  return g;
}

// ---- the shared tokens of groups ------------------------------------------------------
// A block takes a row tile of 64 columns (row of the group, query head), 16 a wave, over
// a cut of the group's shared tokens; all columns see all of them.  A unit's K codes and
// its V, as bf16 once for all waves, go through LDS in the layout of the MFMA operands
// (a lane's 16 bytes side by side, no bank conflicts), the next unit's loads in flight
// beside this one's products.  Scores, probabilities and products are those of
// kv8_attn_kernel.
// Bound: instruction issue; VALU (the joins of the digits, exp, p in three terms) and
// MFMA (32 of int8, 48 of bf16 a unit and wave, heads of 128) take turns more than they
// overlap: 128 sequences of 4 heads a KV head behind 32000 tokens 195 us, 105 of VALU
// and 67-84 of MFMA by their counters, at 1.9 GHz.  (Eight waves over 128 columns, 4
// waves a SIMD: 279 us.)
template <int HD> __device__ __forceinline__ void kv8_shared_block(const Kv8AttnArgs &a) {
  constexpr int DT = HD / 16, HH = HD / 64, NC = kKv8ShareCols;
  constexpr int KF = 4 * HH / kKv8Waves, VF = DT / kKv8Waves;   // fragments that a wave stages
  __shared__ __attribute__((aligned(16))) u32x4 kbuf[2][4 * HH][64], vbuf[2][2 * DT][64];
  const Kv8Args &c = a.c;
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6), cc = 16 * w + col;
  const int g = blockIdx.y, grp = c.nheads / c.nkv, P = c.page;
  const int psh = 31 - __builtin_clz(P);
  const int64_t pbytes = kv8_page_bytes(P, c.nkv, HD);
  const int64_t scales_at = kv8_scales_at(P, c.nkv, HD);
  const int64_t k_at = (int64_t)g * P * HD, v_at = (int64_t)(c.nkv + g) * P * HD;
  const float qscale = 1.44269504088896341f / sqrtf((float)HD);
  const Kv8ShareAt sh = kv8_share_at(c, a.share);
  const Kv8Groups gs = kv8_groups(c, sh, a.shared_target, a.shared_limit);
  const int b = blockIdx.x;
  if (b >= gs.blocks) return;             // (the whole block)
  // the last group that begins at this block or before and has any
  const int i = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(gs.n > 0 && gs.cuts > 0 && gs.base <= b));
  const int lead = __builtin_amdgcn_readlane(gs.lead, i), tokens = __builtin_amdgcn_readlane(gs.tokens, i);
  const int n = __builtin_amdgcn_readlane(gs.n, i), row0 = __builtin_amdgcn_readlane(gs.row0, i);
  const int cuts = __builtin_amdgcn_readlane(gs.cuts, i), local = b - __builtin_amdgcn_readlane(gs.base, i);
  const int units = __builtin_amdgcn_readlane(gs.units, i);
  const int rt = local / cuts, t0 = local % cuts * gs.per, t1 = min(units, t0 + gs.per);
  const int *tab = c.tab + (int64_t)lead * c.maxpages;

  // what a wave stages: K fragments KF w .. (tt = f / HH, dims 64 (f % HH) + 16 g4 ..) and
  // V fragments VF w .. (dims 16 f + col, keys 16 g4 ..); the lane's pages of both
  int idk, idv;
  u32x4 kr[KF], vr[VF];
  float ks = 0.0f, vs = 0.0f, ks1, vs1;
  auto load_ids = [&](int kt) {
    const int kk = kt * kKv8Unit + 16 * (col >> 2), kv = kt * kKv8Unit + 16 * g4;
    idk = kt < t1 && kk < tokens ? tab[kk >> psh] : 0;
    idv = kt < t1 && kv < tokens ? tab[kv >> psh] : 0;
  };
  auto load = [&](int kt) {
    int id = page_or_none(idk, (int)c.npages);
    const uint8_t *p = c.pages + (id < 0 ? 0 : id) * pbytes + k_at +
                       (int64_t)(((kt * kKv8Unit + 16 * (col >> 2)) & (P - 1)) + (col & 3)) * HD + 16 * g4;
#pragma unroll
    for (int f = 0; f < KF; ++f)
      kr[f] = *reinterpret_cast<const u32x4 *>(p + 4 * ((KF * w + f) / HH) * HD + 64 * ((KF * w + f) % HH));
    id = page_or_none(idv, (int)c.npages);
    p = c.pages + (id < 0 ? 0 : id) * pbytes;
    const float *sc = reinterpret_cast<const float *>(p + scales_at);
    ks1 = id < 0 ? __builtin_nanf("") : sc[g];
    vs1 = id < 0 ? __builtin_nanf("") : sc[c.nkv + g];
    p += v_at + (int64_t)col * P + ((kt * kKv8Unit + 16 * g4) & (P - 1));
#pragma unroll
    for (int f = 0; f < VF; ++f) vr[f] = *reinterpret_cast<const u32x4 *>(p + (int64_t)16 * (VF * w + f) * P);
  };
  auto store = [&](int to) {
#pragma unroll
    for (int f = 0; f < KF; ++f) kbuf[to][KF * w + f][lane] = kr[f];
#pragma unroll
    for (int f = 0; f < VF; ++f)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        vbuf[to][2 * (VF * w + f) + e][lane] =
            __builtin_bit_cast(u32x4, codes_to_bf16(vr[f][2 * e], vr[f][2 * e + 1]));
    ks = ks1;
    vs = vs1;
  };
  load_ids(t0);
  load(t0);
  load_ids(t0 + 1);

  // this lane's digits of q
  const int lin = rt * NC + cc, j = lin / grp;
  const int row = clamp_i(sh.row[row0 + (j < n ? j : 0)], 0, c.rows - 1);
  const float *q = a.q + (int64_t)row * a.ldq + (int64_t)(g * grp + lin % grp) * HD + 16 * g4;
  u32x4 qd[4][HH];
  float qs;
  {
    float x[HH][16];
#pragma unroll
    for (int h = 0; h < HH; ++h)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const f32x4 y = *reinterpret_cast<const f32x4_u *>(q + 64 * h + 4 * v);
#pragma unroll
        for (int z = 0; z < 4; ++z) x[h][4 * v + z] = y[z];
      }
    qs = kv8_digits<HD>(x, qscale, qd);
  }
  store(0);
  __syncthreads();

  f32x4 o[DT];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kt = t0; kt < t1; ++kt) {
    const int at = (kt - t0) & 1;
    if (kt + 1 < t1) {
      load(kt + 1);
      load_ids(kt + 2);
    }
    f32x4 s[4];
    const float sc = qs * ks;
    __builtin_amdgcn_s_setprio(1);        // the matrix cores' work first, VALU beside it
    if (__builtin_amdgcn_ballot_w64(fabsf(sc) > kv8_exact_up_to<HD>()) == 0) {
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        i32x4 d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) d[k] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < HH; ++h) {
          const i32x4 kf = __builtin_bit_cast(i32x4, kbuf[at][tt * HH + h][lane]);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            d[k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, __builtin_bit_cast(i32x4, qd[k][h]), d[k], 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v)       // (|d| < 2^21 each: the pairs fit)
          s[tt][v] = __builtin_fmaf((float)((d[3][v] << 8) + d[2][v]), 65536.0f,
                                    (float)((d[1][v] << 8) + d[0][v]));
      }
    } else {
      // q as three bf16 terms (see kv8_attn_kernel)
      const float up = qscale / qs;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int z = 0; z < 2 * HH; ++z) {
        float y[8];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const f32x4 x = *reinterpret_cast<const f32x4_u *>(q + 64 * (z >> 1) + 8 * (z & 1) + 4 * v);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * v + e] = x[e] * up;
        }
        u32x4 qf[3];
        split3x8(y, qf);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const u32x4 kf = kbuf[at][tt * HH + (z >> 1)][lane];
          const bf16x8_t kb = codes_to_bf16(kf[2 * (z & 1)], kf[2 * (z & 1) + 1]);
#pragma unroll
          for (int k = 2; k >= 0; --k)
            s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb, __builtin_bit_cast(bf16x8_t, qf[k]), s[tt], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    // A lane's 16 keys are of one page, so its scores have one scale.  The last unit's keys
    // behind the shared tokens (a page of 16 or 32 may end there) are a path of their own.
    const int left = tokens - (kt * kKv8Unit + 16 * g4);        // this lane's keys, at most 16
    const bool masked = kt * kKv8Unit + kKv8Unit > tokens;
    float top = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) top = fmaxf(top, s[tt][v]);
    if (masked) {
      top = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int v = 0; v < 4; ++v) top = fmaxf(top, 4 * tt + v < left ? s[tt][v] : -INFINITY);
    }
    float tmax = top == -INFINITY ? top : top * sc;
    tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
    tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
    // (the maximum rounded to an integer, see kv8_attn_kernel)
    const float mnew = fmaxf(m, __builtin_rintf(tmax));
    const float ms = mnew == -INFINITY ? 0.0f : mnew;
    const float alpha = __builtin_amdgcn_exp2f(m - ms);
    m = mnew;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) s[tt][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][v], sc, -ms));
    float vsc = vs;
    if (masked) {
      // (a page of NaN scale counts for the rows that see one of its keys)
      if (left <= 0) vsc = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int v = 0; v < 4; ++v) s[tt][v] = 4 * tt + v < left ? s[tt][v] : 0.0f;
    }
    float ps = 0.0f;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int v = 0; v < 4; ++v) ps += s[tt][v];
    l = __builtin_fmaf(l, alpha, ps);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      u32x4 pf[3];
      float x[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) x[v] = s[2 * e + (v >> 2)][v & 3] * vsc;
      split3x8(x, pf);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += 4) {
        u32x4 va[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) va[d] = vbuf[at][2 * (d0 + d) + e][lane];
#pragma unroll
        for (int k = 2; k >= 0; --k)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            o[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, va[d]),
                                                                __builtin_bit_cast(bf16x8_t, pf[k]), o[d0 + d],
                                                                0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    // (the other buffer's last readers are behind the barrier before this unit)
    if (kt + 1 < t1) {
      store(at ^ 1);
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (j >= n) return;
  float *rec = a.shared_rec + ((int64_t)b * c.nkv + g) * kv8_record<HD, NC>();
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_u *>(rec + cc * HD + 16 * d + 4 * g4) = o[d];
  if (g4 == 0) {
    rec[NC * HD + cc] = m;
    rec[NC * HD + NC + cc] = l;
  }
}
template <int HD> __global__ __launch_bounds__(64 * kKv8Waves, 3) void kv8_shared_kernel(Kv8AttnArgs a) {
  kv8_shared_block<HD>(a);
}

// WIDE (pages of 128 tokens, runs): a V column of a page is one 128-byte line,
// of which a unit takes half.  The even unit's load brings the odd unit's half
// into registers too; fetched a unit later, the line had left the L2 by then
// (4 contexts of up to 131000 tokens 142 -> 128 us).
// PART: see above.
template <int HD, int MT, bool WHOLE, bool WIDE, int PART>
__global__ __launch_bounds__(WHOLE ? 512 : 64 * kKv8Waves, 2) void kv8_attn_kernel(Kv8AttnArgs a) {
  // the first blocks: the groups' part, if it has no launch of its own
  const int first = PART == KV8_OWN ? a.shared_first : 0, bx = (int)blockIdx.x - first;
  if constexpr (PART == KV8_OWN) {
    if (bx < 0) {
      kv8_shared_block<HD>(a);
      return;
    }
  }
  constexpr int DT = HD / 16, HH = HD / 64, NC = 16 * MT, NW = WHOLE ? 8 : kKv8Waves;
  constexpr int RW = NW / MT;             // runs of a block
  constexpr int OST = HD + 4;             // floats of a column's sums in LDS
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  // WHOLE: the sums of four waves; the plan behind them
  float *ob = reinterpret_cast<float *>(lds);
  constexpr int kOBytes = WHOLE ? (RW / 2) * NC * OST * 4 : 0;
  __shared__ int wsum[NW];
  __shared__ float wm[RW][NC], wl[RW][NC];
  const Kv8Args &c = a.c;
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6) / MT;    // run of the block
  const int cc = 16 * (__builtin_amdgcn_readfirstlane(t >> 6) % MT) + col;   // this lane's column
  const int g = blockIdx.y, grp = c.nheads / c.nkv, nseq = (int)c.nseq, P = c.page;
  const int psh = 31 - __builtin_clz(P);  // page = 2^psh
  const int cap = (int)(c.maxpages * P);
  const int64_t pbytes = kv8_page_bytes(P, c.nkv, HD);
  const int64_t scales_at = kv8_scales_at(P, c.nkv, HD);
  const int64_t k_at = (int64_t)g * P * HD, v_at = (int64_t)(c.nkv + g) * P * HD;
  const float qscale = 1.44269504088896341f / sqrtf((float)HD);
  Kv8Plan pl;
  pl.pre = reinterpret_cast<int *>(lds + kOBytes);
  pl.row0 = pl.pre + nseq + 1;
  pl.n = pl.row0 + nseq;
  pl.old = pl.n + nseq;
  pl.k0 = pl.old + nseq;

  uint64_t kept = ~(uint64_t)0;           // groups that have a part of their own
  if constexpr (PART == KV8_OWN) {
    if (a.shared_limit < kKv8MaxUnits)
      kept = kv8_groups(c, kv8_share_at(c, a.share), a.shared_target, a.shared_limit).kept;
  }
  const int units = kv8_plan<WHOLE, 64 * NW, PART>(c, a.share, kept, NC, pl, wsum);
  const int runs = ((int)gridDim.x - first) * RW, run = bx * RW + w;
  const int per = WHOLE ? 1 : kv8_units_per_block(units, runs, 1);
  // the merge reads the plan behind the records
  if (!WHOLE && bx == 0 && g == 0)
    for (int i = t; i <= nseq; i += 64 * NW) kv8_plan_at<HD, NC>(a, runs)[i] = pl.pre[i];
  const int u0 = WHOLE ? bx : run * per;
  const int uend = WHOLE ? min(bx + 1, units) : min(u0 + per, units);
  if (u0 >= uend) return;                 // (WHOLE: the whole block)

  // the place of unit u, in sequence i or behind it
  auto place = [&](int u, int i) {
    Kv8Place p;
    while (pl.pre[i + 1] <= u) ++i;
    const int local = u - pl.pre[i], ctx = min(pl.old[i] + pl.n[i], cap);
    p.k0 = PART == KV8_OWN ? pl.k0[i] : 0;
    p.units = (ctx - p.k0 + kKv8Unit - 1) / kKv8Unit;
    p.u = u;
    p.i = i;
    p.ctx = ctx;
    p.rt = WHOLE ? local : local / p.units;
    p.t0 = p.kt = WHOLE ? 0 : local % p.units;
    p.t1 = WHOLE ? p.units : min(p.units, p.t0 + (uend - u));
    return p;
  };

  // The unit that is loaded next; its page ids are there already.  Lanes of a
  // unit's 16-key groups: K rows by col / 4, V columns by g4; page 0 stands
  // behind the context (those keys are masked).
  u32x4 kr[4][HH], vr[DT], vr2[WIDE ? DT : 1];
  float ks = 0.0f, vs = 0.0f;
  int idk = 0, idv = 0;
  bool second = false;                    // vr2 holds the V of the unit loaded next
  const int step = WHOLE ? RW : 1;
  Kv8Place nx = place(u0, kv8_seq_of(pl.pre, nseq, u0));
  Kv8Place cu = nx;
  if (WHOLE) nx.kt = w;
  auto have = [&]() { return nx.kt < nx.t1; };
  auto load_ids = [&]() {
    if (!have()) return;
    const int *tab = c.tab + (int64_t)nx.i * c.maxpages;
    const int kk = nx.k0 + nx.kt * kKv8Unit + 16 * (col >> 2), kv = nx.k0 + nx.kt * kKv8Unit + 16 * g4;
    idk = kk < nx.ctx ? tab[kk >> psh] : 0;
    idv = kv < nx.ctx ? tab[kv >> psh] : 0;
  };
  auto load_k = [&]() {
    if (!have()) return;
    const int id = page_or_none(idk, (int)c.npages);
    const uint8_t *p = c.pages + (id < 0 ? 0 : id) * pbytes + k_at +
                       (int64_t)(((nx.k0 + nx.kt * kKv8Unit + 16 * (col >> 2)) & (P - 1)) + (col & 3)) * HD +
                       16 * g4;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int h = 0; h < HH; ++h)
        kr[tt][h] = *reinterpret_cast<const u32x4 *>(p + 4 * tt * HD + 64 * h);
  };
  auto load_v = [&]() {
    if (!have()) return;
    if (WIDE && second) {                 // (an even unit of the same page came before it)
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[d] = vr2[WIDE ? d : 0];
      second = false;
      return;
    }
    const int id = page_or_none(idv, (int)c.npages);
    const uint8_t *base = c.pages + (id < 0 ? 0 : id) * pbytes;
    const float *sc = reinterpret_cast<const float *>(base + scales_at);
    ks = id < 0 ? __builtin_nanf("") : sc[g];
    vs = id < 0 ? __builtin_nanf("") : sc[c.nkv + g];
    const uint8_t *p = base + v_at + (int64_t)col * P + ((nx.k0 + nx.kt * kKv8Unit + 16 * g4) & (P - 1));
    // non-temporal where a load takes whole lines (64 sequences, pages of 64
    // tokens, 71 -> 67 us; with WIDE's two loads a line 124 -> 132)
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const u32x4 *q = reinterpret_cast<const u32x4 *>(p + (int64_t)16 * d * P);
      vr[d] = WIDE ? *q : __builtin_nontemporal_load(q);
    }
    if (WIDE && (nx.kt & 1) == 0 && nx.kt + 1 < nx.t1) {
      second = true;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        vr2[WIDE ? d : 0] = *reinterpret_cast<const u32x4 *>(p + (int64_t)16 * d * P + kKv8Unit);
    }
  };
  auto advance = [&]() {
    nx.kt += step;
    if (WHOLE || nx.kt < nx.t1) return;
    const int u = nx.u + (nx.t1 - nx.t0);
    if (u < uend) nx = place(u, nx.i);
  };
  // q of this lane's column of a row tile (one that does not exist: the first
  // row's), from dim 16 g4 on
  auto q_at = [&](const Kv8Place &p, int row0, int n) {
    const int lin = p.rt * NC + cc, j = lin / grp;
    return a.q + (int64_t)(row0 + (j < n ? j : 0)) * a.ldq + (int64_t)(g * grp + lin % grp) * HD + 16 * g4;
  };
  load_ids();
  load_k();
  load_v();
  advance();
  load_ids();

  for (;;) {                              // row tiles of the run
    const int row0 = pl.row0[cu.i], n = pl.n[cu.i], old = pl.old[cu.i];
    // ---- this lane's digits of q: column col, dims 64 h + 16 g4 ..; the keys
    // its columns see: 0 .. kend-1 (0: no such column)
    const int lin = cu.rt * NC + cc, j = lin / grp;
    const int kend = j < n ? min(old + j + 1, cap) : 0;
    int kmin = j < n ? kend : INT32_MAX;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) kmin = min(kmin, __shfl_xor(kmin, d));
    u32x4 qd[4][HH];
    float qs;                             // score = ks qs (256^3 d3 + 256^2 d2 + 256 d1 + d0)
    {
      float x[HH][16];
#pragma unroll
      for (int h = 0; h < HH; ++h) {
        const float *q = q_at(cu, row0, n) + 64 * h;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const f32x4 y = *reinterpret_cast<const f32x4_u *>(q + 4 * v);
#pragma unroll
          for (int z = 0; z < 4; ++z) x[h][4 * v + z] = y[z];
        }
      }
      qs = kv8_digits<HD>(x, qscale, qd);
    }

    // ---- the wave's units
    f32x4 o[DT];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int kt = WHOLE ? w : cu.t0; kt < cu.t1; kt += step) {
      f32x4 s[4];
      const float sc = qs * ks, vsc = vs;
      if (__builtin_amdgcn_ballot_w64(fabsf(sc) > kv8_exact_up_to<HD>()) == 0) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          i32x4 d[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            d[k] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int h = 0; h < HH; ++h)
              d[k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, kr[tt][h]),
                                                           __builtin_bit_cast(i32x4, qd[k][h]), d[k], 0,
                                                           0, 0);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v)     // (|d| < 2^21 each: the pairs fit)
            s[tt][v] = __builtin_fmaf((float)((d[3][v] << 8) + d[2][v]), 65536.0f,
                                      (float)((d[1][v] << 8) + d[0][v]));
        }
      } else {
        // step 2 h + x: dims 64 h + 16 g4 + 8 x .. of both operands; q at the integer
        // scores' scale (2^30 / 2^e, exactly), so that no product overflows
        const float up = qscale / qs;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const float *q = q_at(cu, row0, n);
#pragma unroll
        for (int z = 0; z < 2 * HH; ++z) {
          float y[8];
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const f32x4 a = *reinterpret_cast<const f32x4_u *>(q + 64 * (z >> 1) + 8 * (z & 1) + 4 * v);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * v + i] = a[i] * up;
          }
          u32x4 qf[3];
          split3x8(y, qf);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            const bf16x8_t kb = codes_to_bf16(kr[tt][z >> 1][2 * (z & 1)], kr[tt][z >> 1][2 * (z & 1) + 1]);
#pragma unroll
            for (int k = 2; k >= 0; --k)
              s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb, __builtin_bit_cast(bf16x8_t, qf[k]),
                                                              s[tt], 0, 0, 0);
          }
        }
      }
      load_k();
      const int key0 = cu.k0 + kt * kKv8Unit + 16 * g4;
      const bool masked = cu.k0 + kt * kKv8Unit + kKv8Unit > kmin;
      float tmax = -INFINITY;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float x = s[tt][v] * sc;
          if (masked) x = key0 + 4 * tt + v < kend ? x : -INFINITY;
          s[tt][v] = x;
          tmax = fmaxf(tmax, x);
        }
      tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
      tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
      // the maximum rounded to an integer: alpha is a power of two, and 1 for
      // most units
      const float mnew = fmaxf(m, __builtin_rintf(tmax));
      const float ms = mnew == -INFINITY ? 0.0f : mnew;
      const float alpha = __builtin_amdgcn_exp2f(m - ms);
      m = mnew;
      float ps = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float p = __builtin_amdgcn_exp2f(s[tt][v] - ms);
          ps += p;
          // (a page of NaN scale counts for the rows that see one of its keys)
          float x = p * vsc;
          if (masked) x = key0 + 4 * tt + v < kend ? x : 0.0f;
          s[tt][v] = x;
        }
      l = __builtin_fmaf(l, alpha, ps);
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= alpha;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4 pf[3];
        float x[8];
#pragma unroll
        for (int v = 0; v < 8; ++v) x[v] = s[2 * e + (v >> 2)][v & 3];
        split3x8(x, pf);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const bf16x8_t va = codes_to_bf16(vr[d][2 * e], vr[d][2 * e + 1]);
#pragma unroll
          for (int k = 0; k < 3; ++k)
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, __builtin_bit_cast(bf16x8_t, pf[k]), o[d],
                                                           0, 0, 0);
        }
      }
      load_v();
      advance();
      load_ids();
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    if (WHOLE) {                          // the runs of the row tile meet
      if (g4 == 0) {
        wm[w][cc] = m;
        wl[w][cc] = l;
      }
      __syncthreads();
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < RW; ++x) mx = fmaxf(mx, wm[x][cc]);
      const float ms = mx == -INFINITY ? 0.0f : mx;
      l = 0.0f;
#pragma unroll
      for (int x = 0; x < RW; ++x) l = __builtin_fmaf(wl[x][cc], __builtin_amdgcn_exp2f(wm[x][cc] - ms), l);
      const float f = __builtin_amdgcn_exp2f(m - ms);
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
      // (a run without units adds zeros; the order of the sum is fixed)
      for (int half = RW / 2; half > 0; half >>= 1) {
        f32x4 *at = reinterpret_cast<f32x4 *>(ob + ((w % half) * NC + cc) * OST + 4 * g4);
        if (w >= half && w < 2 * half) {
#pragma unroll
          for (int d = 0; d < DT; ++d) at[4 * d] = o[d];
        }
        __syncthreads();
        if (w < half) {
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] += at[4 * d];
        }
        __syncthreads();
      }
      if (w != 0) return;
    }
    if (j < n) {
      const bool whole = WHOLE || (cu.t0 == 0 && cu.t1 == cu.units);
      float *rec = a.ws + (((int64_t)run * c.nkv + g) * 2 + (cu.t0 == 0)) * kv8_record<HD, NC>();
      // (as it is where the join with the group's part follows)
      const float il = whole && !(PART == KV8_OWN && cu.k0 > 0) ? 1.0f / l : 1.0f;
      float *out = whole ? a.out + ((int64_t)(row0 + j) * c.nheads + g * grp + lin % grp) * HD
                         : rec + cc * HD;
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_u *>(out + 16 * d + 4 * g4) = o[d] * il;
      if (!whole && g4 == 0) {
        rec[NC * HD + cc] = m;
        rec[NC * HD + NC + cc] = l;
      }
      if (PART == KV8_OWN && whole && g4 == 0) {      // (for the join with the group's part)
        float *ml = a.ml + 2 * ((int64_t)(row0 + j) * c.nheads + g * grp + lin % grp);
        ml[0] = m;
        ml[1] = l;
      }
    }
    const int u = cu.u + (cu.t1 - cu.t0);
    if (WHOLE || u >= uend) return;
    cu = place(u, cu.i);
  }
}

// Joins the records of the row tiles that several runs served: grid
// (rows, nkv, heads of a group / hb).  The block's threads are groups over hb
// heads x HD / 4 dims; the groups take the records in turn and meet in LDS.
// PART KV8_OWN: also joins the group's records (and the output as it stands, where
// one run served the row).
template <int HD, int MT, int PART>
__global__ __launch_bounds__(512) void kv8_merge_kernel(Kv8AttnArgs a, int runs, int hb) {
  constexpr int NC = 16 * MT, NT = 512;
  __shared__ __attribute__((aligned(16))) float so[NT * 4];
  __shared__ float sm[NT], sl[NT];
  const Kv8Args &c = a.c;
  const int g = blockIdx.y, grp = c.nheads / c.nkv, nseq = (int)c.nseq;
  const int row = blockIdx.x, t = threadIdx.x;
  const int *pre = kv8_plan_at<HD, NC>(a, runs);
  const int per = kv8_units_per_block(pre[nseq], runs, 1);
  // a sequence a lane, where that is all of them, beside the search below: its group, the
  // tokens it takes from it and its place there
  Kv8ShareAt sh;
  Kv8Groups gs;
  int group = -1, pos = 0, shared = 0, unit0 = 0;
  auto load = [&](int i) {
    group = sh.group[i];
    pos = sh.pos[i];
    shared = kv8_shared_tokens(c, sh, i, gs.kept);
    unit0 = pre[i];
  };
  if constexpr (PART == KV8_OWN) {
    sh = kv8_share_at(c, a.share);
    gs = kv8_groups(c, sh, a.shared_target, a.shared_limit);
    if (nseq <= 64) load(min(t & 63, nseq - 1));
  }
  // the sequence of this row: the last one that begins at it or before
  const SeqAt at = find_seq(c.cu, c.len, nseq, c.rows, row, 1, 0);
  const int lo = at.i, j = row - at.r0;
  Kv8Seq sq = kv8_seq(at.r0, at.r1, at.len, c.rows, c.maxpages * c.page, grp, NC);
  // the group's records of this row: cuts of them, from block `cut0` on
  int cuts = 0, cut0 = 0, place = 0;
  if constexpr (PART == KV8_OWN) {
    const int from = nseq <= 64 ? lo : 0;
    if (nseq > 64) load(lo);
    group = __builtin_amdgcn_readlane(group, from);
    pos = __builtin_amdgcn_readlane(pos, from);
    unit0 = __builtin_amdgcn_readlane(unit0, from);
    shared = __builtin_amdgcn_readlane(shared, from);
    kv8_from(sq, shared, c.maxpages * c.page);
    if (shared == 0) group = -1;
    if (group >= 0) {
      cuts = __builtin_amdgcn_readlane(gs.cuts, group);
      cut0 = __builtin_amdgcn_readlane(gs.base, group);
      place = clamp_i((int64_t)pos + j - __builtin_amdgcn_readlane(gs.row0, group), 0,
                      max(0, __builtin_amdgcn_readlane(gs.n, group) - 1));
    }
  } else {
    unit0 = pre[lo];
  }
  if (j < 0 || j >= sq.n) return;             // behind the last sequence
  constexpr int IPH = HD / 4;
  const int sg = NT / (hb * IPH);             // groups of threads
  const int grp_id = t / (hb * IPH), item = t % (hb * IPH);
  {
    const int hh = blockIdx.z * hb + item / IPH, d = 4 * (item % IPH);
    const int lin = j * grp + hh, rt = lin / NC, cc = lin % NC;
    const int64_t ua = unit0 + (int64_t)rt * sq.key_units;
    const int b0 = clamp_i(ua / per, 0, runs - 1);
    const int b1 = clamp_i((ua + sq.key_units - 1) / per, 0, runs - 1);
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    // (b0 == b1: written whole)
    const bool on = grp_id < sg && hh < grp && (b0 != b1 || (PART == KV8_OWN && group >= 0));
    if constexpr (PART == KV8_OWN) {
      if (on && group >= 0) {
        // the group's cuts, then the row's own run where it has one (three at a time: four
        // take more than 64 registers)
        const int slin = place * grp + hh;
        constexpr int cols = kKv8ShareCols;
        const int64_t first = (int64_t)cut0 + (int64_t)(slin / cols) * cuts;
        const int all = cuts + (b0 == b1 && sq.key_units > 0);
        const int64_t h = (int64_t)row * c.nheads + g * grp + hh;
        for (int z0 = grp_id; z0 < all; z0 += 3 * sg) {
          float zm[3], zl[3];
          f32x4 zo[3];
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            const int z = z0 + x * sg < all ? z0 + x * sg : z0;
            const int64_t rb = min(first + z, (int64_t)a.shared_blocks - 1);
            const float *r = a.shared_rec + (rb * c.nkv + g) * kv8_record<HD, cols>();
            const bool rec = z < cuts;
            zm[x] = rec ? r[cols * HD + slin % cols] : a.ml[2 * h];
            zl[x] = rec ? r[cols * HD + cols + slin % cols] : a.ml[2 * h + 1];
            zo[x] = *reinterpret_cast<const f32x4_u *>(rec ? r + slin % cols * HD + d : a.out + h * HD + d);
          }
          float mx = m;
#pragma unroll
          for (int x = 0; x < 3; ++x) mx = fmaxf(mx, zm[x]);
          const float ms = mx == -INFINITY ? 0.0f : mx;
          const float f0 = __builtin_amdgcn_exp2f(m - ms);
          l *= f0;
          o *= f0;
#pragma unroll
          for (int x = 0; x < 3; ++x) {
            if (z0 + x * sg >= all) continue;
            const float f = __builtin_amdgcn_exp2f(zm[x] - ms);
            l = __builtin_fmaf(f, zl[x], l);
#pragma unroll
            for (int v = 0; v < 4; ++v) o[v] = __builtin_fmaf(f, zo[x][v], o[v]);
          }
          m = mx;
        }
      }
    }
    for (int z0 = b0 + grp_id; on && b0 != b1 && z0 <= b1; z0 += 4 * sg) {
      float zm[4], zl[4];
      f32x4 zo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int z = z0 + x * sg <= b1 ? z0 + x * sg : z0;
        const float *r = a.ws + (((int64_t)z * c.nkv + g) * 2 + (z == b0)) * kv8_record<HD, NC>();
        zm[x] = r[NC * HD + cc];
        zl[x] = r[NC * HD + NC + cc];
        zo[x] = *reinterpret_cast<const f32x4 *>(r + cc * HD + d);
      }
      float mx = m;
#pragma unroll
      for (int x = 0; x < 4; ++x) mx = fmaxf(mx, z0 + x * sg <= b1 ? zm[x] : -INFINITY);
      const float ms = mx == -INFINITY ? 0.0f : mx;
      const float f0 = __builtin_amdgcn_exp2f(m - ms);
      l *= f0;
      o *= f0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (z0 + x * sg > b1) continue;
        const float f = __builtin_amdgcn_exp2f(zm[x] - ms);
        l = __builtin_fmaf(f, zl[x], l);
#pragma unroll
        for (int v = 0; v < 4; ++v) o[v] = __builtin_fmaf(f, zo[x][v], o[v]);
      }
      m = mx;
    }
    sm[t] = m;
    sl[t] = l;
    *reinterpret_cast<f32x4 *>(so + 4 * t) = o;
    __syncthreads();
    if (grp_id != 0 || !on) return;
    // groups of threads that took any
    const int with = min(sg, max(b1 - b0, PART == KV8_OWN && group >= 0 ? cuts : 0) + 1);
    float mx = m;
#pragma unroll 4
    for (int x = 1; x < with; ++x) mx = fmaxf(mx, sm[x * hb * IPH + item]);
    const float ms = mx == -INFINITY ? 0.0f : mx;
    const float f0 = __builtin_amdgcn_exp2f(m - ms);
    l *= f0;
    o *= f0;
#pragma unroll 2
    for (int x = 1; x < with; ++x) {
      const int y = x * hb * IPH + item;
      const float f = __builtin_amdgcn_exp2f(sm[y] - ms);
      l = __builtin_fmaf(f, sl[y], l);
#pragma unroll
      for (int v = 0; v < 4; ++v) o[v] = __builtin_fmaf(f, so[4 * y + v], o[v]);
    }
    const float il = 1.0f / l;
    *reinterpret_cast<f32x4_u *>(a.out + ((int64_t)row * c.nheads + g * grp + hh) * HD + d) = o * il;
  }
}

template <int HD, int MT, int PART>
hipError_t launch_kv8_attn_t(const Kv8AttnArgs &a, hipStream_t st) {
  constexpr int NC = 16 * MT, RW = kKv8Waves / MT;
  const Kv8Args &c = a.c;
  const int grp = c.nheads / c.nkv;
  const size_t plan = (size_t)((PART == KV8_OWN ? 5 : 4) * c.nseq + 1) * 4;
  // a sequence of n rows has ceil(n grp / NC) row tiles: no more than each row alone
  // would, nor than n grp / NC and one
  const int64_t tiles = std::min(c.rows * ((grp + NC - 1) / NC), c.rows * grp / NC + c.nseq);
  const int64_t key_units = (c.maxpages * c.page + kKv8Unit - 1) / kKv8Unit;
  if (PART == KV8_ALL && key_units <= kKv8WholeUnits && tiles * c.nkv <= kKv8WholeBlocks) {
    const size_t lds = (size_t)(8 / MT / 2) * NC * (HD + 4) * 4 + plan;
    hipLaunchKernelGGL((kv8_attn_kernel<HD, MT, true, false, KV8_ALL>), dim3((unsigned)tiles, (unsigned)c.nkv),
                       dim3(512), lds, st, a);
    return hipGetLastError();
  }
  // two blocks per CU over all KV heads (one beside the groups' blocks), as far as the
  // work (by its bound) and the records' space reach
  const int first = PART == KV8_OWN ? a.shared_first : 0;
  int64_t nb = ((first ? 256 : 512) + c.nkv - 1) / c.nkv;
  nb = std::min(nb, (tiles * key_units + RW - 1) / RW);
  nb = std::min(nb, (a.ws_floats - c.nseq - 1) / (RW * 2 * (int64_t)c.nkv * kv8_record<HD, NC>()));
  if (nb < 1) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(nb + first), (unsigned)c.nkv), block(64 * kKv8Waves);
  if (c.page == 128)
    hipLaunchKernelGGL((kv8_attn_kernel<HD, MT, false, true, PART>), grid, block, plan, st, a);
  else
    hipLaunchKernelGGL((kv8_attn_kernel<HD, MT, false, false, PART>), grid, block, plan, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // few rows: more blocks, with more groups of threads over a row's records
  int hb = std::min(grp, 512 / (HD / 4));
  while (hb > 1 && c.rows * c.nkv * ((grp + hb - 1) / hb) < 256) hb = (hb + 1) / 2;
  hipLaunchKernelGGL((kv8_merge_kernel<HD, MT, PART>),
                     dim3((unsigned)c.rows, (unsigned)c.nkv, (unsigned)((grp + hb - 1) / hb)),
                     dim3(512), 0, st, a, (int)(nb * RW), hb);
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

template <int MT>
static hipError_t launch_kv8_cols(const Kv8AttnArgs &a, hipStream_t st) {
  return a.c.head_dim == 64 ? launch_kv8_attn_t<64, MT, KV8_ALL>(a, st)
                            : launch_kv8_attn_t<128, MT, KV8_ALL>(a, st);
}

hipError_t launch_kv8_attention(const Kv8AttnArgs &a, hipStream_t st) {
  // row tiles of 16, 32 or 64 columns, as the sequences' rows fill them on
  // average (a tile's keys are read once)
  const int64_t cols = a.c.rows * (a.c.nheads / a.c.nkv);
  for (int64_t i = 0; i < a.c.nseq; i += kKv8PlanSeq) {
    Kv8AttnArgs p = a;
    p.c.cu += i;
    p.c.len += i;
    p.c.tab += i * a.c.maxpages;
    p.c.nseq = std::min<int64_t>(kKv8PlanSeq, a.c.nseq - i);
    const hipError_t e = cols <= 16 * a.c.nseq   ? launch_kv8_cols<1>(p, st)
                         : cols <= 32 * a.c.nseq ? launch_kv8_cols<2>(p, st)
                                                 : launch_kv8_cols<4>(p, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// The groups' part (a row tile of 64 columns cut over blocks), each sequence's own
// part, and the merge that joins them.  Little work in the groups (units of row tiles and
// KV heads) takes one launch with the sequences' parts.  The rule goes by what the tables can
// hold, not by what they do: a launch is sized without the arrays, so that a captured one fits
// all of them, and a table with room to spare takes two launches.  One is a launch less,
// but two blocks a CU where alone it has three (us together / apart, 8 KV heads: 64
// sequences of 500 tokens behind 8000, heads of 128, 128 / 137; 64 behind 8000 with
// pages of 128 73 / 72, behind 16000 98 / 90; 128 behind 32000 252 / 227; heads of 64:
// 8 behind 1000, four layers, 70 / 97, 128 behind 8000 76 / 81, behind 16000 114 / 113,
// behind 32000 188 / 177).
template <int HD> constexpr int64_t kKv8TogetherUnits = HD == 64 ? 16000 : 6000;
template <int HD> static hipError_t launch_kv8_shared_t(Kv8AttnArgs a, hipStream_t st) {
  const Kv8Args &c = a.c;
  constexpr int NC = kKv8ShareCols;
  const int64_t grp = c.nheads / c.nkv, cols = c.rows * grp;
  const int64_t groups = kv8_most_groups(c.nseq, c.rows);
  const int64_t tiles = cols / NC + groups, rec = c.nkv * kv8_record<HD, NC>();
  // maxima and sums per (row, head), the groups' records, then the sequences' own parts (a
  // block of these, whose runs have two records of all columns, at least)
  const int64_t ml = (2 * c.rows * c.nheads + 3) / 4 * 4;
  const int64_t units = (c.maxpages * c.page + kKv8Unit - 1) / kKv8Unit * ((cols + NC - 1) / NC) * c.nkv;
  const bool together = units <= kKv8TogetherUnits<HD>;
  // as many blocks as are resident
  const int64_t want = ((together ? 512 : 768) + c.nkv - 1) / c.nkv;
  const Kv8Room room = kv8_share_room(a.ws_floats, ml, rec, 2 * rec, c.nseq + 1, (512 + c.nkv - 1) / c.nkv,
                                      (cols + NC - 1) / NC, tiles, want);
  // (more rows than there is room for: every sequence for itself)
  if (room.blocks == 0 || groups == 0) return launch_kv8_attention(a, st);
  const int64_t blocks = room.blocks, recs = blocks * rec;
  a.shared_target = room.target;
  a.shared_limit = room.limit;
  a.ml = a.ws;
  a.shared_rec = a.ws + ml;
  a.shared_blocks = (int)blocks;
  // (blocks that leave at once would only be in the way of the sequences' own: 64 groups of 2
  // rows, see kv8_groups, 745 / 573 us in one launch / in two)
  a.shared_first = together && room.limit == kKv8MaxUnits ? (int)blocks : 0;
  a.ws += ml + recs;
  a.ws_floats -= ml + recs;
  if (a.shared_first == 0) {
    hipLaunchKernelGGL(kv8_shared_kernel<HD>, dim3((unsigned)blocks, (unsigned)c.nkv), dim3(64 * kKv8Waves), 0, st,
                       a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return cols <= 16 * c.nseq   ? launch_kv8_attn_t<HD, 1, KV8_OWN>(a, st)
         : cols <= 32 * c.nseq ? launch_kv8_attn_t<HD, 2, KV8_OWN>(a, st)
                               : launch_kv8_attn_t<HD, 4, KV8_OWN>(a, st);
}

hipError_t launch_kv8_attention_shared(const Kv8AttnArgs &a, hipStream_t st) {
  return a.c.head_dim == 64 ? launch_kv8_shared_t<64>(a, st) : launch_kv8_shared_t<128>(a, st);
}

}  // namespace q8
