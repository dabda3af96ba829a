// Host check of the units of work of csrc/q8_ragged.h.  Well-formed calls: every
// unit in one run at each column count, and the records that runs leave.  Offsets
// that hold nonsense: the prefix sums of a cache attention call (the block's scan,
// step by step), the search for a unit's sequence and the place within it, with
// offsets out of order whose sums pass 2^30; every row tile, column and row that a
// block would serve has to lie inside its sequence.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../lama32_mojo_amd/csrc/q8_ragged.h"

using namespace q8;

#define CHECK(x)                                                     \
  do {                                                               \
    if (!(x)) {                                                      \
      std::printf("line %d: %s\n", __LINE__, #x);                    \
      std::exit(1);                                                  \
    }                                                                \
  } while (0)

// Inclusive sums over a block of nt threads, in waves of 64: doubling steps in a
// wave, then the waves before it.
static std::vector<int> block_sums(std::vector<int> u, int &all) {
  const int nt = (int)u.size();
  for (int d = 1; d < 64; d <<= 1)
    for (int t = nt - 1; t >= 0; --t)
      if ((t & 63) >= d) u[t] = kv8_add(u[t], u[t - d]);
  std::vector<int> wsum;
  for (int w = 0; w < nt / 64; ++w) wsum.push_back(u[64 * w + 63]);
  all = 0;
  for (int s : wsum) all = kv8_add(all, s);
  for (int t = 0; t < nt; ++t)
    for (int x = 0; x < t / 64; ++x) u[t] = kv8_add(u[t], wsum[x]);
  return u;
}

static void call(const std::vector<int> &cu, const std::vector<int> &len, int64_t rows, int64_t cap,
                 int grp, int cols, int nt, std::mt19937 &rng) {
  const int nseq = (int)len.size();
  std::vector<Kv8Seq> sq;
  for (int i = 0; i < nseq; ++i) sq.push_back(kv8_seq(cu[i], cu[i + 1], len[i], rows, cap, grp, cols));
  std::vector<int> pre(1, 0);
  int base = 0;
  for (int i0 = 0; i0 < nseq; i0 += nt) {
    std::vector<int> u(nt, 0);
    for (int t = 0; t < nt && i0 + t < nseq; ++t) u[t] = kv8_units_of(sq[i0 + t]);
    int all;
    u = block_sums(u, all);
    for (int t = 0; t < nt && i0 + t < nseq; ++t) pre.push_back(kv8_add(base, u[t]));
    base = kv8_add(base, all);
  }
  const int units = base;
  CHECK(units >= 0 && units <= kKv8MaxUnits && pre[nseq] == units);
  for (int i = 0; i < nseq; ++i) CHECK(pre[i + 1] >= pre[i]);
  for (int runs : {1, 7, 256, 2048}) {
    const int per = kv8_units_per_block(units, runs, 1);
    CHECK(per >= 1);
    for (int n = 0; n < 40; ++n) {
      const int64_t run = n < 2 ? (n ? runs - 1 : 0) : (int64_t)(rng() % (unsigned)runs);
      const int64_t u0 = run * per, uend = u0 + per < units ? u0 + per : units;
      CHECK(u0 + per <= INT32_MAX);
      if (u0 >= uend) continue;
      for (int64_t u : {u0, uend - 1, u0 + (int64_t)(rng() % (unsigned)(uend - u0))}) {
        int i = 0, hi = nseq;
        while (hi - i > 1) {
          const int m = (i + hi) >> 1;
          if (pre[m] <= u) i = m;
          else hi = m;
        }
        while (pre[i + 1] <= u) CHECK(++i < nseq);
        const int local = (int)u - pre[i];
        CHECK(local >= 0 && sq[i].key_units > 0);
        const int rt = local / sq[i].key_units;
        CHECK(rt >= 0 && rt < sq[i].row_tiles);
        for (int cc : {0, cols - 1}) {
          const int64_t lin = (int64_t)rt * cols + cc, j = lin / grp;
          CHECK(lin <= INT32_MAX);
          const int64_t row0 = clamp_i(cu[i], 0, rows);
          if (j < sq[i].n) CHECK(row0 + j < rows);
        }
      }
    }
  }
}

// A well-formed call: every (row tile, 64 keys) in one run, records where the merge
// looks for them, none written twice.
static void cover(const std::vector<int> &cu, const std::vector<int> &len, int64_t rows, int64_t cap,
                  int grp, int cols, int runs) {
  const int nseq = (int)len.size();
  std::vector<Kv8Seq> sq;
  std::vector<int> pre(1, 0);
  int64_t tiles = 0;
  for (int i = 0; i < nseq; ++i) {
    sq.push_back(kv8_seq(cu[i], cu[i + 1], len[i], rows, cap, grp, cols));
    pre.push_back(kv8_add(pre.back(), kv8_units_of(sq[i])));
    tiles += sq[i].row_tiles;
  }
  // the bounds that launches are sized by
  CHECK(tiles <= rows * ((grp + cols - 1) / cols) && tiles <= rows * grp / cols + nseq);
  const int units = pre.back(), per = kv8_units_per_block(units, runs, 1);
  std::vector<int> seen(units, 0);
  for (int r = 0; r < runs; ++r) {
    int slots[2] = {0, 0}, i = 0;
    for (int64_t u = (int64_t)r * per, uend = u + per < units ? u + per : units; u < uend;) {
      while (pre[i + 1] <= u) ++i;
      const int ku = sq[i].key_units, rt = ((int)u - pre[i]) / ku, t0 = ((int)u - pre[i]) % ku;
      const int t1 = ku < t0 + uend - u ? ku : (int)(t0 + uend - u);
      CHECK(rt < sq[i].row_tiles && t1 > t0);
      for (int t = t0; t < t1; ++t) ++seen[u + t - t0];
      const int ua = pre[i] + rt * ku, b0 = ua / per, b1 = (ua + ku - 1) / per;
      CHECK((t0 == 0 && t1 == ku) == (b0 == b1));
      if (b0 != b1) {
        CHECK((t0 == 0) == (r == b0));
        CHECK(++slots[t0 == 0] == 1);
      }
      u += t1 - t0;
    }
  }
  for (int v : seen) CHECK(v == 1);
}

int main() {
  std::mt19937 rng(11);
  for (int round = 0; round < 200; ++round) {
    std::vector<int> cu(1, 0), len;
    for (int i = 0, nseq = 1 + (int)(rng() % 90u), most = 1 + (int)(rng() % 40u); i < nseq; ++i) {
      cu.push_back(cu.back() + (rng() % 5u ? (int)(rng() % (unsigned)most) : 0));
      len.push_back((int)(rng() % 900u));
    }
    for (int cols : {16, 32, 64})
      for (int runs : {1, 5, 64, 2048})
        cover(cu, len, cu.back() + (int)(rng() % 9u), 16 * (1 + (int)(rng() % 64u)), 1 + (int)(rng() % 70u),
              cols, runs);
  }
  for (int a : {0, 1, kKv8MaxUnits / 2, kKv8MaxUnits - 1, kKv8MaxUnits})
    for (int b : {0, 1, kKv8MaxUnits / 2, kKv8MaxUnits - 1, kKv8MaxUnits}) {
      const int64_t s = (int64_t)a + b;
      CHECK(kv8_add(a, b) == (s < kKv8MaxUnits ? s : kKv8MaxUnits));
    }
  // every second sequence with nearly all the units that a call may have
  for (int nseq : {2, 18, 63, 64, 65, 400, 1024}) {
    const int64_t rows = 1 << 20, cap = 256000;
    std::vector<int> cu(1, 0), len;
    for (int i = 0; i < nseq; ++i) {
      cu.push_back(i % 2 ? 0 : (int)rows);
      len.push_back((int)cap);
    }
    for (int nt : {256, 512})
      for (int cols : {16, 32, 64}) call(cu, len, rows, cap, 4, cols, nt, rng);
  }
  for (int round = 0; round < 300; ++round) {
    const int nseq = 1 + (int)(rng() % 1024u), grp = 1 + (int)(rng() % 9u);
    const int64_t rows = 1 + (int64_t)(rng() % (1u << (rng() % 21u))), cap = 16 * (1 + (int64_t)(rng() % 20000u));
    std::vector<int> cu, len;
    for (int i = 0; i <= nseq; ++i) cu.push_back(rng() & 1 ? (int)rng() : (int)(rng() % (unsigned)(rows + 1)));
    for (int i = 0; i < nseq; ++i) len.push_back((int)rng());
    call(cu, len, rows, cap, grp, 16 << (rng() % 3u), rng() & 1 ? 256 : 512, rng);
  }
  std::printf("ok\n");
  return 0;
}
