// Host check of csrc/q8_ragged.h: which blocks of a call over several sequences
// serve which rows, pages and units of work, for random ragged calls.
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

// The kernels' search: the last i with seq_first_block(cu[i], i) <= b, 64
// candidates a step.
static int find_seq(const std::vector<int> &cu, int nseq, int64_t rows, int64_t b, int tile,
                    int spare) {
  int lo = 0, n = nseq;
  while (n > 1) {
    const int step = (n + 63) / 64;
    int k = 0;
    for (int lane = 0; lane < 64; ++lane) {
      const int i = lo + lane * step;
      CHECK((i < nseq ? i : nseq - 1) >= 0);
      if (lane * step < n &&
          seq_first_block(clamp_i(cu[i < nseq ? i : nseq - 1], 0, rows), i, tile, spare) <= b)
        k = lane;
    }
    n = n - k * step < step ? n - k * step : step;
    lo += k * step;
  }
  CHECK(lo >= 0 && lo < nseq);
  return lo;
}

int main() {
  std::mt19937 rng(7);
  auto draw = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
  for (int round = 0; round < 400; ++round) {
    const int nseq = round % 7 == 0 ? draw(65, 300) : draw(1, 40);
    const int most = round % 3 ? draw(0, 40) : draw(0, 700);
    std::vector<int> cu(1, 0), len;
    for (int i = 0; i < nseq; ++i) {
      cu.push_back(cu.back() + (draw(0, 4) ? draw(0, most) : 0));
      len.push_back(draw(0, 500));
    }
    const int64_t rows = cu.back() + draw(0, 50);
    // row tiles of the packed attention
    for (int tile : {1, 3, 16, 32, 128}) {
      std::vector<int> seen(rows, 0);
      for (int64_t b = 0; b < seq_blocks(rows, nseq, tile, 1); ++b) {
        const int i = find_seq(cu, nseq, rows, b, tile, 1);
        const int64_t t = b - seq_first_block(cu[i], i, tile, 1);
        if (t < 0) continue;
        for (int64_t r = t * tile; r < (t + 1) * tile && r < cu[i + 1] - cu[i]; ++r) ++seen[cu[i] + r];
      }
      for (int r = 0; r < cu.back(); ++r) CHECK(seen[r] == 1);
      for (int64_t r = cu.back(); r < rows; ++r) CHECK(seen[r] == 0);
    }
    // pages that the append touches
    for (int page : {16, 32, 64, 128}) {
      std::vector<int> seen(rows, 0);
      for (int64_t b = 0; b < seq_blocks(rows, nseq, page, 2); ++b) {
        const int i = find_seq(cu, nseq, rows, b, page, 2);
        const int64_t k = b - seq_first_block(cu[i], i, page, 2);
        const int64_t p0 = (len[i] / page + k) * page;
        const int64_t a = p0 > len[i] ? p0 : len[i], n = cu[i + 1] - cu[i];
        const int64_t z = p0 + page < len[i] + n ? p0 + page : len[i] + n;
        if (k < 0) continue;
        for (int64_t t = a; t < z; ++t) ++seen[cu[i] + t - len[i]];
      }
      for (int r = 0; r < cu.back(); ++r) CHECK(seen[r] == 1);
    }
    // units of the cache attention: every (row tile, 64 keys) in one run of one
    // block, records where the merge looks for them
    for (int cols : {16, 32})
      for (int nblocks : {1, 5, 64}) {
        const int grp = draw(1, 9), page = 16 << draw(0, 3);
        const int64_t cap = (int64_t)page * draw(1, 40);
        std::vector<int> pre(1, 0);
        std::vector<Kv8Seq> sq;
        for (int i = 0; i < nseq; ++i) {
          sq.push_back(kv8_seq(cu[i], cu[i + 1], len[i], rows, cap, grp, cols));
          CHECK((sq[i].n == 0) == (sq[i].row_tiles == 0));
          CHECK(sq[i].n == 0 || sq[i].key_units >= 1);
          CHECK((int64_t)sq[i].key_units * 64 < cap + 64);
          pre.push_back(pre.back() + sq[i].row_tiles * sq[i].key_units);
        }
        const int units = pre.back(), per = kv8_units_per_block(units, nblocks, 4);
        std::vector<int> seen(units, 0);
        for (int b = 0; b < nblocks; ++b) {
          int slots[2] = {0, 0};
          int u = b * per, uend = u + per < units ? u + per : units;
          while (u < uend) {
            int i = 0;
            while (i + 1 < nseq && pre[i + 1] <= u) ++i;
            const int local = u - pre[i], rt = local / sq[i].key_units, t0 = local % sq[i].key_units;
            const int t1 = sq[i].key_units < t0 + uend - u ? sq[i].key_units : t0 + uend - u;
            CHECK(rt < sq[i].row_tiles && t1 > t0);
            for (int t = t0; t < t1; ++t) ++seen[u + t - t0];
            const int ua = pre[i] + rt * sq[i].key_units, b0 = ua / per,
                      b1 = (ua + sq[i].key_units - 1) / per;
            const bool whole = t0 == 0 && t1 == sq[i].key_units;
            CHECK(whole == (b0 == b1));
            if (!whole) {
              CHECK((t0 == 0) == (b == b0));       // the merge's slot
              CHECK(++slots[t0 == 0] == 1);        // no record written twice
            }
            u += t1 - t0;
          }
        }
        for (int v : seen) CHECK(v == 1);
      }
  }
  // arrays that hold nonsense: still inside the buffers
  for (int round = 0; round < 200; ++round) {
    const int nseq = draw(1, 90);
    const int64_t rows = draw(1, 300), cap = 16 * draw(1, 50);
    std::vector<int> cu;
    for (int i = 0; i <= nseq; ++i) cu.push_back((int)rng());
    for (int64_t b = 0; b < seq_blocks(rows, nseq, 32, 1); ++b) find_seq(cu, nseq, rows, b, 32, 1);
    for (int i = 0; i < nseq; ++i) {
      const Kv8Seq s = kv8_seq(cu[i], cu[i + 1], (int)rng(), rows, cap, 4, 16);
      CHECK(s.n >= 0 && s.n <= rows && s.old >= 0 && s.old <= cap && s.row_tiles <= (rows * 4 + 15) / 16);
      CHECK((int64_t)s.key_units * kKv8Unit < cap + kKv8Unit);
    }
  }
  CHECK(page_or_none(-1, 5) == -1 && page_or_none(5, 5) == -1 && page_or_none(4, 5) == 4);
  CHECK(page_or_none(INT32_MIN, 5) == -1 && page_or_none(INT32_MAX, 5) == -1 && page_or_none(0, 1) == 0);
  CHECK(kv8_page_bytes(16, 1, 64) == 2 * 16 * 64 + 16 && kv8_page_bytes(64, 8, 128) == 131072 + 64);
  std::printf("ok\n");
  return 0;
}
