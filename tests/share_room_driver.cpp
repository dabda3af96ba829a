// The space of a call with shared prefixes (csrc/q8_ragged.h): what the groups' records and
// the sequences' own parts take fits, and a call's groups keep to the blocks that they have.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../lama32_mojo_amd/csrc/q8_ragged.h"

using namespace q8;

#define CHECK(x)                                                     \
  do {                                                               \
    if (!(x)) {                                                      \
      std::printf("line %d: %s (nkv %lld rows %lld nseq %lld)\n",    \
                  __LINE__, #x, nkv, rows, nseq);                    \
      std::exit(1);                                                  \
    }                                                                \
  } while (0)

int main() {
  std::mt19937 rng(1);
  const long long ws = 16777216;
  long long limited = 0, dropped = 0, none = 0;
  for (int i = 0; i < 40000; ++i) {
    long long nkv = 1 + rng() % 512, grp = 1 + rng() % 8, hd = rng() % 2 ? 64 : 128;
    if (rng() % 2) nkv = 1 << rng() % 10;
    const long long nseq = 1 + rng() % 1024, rows = nseq + (rng() % 4 ? 0 : rng() % 3000);
    const long long cols = rows * grp, rec = nkv * 64 * (hd + 2), ml = (2 * rows * nkv * grp + 3) / 4 * 4;
    const long long one = (cols + 63) / 64, groups = std::min<long long>(std::min(nseq, rows) / 2, 64);
    const long long most = cols / 64 + groups, want = ((rng() % 2 ? 512 : 768) + nkv - 1) / nkv;
    const long long own = 2 * rec, plan = nseq + 1, nb = (512 + nkv - 1) / nkv;
    const Kv8Room r = kv8_share_room(ws, ml, rec, own, plan, nb, one, most, want);
    if (r.blocks == 0) {
      // there is no room for all rows' tiles and 8 cuts beside the blocks of the others
      CHECK(ml + (one + std::min<long long>(want, 8)) * rec + nb * own + plan > ws);
      ++none;
      continue;
    }
    CHECK(ml + r.blocks * rec + own + plan <= ws);
    CHECK(r.limit == kKv8MaxUnits ? ml + r.blocks * rec <= ws / 4 * 3 : ml + r.blocks * rec + nb * own + plan <= ws);
    CHECK(r.target >= 1 && r.target <= want && r.target <= r.blocks && r.blocks >= one);
    CHECK(r.limit == kKv8MaxUnits ? r.blocks == r.target + most && r.target >= std::min<long long>(want, 8)
                                  : r.limit == r.blocks);
    // groups of some of the rows
    std::vector<long long> tiles, units;
    long long left = rows, all = 0, t = 0;
    for (long long g = 0; g < groups && left > 1; ++g) {
      const long long n = g == 0 && rng() % 2 ? left : 2 + rng() % std::max<long long>(1, std::min(left - 1, rows / groups * 2));
      tiles.push_back((std::min(n, left) * grp + 63) / 64);
      units.push_back(rng() % 3 ? 1 + rng() % 40 : rng() % 3000);
      left -= std::min(n, left);
      all += tiles.back() * units.back();
      t += tiles.back();
    }
    CHECK(t <= most);
    auto blocks = [&](int target) {
      const int per = kv8_units_per_block(all, target, 1);
      long long b = 0;
      for (size_t g = 0; g < tiles.size(); ++g) b += tiles[g] * ((units[g] + per - 1) / per);
      return b;
    };
    long long b = blocks(r.target);
    if (r.limit == kKv8MaxUnits) CHECK(b <= r.blocks);
    if (b > r.limit) {
      ++limited;
      b = blocks(kv8_fewer_blocks(r.limit, (int)t));
      if (t <= r.limit) CHECK(b <= r.limit);
      else ++dropped;
      if (tiles.size() == 1) CHECK(b <= r.limit);
    }
  }
  long long nkv = 0, rows = 0, nseq = 0;
  CHECK(limited > 100 && dropped > 100 && none > 100);
  // 78 to 1024 sequences of 32 heads of 128
  nkv = 32;
  for (rows = nseq = 78; rows <= 1024; rows = nseq = rows + 1) {
    const long long rec = 32 * 64 * 130, one = (rows + 63) / 64;
    const Kv8Room r = kv8_share_room(ws, 64 * rows, rec, 2 * rec, rows + 1, 16, one, rows / 64 + std::min<long long>(64, rows / 2), 24);
    CHECK(r.blocks >= one + 8 && r.target >= 8);
  }
  std::puts("ok");
  return 0;
}
