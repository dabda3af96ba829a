// q8_ragged.h -- index arithmetic of calls over several sequences (host and
// device; no HIP types, so that a CPU program can check it).
//
// Sequence i of a call has the rows cu[i] .. cu[i+1]-1 of its packed arrays.
// The offsets live on the device and the host knows only their number and the
// last one's bound, so launches are sized by upper bounds and every block
// finds its own sequence.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define Q8_HD __host__ __device__ __forceinline__
#else
#define Q8_HD inline
#endif

namespace q8 {

// First block of sequence i in a launch that gives each sequence enough
// blocks of `tile` rows: cu / tile + spare * i.  Consecutive sequences of n
// rows lie at least n / tile + spare apart, so spare = 1 covers ceil(n / tile)
// tiles and spare = 2 the n rows of tiles that start inside one
// (kv8 pages: ceil(n / tile) + 1 at most, and one for the rounding of cu).
Q8_HD int64_t seq_first_block(int cu, int i, int tile, int spare) {
  return (int64_t)(cu / tile) + (int64_t)spare * i;
}
// Blocks of the whole launch.
Q8_HD int64_t seq_blocks(int64_t rows, int64_t nseq, int tile, int spare) {
  return rows / tile + spare * nseq;
}

Q8_HD int clamp_i(int64_t v, int64_t lo, int64_t hi) {
  return (int)(v < lo ? lo : v > hi ? hi : v);
}

// A page id as read from a table: itself if it names a page, else -1.
Q8_HD int page_or_none(int id, int npages) { return id >= 0 && id < npages ? id : -1; }

// Pages that n tokens take.
Q8_HD int pages_of(int64_t n, int page) { return (int)((n + page - 1) / page); }

// Bytes of a cache page: K codes [nkv][page][hd], V codes [nkv][hd][page],
// nkv K scales and nkv V scales (f32), padded to 16 bytes.
Q8_HD int64_t kv8_scales_at(int page, int nkv, int hd) { return 2 * (int64_t)nkv * page * hd; }
Q8_HD int64_t kv8_page_bytes(int page, int nkv, int hd) {
  return kv8_scales_at(page, nkv, hd) + (8 * (int64_t)nkv + 15) / 16 * 16;
}

// The work of a cache attention call: units of 64 keys, counted over
// sequences and, within one, over its row tiles of `cols` (row, query head)
// columns.  Run r of the call (a wave's, or of as many waves as a row tile has
// 16-column parts) serves the units [r * per, (r + 1) * per).
constexpr int kKv8Unit = 64;
struct Kv8Seq {
  int n, old, row_tiles, key_units;
};
Q8_HD Kv8Seq kv8_seq(int cu0, int cu1, int len, int64_t rows, int64_t cap, int grp, int cols) {
  Kv8Seq s;
  const int a = clamp_i(cu0, 0, rows), b = clamp_i(cu1, 0, rows);
  s.n = b > a ? b - a : 0;
  s.old = clamp_i(len, 0, cap);
  const int64_t ctx = (int64_t)s.old + s.n < cap ? (int64_t)s.old + s.n : cap;
  s.row_tiles = (int)(((int64_t)s.n * grp + cols - 1) / cols);
  s.key_units = s.n ? (int)((ctx + kKv8Unit - 1) / kKv8Unit) : 0;
  return s;
}
// The unit counts are summed up to this (arrays that hold nonsense cannot make
// them overflow; a call that could reach it is refused).
constexpr int kKv8MaxUnits = 1 << 30;
Q8_HD int kv8_units_of(const Kv8Seq &s) {
  const int64_t u = (int64_t)s.row_tiles * s.key_units;
  return u < kKv8MaxUnits ? (int)u : kKv8MaxUnits;
}
// (of counts from 0 to the limit; two at the limit would not fit an int32)
Q8_HD int kv8_add(int a, int b) { return a < kKv8MaxUnits - b ? a + b : kKv8MaxUnits; }
// Units of each of nruns runs; at least `least` (the kernels': 1), so a small call
// uses fewer of them.
Q8_HD int kv8_units_per_block(int64_t units, int nruns, int least) {
  const int64_t per = ((int64_t)units + nruns - 1) / nruns;
  return (int)(per < least ? least : per);
}

}  // namespace q8
