// q8_pages.hip -- the pages of a cache: allocation with copies of shared pages,
// forks, lengths and release, compaction.
//
// State, all int32 on the device: tab[nslots][maxpages] page ids (-1 behind a
// slot's held pages), len[nslots] tokens, held[nslots] pages, ref[npages] how
// many table entries name a page (0: free).  No free list: a free page is one
// that nobody names, and pages are handed out from the lowest id up, so the
// result of every call depends on its inputs alone.  Counts change through
// integer atomics, whose order does not matter.
//
// What bounds these calls: the copies of page contents are HBM-bound (a page
// is read and written once per layer); everything else is a few KB of int32,
// where the launches and the round trips of dependent reads count.
#include "q8_launch.h"
#include "q8_ragged.h"

namespace q8 {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kSlotsPerThread = kPagesMaxSlots / kScanThreads;

// Exclusive sum over the block's threads in thread order; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int *wsum, int *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  if (lane == 63) wsum[w] = s;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int x = 0; x < kScanThreads / 64; ++x) {
    const int t = wsum[x];
    base += x < w ? t : 0;
    all += t;
  }
  __syncthreads();
  *total = all;
  return base + s - v;
}

// Four consecutive reference counts from p on (1 past the end: not free).
__device__ __forceinline__ void refs4(const int *ref, int64_t p, int64_t npages, int (&r)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) r[u] = p + u < npages ? ref[p + u] : 1;
}

// Free pages as a wave reads them: bit r of a lane is page first + 64 r + lane,
// r < rows <= 32.  The loads are coalesced, and independent within a group of 8.
__device__ __forceinline__ uint32_t free_pages(const int *ref, int64_t first, int rows,
                                               int64_t npages) {
  const int lane = threadIdx.x & 63;
  uint32_t bits = 0;
  for (int r0 = 0; r0 < rows; r0 += 8) {
    int v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t p = first + 64 * (r0 + r) + lane;
      v[r] = r0 + r < rows && p < npages ? ref[p] : 1;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) bits |= (uint32_t)(v[r] == 0) << (r0 + r);
  }
  return bits;
}
// Free pages of the wave.
__device__ __forceinline__ int count_free(uint32_t bits, int rows) {
  int n = 0;
  for (int r = 0; r < rows; ++r) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(bits >> r & 1u));
  return n;
}
constexpr int kList = 4096;

// The pages of a slot that growing from len to want tokens writes to and that
// other slots name too: places len / page .. to pages_of(want) of what it holds.
// visit(place, id) for each, in order; returns their number.
template <class F>
__device__ __forceinline__ int shared_pages(const PagesArgs &a, int s, int len, int want, int held,
                                            F visit) {
  int n = 0;
  if (want <= len) return 0;
  const int to = min(held, pages_of(want, a.page));
  for (int j = len / a.page; j < to; ++j) {
    const int id = page_or_none(a.tab[(int64_t)s * a.maxpages + j], (int)a.npages);
    if (id >= 0 && a.ref[id] > 1) {
      if (visit(j, id, n)) return n + 1;
      ++n;
    }
  }
  return n;
}

// One block.  Slots in ascending order ask for the pages they lack and for one
// in the place of each shared page they are to write to (the first of which may
// be partly filled: its contents are copied); an exclusive sum of the needs
// gives each slot a run of ranks, and the free page of rank r, found by a second
// sum over the pages, goes to the slot whose run holds r.  When the free pages
// do not reach, the slots behind the last run that fits get nothing.  ws: the
// number of copies and (from, to) pairs, at most one per slot; behind them the
// pages replaced as (table entry, old, new).  Bound: the chain length, page id, reference count, sums; the
// free pages are looked up beside it.
__global__ __launch_bounds__(kScanThreads) void pages_reserve_kernel(PagesArgs a,
                                                                     const int *__restrict__ want,
                                                                     int *__restrict__ ws) {
  __shared__ int off[kPagesMaxSlots + 1];
  __shared__ int cow[kPagesMaxSlots];          // shared pages replaced
  __shared__ int list[kList];
  __shared__ int wsum[kScanThreads / 64];
  __shared__ int ncopy, nswap, granted_end;
  int *copies = ws, *swaps = ws + 1 + 2 * a.nslots;
  const int t = threadIdx.x, wave = t >> 6;
  const int64_t cap = a.maxpages * a.page;
  if (t == 0) ncopy = nswap = granted_end = 0;
  // pages in goes of 16 waves x rows x 64; the first go's counts are in flight
  // beside the slots' reads
  const int rows = (int)(a.npages < 32 * kScanThreads ? (a.npages + kScanThreads - 1) / kScanThreads : 32);
  const int64_t go = (int64_t)rows * kScanThreads;
  const int64_t first = (int64_t)64 * rows * wave;
  uint32_t bits = free_pages(a.ref, first, rows, a.npages);
  int need[kSlotsPerThread], mine = 0;
#pragma unroll
  for (int u = 0; u < kSlotsPerThread; ++u) {
    const int s = t * kSlotsPerThread + u;
    need[u] = 0;
    if (s >= a.nslots) continue;
    const int len = clamp_i(a.len[s], 0, cap), w = clamp_i(want[s], 0, cap);
    const int held = clamp_i(a.held[s], 0, a.maxpages);
    const int c = shared_pages(a, s, len, w, held, [](int, int, int) { return false; });
    cow[s] = c;
    const int more = pages_of(w, a.page) - held;
    need[u] = (more > 0 ? more : 0) + c;
    mine += need[u];
  }
  int total, at = block_scan(mine, wsum, &total);
  if (total == 0) {
    if (t == 0) copies[0] = 0;
    return;
  }
#pragma unroll
  for (int u = 0; u < kSlotsPerThread; ++u) {
    const int s = t * kSlotsPerThread + u;
    if (s < a.nslots) off[s] = at;
    at += need[u];
  }
  if (t == 0) off[a.nslots] = total;
  // free pages: as many as are needed, or all there are
  // (of the first go: rank of the wave's first free page, and how many there are)
  int nfree = 0, base0 = 0, got0 = 0;
  for (int64_t p0 = 0; p0 < a.npages && nfree < total; p0 += go) {
    const int n = count_free(p0 ? free_pages(a.ref, p0 + first, rows, a.npages) : bits, rows);
    int got;
    const int r = block_scan((t & 63) == 0 ? n : 0, wsum, &got);
    if (p0 == 0) {
      base0 = __builtin_amdgcn_readfirstlane(r);
      got0 = got;
    }
    nfree += got;
  }
  int end = 0;
#pragma unroll
  for (int u = 0; u < kSlotsPerThread; ++u) {
    const int s = t * kSlotsPerThread + u;
    if (s < a.nslots && need[u] > 0 && off[s] + need[u] <= nfree) end = off[s] + need[u];
  }
  if (end) atomicMax(&granted_end, end);
  __syncthreads();
  // The free pages' ids by rank, kList at a time in LDS, then a thread per rank.
  const int take = granted_end;
  int done = 0;                               // ranks handed out
  for (int64_t p0 = 0, run = 0; p0 < a.npages && run < take; p0 += go) {
    int got = got0, base = base0;
    if (p0) {
      bits = free_pages(a.ref, p0 + first, rows, a.npages);
      const int n = count_free(bits, rows);
      base = (int)run + __builtin_amdgcn_readfirstlane(block_scan((t & 63) == 0 ? n : 0, wsum, &got));
    }
    run += got;
    const int upto = (int)(run < take ? run : take);
    while (done < upto) {
      const int stop = done + kList < upto ? done + kList : upto;
      int rank = base;
      for (int r = 0; r < rows && rank < stop; ++r) {
        const uint64_t m = __builtin_amdgcn_ballot_w64(bits >> r & 1u);
        const int at = rank + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                                            __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if ((bits >> r & 1u) && at >= done && at < stop)
          list[at - done] = (int)(p0 + first + 64 * r) + (t & 63);
        rank += __builtin_popcountll(m);
      }
      __syncthreads();
      for (int x = t; x < stop - done; x += kScanThreads) {
        int lo = 0, hi = (int)a.nslots;       // the slot with off[lo] <= rank < off[lo + 1]
        while (hi - lo > 1) {
          const int m = (lo + hi) >> 1;
          if (off[m] <= done + x) lo = m;
          else hi = m;
        }
        const int id = list[x], k = done + x - off[lo];
        int *row = a.tab + (int64_t)lo * a.maxpages;
        const int held = clamp_i(a.held[lo], 0, a.maxpages);
        if (k < cow[lo]) {                    // the k-th shared page
          const int len = clamp_i(a.len[lo], 0, cap);
          int place = 0, was = 0;
          shared_pages(a, lo, len, clamp_i(want[lo], 0, cap), held, [&](int j, int old, int n) {
            place = j;
            was = old;
            return n == k;
          });
          if (place == len / a.page && len % a.page != 0) {
            const int y = atomicAdd(&ncopy, 1);
            copies[1 + 2 * y] = was;
            copies[2 + 2 * y] = id;
          }
          // entered below, once no thread counts a row's shared pages any more
          int *e = swaps + 3 * (int64_t)atomicAdd(&nswap, 1);
          e[0] = (int)((int64_t)lo * a.maxpages) + place;
          e[1] = was;
          e[2] = id;
        } else {
          row[held + k - cow[lo]] = id;
        }
        a.ref[id] = 1;
      }
      __syncthreads();
      done = stop;
    }
  }
  __syncthreads();
  // (only now: a page that this call gives up is not handed out by it)
  for (int x = t; x < nswap; x += kScanThreads) {
    a.tab[swaps[3 * (int64_t)x]] = swaps[3 * (int64_t)x + 2];
    atomicSub(&a.ref[swaps[3 * (int64_t)x + 1]], 1);
  }
#pragma unroll
  for (int u = 0; u < kSlotsPerThread; ++u) {
    const int s = t * kSlotsPerThread + u;
    if (s < a.nslots && need[u] > 0 && off[s] + need[u] <= nfree)
      a.held[s] = clamp_i(a.held[s], 0, a.maxpages) + need[u] - cow[s];
  }
  if (t == 0) copies[0] = ncopy;
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
constexpr int kCopyChunk = 16384;       // bytes a block moves at a time

// pairs: *count (from, to) page ids, from at pairs[x * stride], to behind it
// at pairs[x * stride + gap].  Every layer's page is copied in 16 KiB chunks.
__device__ __forceinline__ void copy_pages(const int *count, const int *pairs, int stride,
                                           int64_t gap, PagePool pool, int64_t block,
                                           int64_t nblocks) {
  const int64_t chunks = (pool.page_bytes + kCopyChunk - 1) / kCopyChunk;
  const int64_t items = (int64_t)*count * pool.layers * chunks;
  for (int64_t it = block; it < items; it += nblocks) {
    const int64_t c = it % chunks, r = it / chunks, l = r % pool.layers, x = r / pool.layers;
    uint8_t *base = pool.pages + l * pool.stride + c * kCopyChunk;
    const u32x4_t *src =
        reinterpret_cast<const u32x4_t *>(base + (int64_t)pairs[x * stride] * pool.page_bytes);
    u32x4_t *dst =
        reinterpret_cast<u32x4_t *>(base + (int64_t)pairs[x * stride + gap] * pool.page_bytes);
    const int64_t left = pool.page_bytes - c * kCopyChunk;
    const int n = (int)((left < kCopyChunk ? left : kCopyChunk) / 16);
    u32x4_t v[kCopyChunk / 16 / 256];
#pragma unroll
    for (int u = 0; u < kCopyChunk / 16 / 256; ++u) {
      const int i = threadIdx.x + 256 * u;
      if (i < n) v[u] = src[i];
    }
#pragma unroll
    for (int u = 0; u < kCopyChunk / 16 / 256; ++u) {
      const int i = threadIdx.x + 256 * u;
      if (i < n) dst[i] = v[u];
    }
  }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(const int *copies, PagePool pool) {
  copy_pages(copies, copies + 1, 2, 1, pool, blockIdx.x, gridDim.x);
}

// One wave per slot.
__global__ __launch_bounds__(256) void pages_set_len_kernel(PagesArgs a,
                                                            const int *__restrict__ new_len) {
  const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (s >= a.nslots) return;
  const int want = new_len[s];
  if (want < 0) return;
  const int held = clamp_i(a.held[s], 0, a.maxpages);
  const int len = clamp_i(want, 0, (int64_t)held * a.page);
  const int keep = pages_of(len, a.page);
  int *row = a.tab + (int64_t)s * a.maxpages;
  for (int j = keep + lane; j < held; j += 64) {
    const int id = page_or_none(row[j], (int)a.npages);
    row[j] = -1;
    if (id >= 0) atomicSub(&a.ref[id], 1);
  }
  if (lane == 0) {
    a.len[s] = len;
    a.held[s] = keep;
  }
}

// Slot s becomes a copy of slot source[s], every source as it was before the
// call.  A block owns `cols` table columns of all slots and holds their old
// entries in LDS, so no entry is written before its readers have it; block 0
// does the same for the lengths, in registers.
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesArgs a,
                                                         const int *__restrict__ source,
                                                         int cols) {
  extern __shared__ int old[];           // [nslots][cols]
  const int t = threadIdx.x, nslots = (int)a.nslots, npages = (int)a.npages;
  const int64_t c0 = (int64_t)blockIdx.x * cols;
  const int nc = (int)(a.maxpages - c0 < cols ? a.maxpages - c0 : cols);
  for (int i = t; i < nslots * cols; i += 256) {
    const int c = i % cols;
    old[i] = c < nc ? a.tab[(int64_t)(i / cols) * a.maxpages + c0 + c] : -1;
  }
  constexpr int N = kPagesMaxSlots / 256;
  int len[N], held[N];
  if (blockIdx.x == 0) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int s = t + 256 * u, f = s < nslots ? source[s] : -1;
      held[u] = -1;
      if (f >= 0 && f < nslots) {
        len[u] = a.len[f];
        held[u] = clamp_i(a.held[f], 0, a.maxpages);
      }
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (held[u] < 0) continue;
      a.len[t + 256 * u] = len[u];
      a.held[t + 256 * u] = held[u];
    }
  }
  for (int i = t; i < nslots * cols; i += 256) {
    const int s = i / cols, c = i % cols, f = source[s];
    if (c >= nc || f < 0 || f >= nslots) continue;
    const int was = old[i], now = old[f * cols + c];
    if (was == now) continue;
    a.tab[(int64_t)s * a.maxpages + c0 + c] = now;
    if (page_or_none(was, npages) >= 0) atomicSub(&a.ref[was], 1);
    if (page_or_none(now, npages) >= 0) atomicAdd(&a.ref[now], 1);
  }
}

// One block: the number of live pages n, and the moves that leave them at
// ids 0 .. n-1: the live pages from n on, ascending, to the free ids below n,
// ascending (as many of one as of the other).  ws: the number of moves, -, src
// [npages], dst[npages], to[npages] (where a moved page went).
__global__ __launch_bounds__(kScanThreads) void pages_compact_kernel(PagesArgs a,
                                                                     int *__restrict__ live,
                                                                     int *__restrict__ ws) {
  __shared__ int wsum[kScanThreads / 64];
  const int t = threadIdx.x;
  int *src = ws + 2, *dst = src + a.npages, *to = dst + a.npages;
  int mine = 0, n;
  for (int64_t p = 4 * t; p < a.npages; p += 4 * kScanThreads) {
    int r[4];
    refs4(a.ref, p, a.npages, r);
#pragma unroll
    for (int u = 0; u < 4; ++u) mine += p + u < a.npages && r[u] > 0;
  }
  block_scan(mine, wsum, &n);
  int nd = 0, ns = 0;
  for (int64_t p0 = 0; p0 < a.npages; p0 += 4 * kScanThreads) {
    const int64_t p = p0 + 4 * t;
    int r[4], d = 0, s = 0, all;
    refs4(a.ref, p, a.npages, r);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u >= a.npages) continue;
      d += p + u < n && r[u] <= 0;
      s += p + u >= n && r[u] > 0;
    }
    // a thread's four pages and a chunk's 4096 lie on one side of n or hold
    // few of either, so one sum carries both counts (each below 2^15)
    const int at = block_scan(d | s << 16, wsum, &all);
    int da = nd + (at & 0xffff), sa = ns + (at >> 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u >= a.npages) continue;
      if (p + u < n && r[u] <= 0) dst[da++] = (int)(p + u);
      if (p + u >= n && r[u] > 0) src[sa++] = (int)(p + u);
    }
    nd += all & 0xffff;
    ns += all >> 16;
  }
  __syncthreads();
  for (int x = t; x < ns; x += kScanThreads) {
    const int f = src[x], g = dst[x];
    to[f] = g;
    a.ref[g] = a.ref[f];
    a.ref[f] = 0;
  }
  if (t == 0) {
    ws[0] = ns;
    ws[1] = n;
    *live = n;
  }
}

// Blocks below `rblocks` rewrite the tables, the others move the pages (the
// sources are live and the targets free, so no move reads what another wrote).
__global__ __launch_bounds__(256) void pages_move_kernel(PagesArgs a, const int *__restrict__ ws,
                                                         PagePool pool, int rblocks) {
  const int ns = ws[0], n = ws[1];
  if ((int)blockIdx.x >= rblocks) {
    copy_pages(ws, ws + 2, 1, a.npages, pool, blockIdx.x - rblocks, gridDim.x - rblocks);
    return;
  }
  if (ns == 0) return;
  const int *to = ws + 2 + 2 * a.npages;
  const int64_t entries = a.nslots * a.maxpages;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries;
       i += (int64_t)rblocks * 256) {
    if (i % a.maxpages >= a.held[i / a.maxpages]) continue;
    const int id = a.tab[i];
    if (id >= n && id < a.npages) a.tab[i] = to[id];
  }
}

int64_t copy_blocks(int64_t pairs, const PagePool &pool) {
  const int64_t items = pairs * pool.layers * ((pool.page_bytes + kCopyChunk - 1) / kCopyChunk);
  return items < 2048 ? items : 2048;
}

}  // namespace

hipError_t launch_pages_reserve(const PagesArgs &a, const int *want, const PagePool &pool, int *ws,
                                hipStream_t st) {
  hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(kScanThreads), 0, st, a, want, ws);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t blocks = copy_blocks(a.nslots, pool);
  if (blocks > 0)
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)blocks), dim3(256), 0, st, ws, pool);
  return hipGetLastError();
}

hipError_t launch_pages_set_len(const PagesArgs &a, const int *new_len, hipStream_t st) {
  hipLaunchKernelGGL(pages_set_len_kernel, dim3((unsigned)((a.nslots + 3) / 4)), dim3(256), 0, st,
                     a, new_len);
  return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesArgs &a, const int *source, hipStream_t st) {
  // columns of a block: at most 4 entries a thread where there are columns
  // enough, and 64 KB of LDS (64 slots of 34 pages: one block of 64 columns
  // 16.0 us, nine of 4 3.8)
  int cols = 64;
  while (cols > 4 && a.nslots * cols > 1024) cols >>= 1;
  while (cols > 4 && (a.maxpages + cols - 1) / cols < 64) cols >>= 1;
  hipLaunchKernelGGL(pages_fork_kernel, dim3((unsigned)((a.maxpages + cols - 1) / cols)),
                     dim3(256), (size_t)(a.nslots * cols * 4), st, a, source, cols);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesArgs &a, int *live, const PagePool &pool, int *ws,
                                hipStream_t st) {
  hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kScanThreads), 0, st, a, live, ws);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t entries = a.nslots * a.maxpages;
  const int rblocks = (int)((entries + 4095) / 4096 < 256 ? (entries + 4095) / 4096 : 256);
  const int64_t blocks = copy_blocks(a.npages / 2, pool);
  hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)(rblocks + (blocks > 0 ? blocks : 1))),
                     dim3(256), 0, st, a, ws, pool, rblocks);
  return hipGetLastError();
}

}  // namespace q8
