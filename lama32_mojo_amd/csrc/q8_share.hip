// q8_share.hip -- which sequences of a step name the same pages for their first
// tokens: what q8_kv8_attention_shared reads once for all of them.
//
// Written, int32: the number of groups G; group[nseq]; tokens[nseq]; pos[nseq], the
// place of the sequence's first row in the list of rows; lead[nseq] and gtokens[nseq],
// of group g at g; gcu[nseq + 1], group g's rows being the places gcu[g] .. gcu[g+1]-1;
// row[rows], the list.  Bound: two launches and their chains of dependent reads (tables of 8000 pages
// a sequence are 2 MB for 64).
#include "q8_launch.h"
#include "q8_ragged.h"

namespace q8 {
namespace {

constexpr int kThreads = 256;

// Whole pages that hold cached tokens only, of a sequence with rows (0: none).
__device__ __forceinline__ int whole_pages(const Kv8Args &c, int i) {
  const int r0 = clamp_i(c.cu[i], 0, c.rows), r1 = clamp_i(c.cu[i + 1], 0, c.rows);
  return r1 > r0 ? clamp_i(c.len[i], 0, c.maxpages * c.page) / c.page : 0;
}

// Block i: the first sequence whose table begins with the page that sequence i's
// begins with (to lead[i]; -1: no whole page) and how many whole pages the two have in
// common (to pos[i]).
__global__ __launch_bounds__(kThreads) void share_find_kernel(Kv8Args c, int *share) {
  __shared__ int first, common;
  const int i = blockIdx.x, t = threadIdx.x, nseq = (int)c.nseq;
  int *pos = share + 1 + 2 * nseq, *lead = share + 1 + 3 * nseq;
  if (t == 0) first = i;
  const int mine = whole_pages(c, i);
  const int *tab = c.tab + (int64_t)i * c.maxpages;
  const int id = mine ? page_or_none(tab[0], (int)c.npages) : -1;
  if (id < 0) {                                       // (the whole block)
    if (t == 0) {
      lead[i] = -1;
      pos[i] = 0;
    }
    return;
  }
  __syncthreads();
  for (int j = t; j < i; j += kThreads)
    if (c.tab[(int64_t)j * c.maxpages] == id && whole_pages(c, j) > 0) {
      atomicMin(&first, j);
      break;
    }
  __syncthreads();
  const int f = first, most = min(mine, whole_pages(c, f));
  const int *other = c.tab + (int64_t)f * c.maxpages;
  if (t == 0) common = most;
  __syncthreads();
  for (int p0 = 0; p0 < most; p0 += kThreads) {
    const int p = p0 + t;
    if (p < most && (tab[p] != other[p] || page_or_none(tab[p], (int)c.npages) < 0)) atomicMin(&common, p);
    __syncthreads();
    if (common < most) break;
    __syncthreads();
  }
  if (t == 0) {
    lead[i] = f;
    pos[i] = common;
  }
}

// One block, a thread a sequence.  Of the sequences with one leader, the p pages that
// save the most reads, (members with p pages and more in common - 1) * p, are the
// group's.
__global__ __launch_bounds__(kKv8ShareSeq) void share_group_kernel(Kv8Args c, int *share) {
  // (read four at a time; behind nseq: no sequence)
  __shared__ __attribute__((aligned(16))) int who[kKv8ShareSeq], pages[kKv8ShareSeq], rows[kKv8ShareSeq],
      index[kKv8ShareSeq];
  __shared__ unsigned long long best[kKv8ShareSeq];
  __shared__ int groups;
  const int t = threadIdx.x, nseq = (int)c.nseq;
  int *group = share + 1, *tok = share + 1 + nseq, *pos = share + 1 + 2 * nseq, *lead = share + 1 + 3 * nseq;
  int *gtok = share + 1 + 4 * nseq, *gcu = share + 1 + 5 * nseq, *list = share + 2 + 6 * nseq;
  int r0 = 0, n = 0, me = -1, p = 0;
  if (t < nseq) {
    r0 = clamp_i(c.cu[t], 0, c.rows);
    n = max(clamp_i(c.cu[t + 1], 0, c.rows) - r0, 0);
    me = lead[t];
    p = pos[t];
  }
  best[t] = 0;
  who[t] = me;
  pages[t] = p;
  rows[t] = n;
  __syncthreads();
  const int4 *who4 = reinterpret_cast<const int4 *>(who), *pages4 = reinterpret_cast<const int4 *>(pages);
  const int4 *rows4 = reinterpret_cast<const int4 *>(rows), *index4 = reinterpret_cast<const int4 *>(index);
  const int quads = (nseq + 3) / 4;
  if (me >= 0) {
    int members = 0;
#pragma unroll 4
    for (int j = 0; j < quads; ++j) {
      const int4 w = who4[j], g = pages4[j];
      members += ((w.x == me) & (g.x >= p)) + ((w.y == me) & (g.y >= p)) + ((w.z == me) & (g.z >= p)) +
                 ((w.w == me) & (g.w >= p));
    }
    // (members below 2^10, pages at most 2^26: 36 bits and 28; the longest of equal ones)
    atomicMax(&best[me], (unsigned long long)(members - 1) * p << 28 | (unsigned)p);
  }
  __syncthreads();
  const unsigned long long b = me >= 0 ? best[me] : 0;
  const int take = b >> 28 ? (int)(b & 0xfffffffu) : 0;
  bool in = take > 0 && p >= take;
  // groups in the order of their leaders, which are their first members
  const bool leads = in && me == t;
  if (!in) who[t] = -1;
  index[t] = leads;
  if (t == 0) groups = 0;
  __syncthreads();
  int g = 0;
#pragma unroll 4
  for (int j = 0; j < quads; ++j) {
    const int4 x = index4[j];
    g += (4 * j < me ? x.x : 0) + (4 * j + 1 < me ? x.y : 0) + (4 * j + 2 < me ? x.z : 0) + (4 * j + 3 < me ? x.w : 0);
  }
  in = in && g < kKv8ShareGroups;
  __syncthreads();
  if (!in) who[t] = -1;
  __syncthreads();
  // the rows of the groups before, of the group's members before, of all
  // (unsigned: nonsense in cu may wrap)
  uint32_t before = 0, at = 0, all = 0;
#pragma unroll 4
  for (int j = 0; j < quads; ++j) {
    const int4 w = who4[j], x = rows4[j];
    const int wj[4] = {w.x, w.y, w.z, w.w}, xj[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at += wj[u] == me && 4 * j + u < t ? (uint32_t)xj[u] : 0;
      before += wj[u] >= 0 && wj[u] < me ? (uint32_t)xj[u] : 0;
      all += wj[u] >= 0 ? (uint32_t)xj[u] : 0;
    }
  }
  if (leads && in) {
    atomicAdd(&groups, 1);
    lead[g] = t;
    gtok[g] = take * c.page;
    gcu[g] = (int)before;
  }
  __syncthreads();
  if (t < nseq) {
    group[t] = in ? g : -1;
    tok[t] = in ? take * c.page : 0;
    pos[t] = in ? (int)(before + at) : 0;
  }
  if (t == 0) {
    share[0] = groups;
    gcu[groups] = (int)all;
  }
  if (in)
    for (int k = 0; k < n && before + at + k < (uint32_t)c.rows; ++k) list[before + at + k] = r0 + k;
}

}  // namespace

hipError_t launch_kv8_share(const Kv8Args &c, int *share, hipStream_t st) {
  hipLaunchKernelGGL(share_find_kernel, dim3((unsigned)c.nseq), dim3(kThreads), 0, st, c, share);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(share_group_kernel, dim3(1), dim3((unsigned)((c.nseq + 63) / 64 * 64)), 0, st, c, share);
  return hipGetLastError();
}

}  // namespace q8
