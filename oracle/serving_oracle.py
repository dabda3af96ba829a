"""Float64 restatement of the calls for requests that differ: drawing tokens,
low-rank adapters, attention after a shared prefix.

  sample   w_i = exp((x_i - max) / T); order x descending, index ascending; kept: the
           first k, of these the ones with less than top_p of the sum before them, of
           these the ones with w_i >= min_p; drawn: the first whose running sum exceeds
           u times the kept sum
  lora     y = base + scale B (A x), an A per part of the columns
  share    sequences whose tables begin with the same page: the lowest leads; tokens
           shared: the whole cached pages p that maximise (members with p pages in
           common with it - 1) * p, the longest of equal ones
"""

from __future__ import annotations

import numpy as np


def sample_row(x, temp=1.0, k=0, top_p=1.0, min_p=0.0, u=0.0):
    """(id, log-probability) of one row of logits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return -1, -np.inf
    temp, top_p, min_p, u = (np.float64(np.float32(v)) for v in (temp, top_p, min_p, u))
    if not temp > 0:
        return int(order[0]), 0.0
    v = x[order]
    if v[0] == np.inf:
        w = (v == np.inf).astype(np.float64)
    else:
        with np.errstate(under="ignore"):
            w = np.exp((v - v[0]) / temp)
    n = k if 0 < k < len(w) else len(w)
    w = w[:n]
    if top_p < 1:
        w = w[:max(1, int((np.cumsum(w) - w < top_p * w.sum()).sum()))]
    if min_p > 0:
        w = w[:max(1, int((w >= min(min_p, 1.0)).sum()))]
    c = np.cumsum(w)
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    at = min(int((c <= u * c[-1]).sum()), int((w > 0).sum()) - 1)
    return int(order[at]), float(np.log(w[at] / c[-1]))


def lora(x, base, cu, ids, A, B, scale, widths):
    """A[i]: the parts' [rank, m] matrices one under the other, B[i] [n, rank] (lists, by
    adapter; None: rank 0).  (y, the sum of magnitudes behind each of its elements)."""
    x, y = x.astype(np.float64), base.astype(np.float64).copy()
    size = np.abs(y)
    first = np.concatenate([[0], np.cumsum(widths)])
    for s, i in enumerate(ids):
        rows = slice(cu[s], cu[s + 1])
        if not 0 <= i < len(A) or A[i] is None or cu[s + 1] <= cu[s]:
            continue
        a, b, r = A[i].astype(np.float64), B[i].astype(np.float64), B[i].shape[1]
        for p in range(len(widths)):
            ap, bp = a[p * r:(p + 1) * r], b[first[p]:first[p + 1]]
            cols = slice(first[p], first[p + 1])
            with np.errstate(invalid="ignore", over="ignore"):
                y[rows, cols] += float(scale[i]) * (x[rows] @ ap.T) @ bp.T
                size[rows, cols] += abs(float(scale[i])) * (np.abs(x[rows]) @ np.abs(ap).T) @ np.abs(bp).T
    return y, size


def share(cu, length, table, page, npages, most_groups=64):
    """(group, tokens) of every sequence."""
    ns = len(length)
    whole = [min(length[i], table.shape[1] * page) // page if cu[i + 1] > cu[i] else 0 for i in range(ns)]

    def common(i, j):
        n = 0
        while n < min(whole[i], whole[j]) and table[i][n] == table[j][n] and 0 <= table[i][n] < npages:
            n += 1
        return n
    lead = [next((j for j in range(i + 1) if whole[j] and table[j][0] == table[i][0]), -1)
            if whole[i] and 0 <= table[i][0] < npages else -1 for i in range(ns)]
    group, tokens, count = [-1] * ns, [0] * ns, 0
    for f in range(ns):
        member = {i: common(i, f) for i in range(ns) if lead[i] == f}
        if lead[f] != f or count == most_groups:
            continue
        saves = {p: (sum(c >= p for c in member.values()) - 1) * p for p in member.values()}
        saved = max(saves.values())
        take = max(p for p, v in saves.items() if v == saved)
        if saved <= 0:
            continue
        for i, c in member.items():
            if c >= take:
                group[i], tokens[i] = count, take * page
        count += 1
    return group, tokens
