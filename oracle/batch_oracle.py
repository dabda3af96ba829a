"""Float64 restatement of the calls over several sequences: attention over packed
prompts, the 8-bit paged cache (append, attention) and the state of its pages.

Formulas (rows of sequence i: cu[i] .. cu[i+1]-1, at positions len[i] + j):

  attention  out[r, h] = sum_t softmax_t(q[r, h] . k[t, h / grp] / sqrt(hd)) v[t, h / grp]
             over the t that row r sees
  rotation   (a, b) -> (a cos - b sin, b cos + a sin), angle position * inv_freq,
             keys rounded to f32 once
  codes      s = max(s_old, f32(max |x| * f32(1 / 127))); rint(x / s), half to even, in
             [-127, 127]; older codes rint(c s_old / s) where s grew
"""

from __future__ import annotations

import numpy as np


def attend(q, k, v, first):
    """q [n, nheads, hd], k and v [ctx, nkv, hd] (float64): row j sees keys
    0 .. first + j, whatever the others hold."""
    n, nh, hd = q.shape
    grp = nh // k.shape[1]
    out = np.empty((n, nh, v.shape[2]))
    with np.errstate(all="ignore"):
        for j in range(n):
            kk, vv = k[:first + j + 1], v[:first + j + 1]
            for h in range(nh):
                s = kk[:, h // grp] @ q[j, h] / np.sqrt(hd)
                p = np.exp(s - s.max())
                out[j, h] = p @ vv[:, h // grp] / p.sum()
    return out


def attention_packed(q, k, v, cu):
    """q [rows, nheads, hd], k and v [rows, nkv, hd]; rows from cu[-1] on are NaN."""
    out = np.full(q.shape, np.nan)
    for a, b in zip(cu[:-1], cu[1:]):
        out[a:b] = attend(q[a:b].astype(np.float64), k[a:b].astype(np.float64),
                          v[a:b].astype(np.float64), 0)
    return out


def rotate(x, pos, inv):
    """rotate_half RoPE of x [n, heads, hd] at the positions pos [n], float64."""
    ang = np.asarray(pos, np.float64)[:, None, None] * inv.astype(np.float64)
    c, s = np.cos(ang), np.sin(ang)
    a, b = np.split(x.astype(np.float64), 2, axis=-1)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def page_bytes(P, nkv, hd):
    return 2 * nkv * P * hd + (8 * nkv + 15) // 16 * 16


class Cache:
    """Pages as arrays: K codes [npages, nkv, P, hd], V codes [npages, nkv, hd, P],
    scales [npages, 2, nkv]."""

    def __init__(self, npages, P, nkv, hd):
        self.npages, self.P, self.nkv, self.hd = npages, P, nkv, hd
        self.k = np.zeros((npages, nkv, P, hd), np.int8)
        self.v = np.zeros((npages, nkv, hd, P), np.int8)
        self.s = np.zeros((npages, 2, nkv), np.float32)

    def random(self, rng, scale=0.02):
        self.k[:] = rng.integers(-127, 128, self.k.shape)
        self.v[:] = rng.integers(-127, 128, self.v.shape)
        self.s[:] = scale * np.exp(0.3 * rng.standard_normal(self.s.shape))
        return self

    def to_bytes(self):
        out = np.zeros((self.npages, page_bytes(self.P, self.nkv, self.hd)), np.uint8)
        n = self.nkv * self.P * self.hd
        out[:, :n] = self.k.reshape(self.npages, -1).view(np.uint8)
        out[:, n:2 * n] = self.v.reshape(self.npages, -1).view(np.uint8)
        out[:, 2 * n:2 * n + 8 * self.nkv] = self.s.reshape(self.npages, -1).view(np.uint8)
        return out

    @classmethod
    def from_bytes(cls, raw, P, nkv, hd):
        c = cls(len(raw), P, nkv, hd)
        n = nkv * P * hd
        c.k[:] = raw[:, :n].view(np.int8).reshape(c.k.shape)
        c.v[:] = raw[:, n:2 * n].view(np.int8).reshape(c.v.shape)
        c.s[:] = np.ascontiguousarray(raw[:, 2 * n:2 * n + 8 * nkv]).view(np.float32).reshape(c.s.shape)
        return c

    def values(self, row, count):
        """K and V of tokens 0 .. count-1 behind a table row, float64 (missing
        pages: NaN)."""
        k = np.full((count, self.nkv, self.hd), np.nan)
        v = k.copy()
        for t in range(count):
            p = row[t // self.P]
            if 0 <= p < self.npages:
                k[t] = self.k[p, :, t % self.P].astype(np.float64) * self.s[p, 0].astype(np.float64)[:, None]
                v[t] = self.v[p, :, :, t % self.P].astype(np.float64) * self.s[p, 1].astype(np.float64)[:, None]
        return k, v

    def append(self, q, k, v, inv, cu, length, table):
        """The rotated q (float64) and the binary16 K and V rows of the call;
        the pages are updated."""
        P, qr = self.P, np.full(q.shape, np.nan)
        rows = np.zeros((2, *k.shape), np.float16)
        cap = table.shape[1] * P
        for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
            pos = length[i] + np.arange(b - a)
            qr[a:b] = rotate(q[a:b], pos, inv)
            with np.errstate(all="ignore"):
                kr = rotate(k[a:b], pos, inv).astype(np.float32)
                rows[0, a:b], rows[1, a:b] = kr, v[a:b]
            for page in sorted(set((pos // P).tolist())):
                if page * P >= cap or not 0 <= table[i, page] < self.npages:
                    continue
                at = np.nonzero(pos // P == page)[0]
                old = max(0, length[i] - page * P)
                for w, (x, codes) in enumerate(((kr[at], self.k[table[i, page]]),
                                                (v[a:b][at], self.v[table[i, page]].transpose(0, 2, 1)))):
                    for g in range(self.nkv):
                        self.s[table[i, page], w, g] = self._block(
                            codes[g], x[:, g], pos[at] % P, old, self.s[table[i, page], w, g])
        return qr, rows

    @staticmethod
    def _block(codes, x, at, old, s_old):
        """New codes of one head in one page; returns the scale."""
        s0 = np.float32(s_old) if old else np.float32(0)
        top = np.abs(x).max()
        s1 = np.float32(top) * (np.float32(1) / np.float32(127))
        if np.isfinite(s1) and not s1 > s0:
            s1 = s0
        if not (np.isfinite(s1) and np.isfinite(s0)):
            codes[at] = 0
            return np.float32(np.nan)
        if s1 > s0 and old:
            codes[:old] = np.rint(codes[:old].astype(np.float64) * np.float64(s0) / np.float64(s1))
        if s1 == 0:
            codes[at] = 0
        else:
            codes[at] = np.clip(np.rint(x.astype(np.float64) / np.float64(s1)), -127, 127)
        return s1

    def attention(self, q, cu, length, table):
        out = np.full(q.shape, np.nan)
        cap = table.shape[1] * self.P
        for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
            for r in range(a, b):
                k, v = self.values(table[i], min(int(length[i]) + r - a + 1, cap))
                out[r] = attend(q[r:r + 1].astype(np.float64), k, v, len(k) - 1)[0]
        return out


class Pages:
    """The page state of slots as plain lists."""

    def __init__(self, nslots, maxpages, npages, P):
        self.P, self.maxpages, self.npages = P, maxpages, npages
        self.rows = [[] for _ in range(nslots)]       # page ids held
        self.len = [0] * nslots

    def refs(self):
        r = [0] * self.npages
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def arrays(self):
        tab = np.full((len(self.rows), self.maxpages), -1, np.int32)
        for s, row in enumerate(self.rows):
            tab[s, :len(row)] = row
        return dict(table=tab, len=np.array(self.len, np.int32),
                    held=np.array([len(r) for r in self.rows], np.int32),
                    ref=np.array(self.refs(), np.int32))

    def reserve(self, want):
        """Returns the copies (from, to)."""
        ref = self.refs()
        free = [p for p in range(self.npages) if ref[p] == 0]
        copies, short = [], False
        plan = []
        for s, row in enumerate(self.rows):
            w = min(max(want[s], 0), self.maxpages * self.P)
            to = min(len(row), -(-w // self.P)) if w > self.len[s] else 0
            own = [j for j in range(self.len[s] // self.P, to) if ref[row[j]] > 1]
            plan.append((own, max(0, -(-w // self.P) - len(row))))
        at = 0
        for s, (own, more) in enumerate(plan):
            n = len(own) + more
            if n == 0:
                continue
            short = short or at + n > len(free)
            if short:
                continue
            got = free[at:at + n]
            at += n
            for j, p in zip(own, got):
                if j == self.len[s] // self.P and self.len[s] % self.P:
                    copies.append((self.rows[s][j], p))
                self.rows[s][j] = p
            self.rows[s] += got[len(own):]
        return copies

    def set_len(self, new):
        for s, n in enumerate(new):
            if n >= 0:
                self.len[s] = min(n, len(self.rows[s]) * self.P)
                del self.rows[s][-(-self.len[s] // self.P):]

    def fork(self, source):
        rows, length = [list(r) for r in self.rows], list(self.len)
        for s, f in enumerate(source):
            if 0 <= f < len(rows):
                self.rows[s], self.len[s] = list(rows[f]), length[f]

    def compact(self):
        """Returns (pages in use, moves (from, to))."""
        ref = self.refs()
        n = sum(r > 0 for r in ref)
        src = [p for p in range(n, self.npages) if ref[p] > 0]
        dst = [p for p in range(n) if ref[p] == 0]
        to = dict(zip(src, dst))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return n, list(zip(src, dst))
