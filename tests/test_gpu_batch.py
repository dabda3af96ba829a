"""GPU parity of the calls over several sequences (through the C ABI) against the
float64 restatement in oracle/batch_oracle.py.

Bars, by arithmetic:
  * f32 attention: 1e-5 of the largest output.  Products are exact (the operands'
    terms add up to the f32 value), so what is left are f32 sums of at most some
    thousand terms and one exp2 per probability, a few 2^-24 each.
  * bf16 attention: half a bf16 step (2^-8 of the value) for the output, half a
    binary16 step (2^-11) of the largest |v| for the rounded probabilities, and
    the f32 bar.
  * codes, scales, page tables: equal.  (A key next to a border of two codes
    could differ where the f64 cos or sin does in its last bits; none of these
    inputs is that near.)
  * rotated q: 4 steps of 2^-24 of the pair's size (two products, one sum, and the
    rounded cos and sin)."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import batch_oracle as bo
from oracle.q8_oracle import max_rel_err

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def dev(ctx, *arrays, pad=0):
    """The arrays back to back in one buffer, and their byte offsets."""
    offs, top = [], pad
    for a in arrays:
        offs.append(top)
        top += a.nbytes
    b = ctx.alloc(max(top, 16))
    for a, o in zip(arrays, offs):
        if a.nbytes:
            b.upload(a, o)
    return b, offs


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_to_f32(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def inv_freq(hd, theta=500000.0):
    return np.array([theta ** (-2.0 * d / hd) for d in range(hd // 2)], np.float32)


# ---- attention over packed prompts --------------------------------------------------

def run_packed(ctx, q, k, v, cu, act="f32", extra=0, dead=0):
    """q [T, nh, hd] ... -> out [T + dead, nh, hd]; q rows `extra` elements apart
    from each other, `dead` rows behind the last sequence."""
    T, nh, hd = q.shape
    nkv = k.shape[1]
    rows, ld = T + dead, nh * hd + extra
    qd = np.zeros((rows, ld), np.uint16 if act == "bf16" else np.float32)
    qd[:T, :nh * hd] = (bf16_bits(q) if act == "bf16" else q).reshape(T, -1)
    kv = np.full((2, rows, nkv * hd), np.nan, np.float16)
    kv[0, :T], kv[1, :T] = k.reshape(T, -1), v.reshape(T, -1)
    mark = np.full((rows, nh * hd), 7, qd.dtype)
    qb, kb, ob, ib = (dev(ctx, x)[0] for x in (qd, kv, mark, np.asarray(cu, np.int32)))
    q8hip.attention_packed(ctx, qb, 0, kb, 0, rows * nkv * hd, ob, 0, ib, 0, len(cu) - 1, rows, nh, nkv,
                           hd, act, ld if extra else 0)
    out = ob.download((rows, nh * hd), qd.dtype)
    for b in (qb, kb, ob, ib):
        b.free()
    assert (out[T:] == mark[T:]).all()
    return (bf16_to_f32(out) if act == "bf16" else out)[:T].reshape(T, nh, hd)


def packed_inputs(rng, lens, nh, nkv, hd):
    T = sum(lens)
    q = rng.standard_normal((T, nh, hd)).astype(np.float32) * np.exp(rng.standard_normal((T, 1, 1)) * 0.5)
    k, v = rng.standard_normal((2, T, nkv, hd)).astype(np.float16)
    return q.astype(np.float32), k, v


@pytest.mark.parametrize("lens", [[1], [0, 1, 0, 2], [33, 1, 64, 65, 0], [130, 257], [5] * 70, [700]],
                         ids=lambda x: "-".join(map(str, x[:5])))
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (3, 3, 128), (6, 2, 64), (5, 1, 64)])
def test_packed(ctx, lens, nh, nkv, hd):
    say("packed", lens, nh, nkv, hd)
    rng = np.random.default_rng(len(lens) + hd)
    if sum(lens) > 600 and nh != 8:
        lens = lens[:1] + [9]
    q, k, v = packed_inputs(rng, lens, nh, nkv, hd)
    cu = offsets(lens)
    ref = bo.attention_packed(q, k, v, cu)
    assert max_rel_err(run_packed(ctx, q, k, v, cu, extra=2 * nkv * hd, dead=3), ref) <= 1e-5
    qb = bf16_to_f32(bf16_bits(q))
    ref = bo.attention_packed(qb, k, v, cu)
    y = run_packed(ctx, q, k, v, cu, act="bf16", extra=8)
    bar = 2.0 ** -8 * np.abs(ref) + 2.0 ** -11 * np.abs(v.astype(np.float64)).max() + 1e-5
    assert (np.abs(y - ref) <= bar).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_packed_hidden_values(ctx, act):
    """Infinities, NaN and the largest binary16 values in rows that a row does not
    see leave it as it was; rows that see them have what the formula gives."""
    say("packed hidden", act)
    rng = np.random.default_rng(5)
    lens = [40, 100, 7]
    q, k, v = packed_inputs(rng, lens, 4, 2, 64)
    cu = offsets(lens)
    clean = run_packed(ctx, q, k, v, cu, act)
    k2, v2 = k.copy(), v.copy()
    v2[20] = np.nan
    v2[60, 0, 3] = np.inf
    k2[90, 1] = -np.inf
    k2[139] = 65504.0
    k2[145] = np.nan
    y = run_packed(ctx, q, k2, v2, cu, act)
    ref = bo.attention_packed(bf16_to_f32(bf16_bits(q)) if act == "bf16" else q, k2, v2, cu)
    same = np.r_[0:20, 40:60, 140:145]
    bar = 1e-5 if act == "f32" else 2.0 ** -6
    assert max_rel_err(y[same], clean[same]) <= bar
    assert (np.isnan(y) == np.isnan(ref)).all() and (np.isposinf(y) == np.isposinf(ref)).all()
    f = np.isfinite(ref)
    assert max_rel_err(y[f], ref[f]) <= bar


def test_packed_large_scores(ctx):
    """Scores far from 0 (the softmax's maximum is subtracted), rows whose dims
    span many powers of two, q of zeros."""
    say("packed large")
    rng = np.random.default_rng(6)
    q, k, v = packed_inputs(rng, [90, 50], 4, 4, 128)
    q *= np.exp2(rng.integers(-12, 6, (1, 1, 128))).astype(np.float32)
    q[7] = 0
    q[100:] *= 100
    ref = bo.attention_packed(q, k, v, offsets([90, 50]))
    # a score of size S carries S 2^-22: here S < 2^13, of which e^x makes a factor
    assert max_rel_err(run_packed(ctx, q, k, v, offsets([90, 50])), ref) <= 2e-3
    assert max_rel_err(run_packed(ctx, q, k, v, offsets([90, 50]))[:90], ref[:90]) <= 1e-4


def test_packed_nonsense_offsets(ctx):
    """Offsets out of order or out of range stay inside the buffers (the rows of
    well-formed sequences among them are right)."""
    say("packed nonsense")
    rng = np.random.default_rng(8)
    q, k, v = packed_inputs(rng, [64], 2, 1, 64)
    y = run_packed(ctx, q, k, v, [-5, 10, 10, 4, 1 << 30])
    ref = bo.attention_packed(q, k, v, [0, 10])
    assert max_rel_err(y[:4], ref[:4]) <= 1e-5


# ---- the 8-bit cache --------------------------------------------------------------------

class Paged:
    """A cache, its table and lengths on the GPU beside the oracle's."""

    def __init__(self, ctx, rng, lens, old, P, nkv, hd, spare=2, random=True):
        self.ctx, self.P, self.nkv, self.hd, self.nseq = ctx, P, nkv, hd, len(lens)
        pages = [-(-(o + n) // P) for o, n in zip(old, lens)]
        self.maxpages = max(pages + [1]) + 1
        self.c = bo.Cache(sum(pages) + spare, P, nkv, hd)
        if random:
            self.c.random(rng)
        ids = rng.permutation(self.c.npages)
        self.table = np.full((self.nseq, self.maxpages), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = ids[at:at + n]
            at += n
        self.old, self.cu = np.asarray(old, np.int32), offsets(lens)
        self.rows = int(self.cu[-1])
        self.pool, _ = dev(ctx, self.c.to_bytes())
        self.upload()

    def upload(self):
        flat = np.concatenate([self.cu, self.old, self.table.reshape(-1)]).astype(np.int32)
        self.ix, _ = dev(self.ctx, flat)
        self.at = (0, self.nseq + 1, 2 * self.nseq + 1)

    def where(self, rows=None):
        return (self.pool, 0, self.c.npages, self.P, self.ix, *self.at, self.nseq,
                self.rows if rows is None else rows, self.maxpages)

    def download(self):
        raw = self.pool.download((self.c.npages, bo.page_bytes(self.P, self.nkv, self.hd)), np.uint8)
        return raw


def run_append(p, q, k, v, inplace=False, off=0, rows16=True):
    """Through the GPU: rotated q and binary16 rows (the pages in p.pool)."""
    T, nh, hd = q.shape
    nkv = p.nkv
    ld = (nh + 2 * nkv) * hd + (3 if off else 0)
    arena = np.full(off + T * ld + T * nh * hd + hd // 2, 5, np.float32)
    st = arena[off:off + T * ld].reshape(T, ld)
    st[:, :nh * hd], st[:, nh * hd:(nh + nkv) * hd] = q.reshape(T, -1), k.reshape(T, -1)
    st[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd] = v.reshape(T, -1)
    oqr, oinv = off + T * ld, off + T * ld + T * nh * hd
    arena[oinv:] = inv_freq(hd)
    ab, _ = dev(p.ctx, arena)
    kv, _ = dev(p.ctx, np.full((2, T, nkv * hd), 9, np.float16))
    q8hip.kv8_append(p.ctx, ab, off, off + nh * hd, off + (nh + nkv) * hd, oinv, off if inplace else oqr,
                     *p.where(T), nh, nkv, hd, ld=ld, kv=kv if rows16 else None, okc_f16=0,
                     ovc_f16=T * nkv * hd)
    now = ab.download(arena.shape, np.float32)
    rows = kv.download((2, T, nkv, hd), np.float16)
    if inplace:
        qr = now[off:off + T * ld].reshape(T, ld)[:, :nh * hd]
        arena[off:off + T * ld].reshape(T, ld)[:, :nh * hd] = qr
    else:
        qr = now[oqr:oinv].reshape(T, -1)
        arena[oqr:oinv] = qr.reshape(-1)
    assert np.array_equal(now, arena, equal_nan=True)           # nothing else is written
    ab.free()
    kv.free()
    return qr.reshape(T, nh, hd), rows


def check_append(p, q, k, v, **kw):
    qr, rows = run_append(p, q, k, v, **kw)
    ref, rref = p.c.append(q, k, v, inv_freq(p.hd), p.cu, p.old, p.table)
    n = int(p.cu[-1])
    got = p.download()
    assert np.array_equal(got, p.c.to_bytes()) or np.array_equal(
        np.nan_to_num(bo.Cache.from_bytes(got, p.P, p.nkv, p.hd).s, nan=-1), np.nan_to_num(p.c.s, nan=-1)) \
        and np.array_equal(got[:, :2 * p.nkv * p.P * p.hd], p.c.to_bytes()[:, :2 * p.nkv * p.P * p.hd])
    if n == 0:
        return
    a, b = np.split(np.abs(q[:n].astype(np.float64)), 2, -1)
    size = np.concatenate([np.hypot(a, b)] * 2, -1)
    ok = np.isfinite(ref[:n])
    assert (np.abs(qr[:n] - ref[:n])[ok] <= 4 * 2.0 ** -24 * size[ok]).all()
    if kw.get("rows16", True):
        assert np.array_equal(rows[:, :n], rref[:, :n], equal_nan=True)


@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (4, 1, 128), (3, 3, 64), (10, 2, 128)])
def test_append(ctx, P, nh, nkv, hd):
    """Fresh pages, partly filled ones, runs over several pages, sequences
    without rows; q in place and apart, at any 4-byte alignment."""
    say("append", P, nh, nkv, hd)
    rng = np.random.default_rng(P + nh + hd)
    lens = [1, 0, P, P + 1, 3 * P - 5, 1, 2, 0, 17]
    old = [0, 5, 0, P - 1, 7, 4 * P, 5 * P - 1, 3, 1]
    for off, inplace, rows16 in ((0, False, True), (0, True, False), (1, True, True), (3, False, True)):
        p = Paged(ctx, rng, lens, old, P, nkv, hd)
        T = p.rows
        q, k, v = (rng.standard_normal((T, h, hd)).astype(np.float32) for h in (nh, nkv, nkv))
        k *= np.exp(rng.standard_normal((T, 1, 1)) * 0.7).astype(np.float32)
        check_append(p, q, k, v, off=off, inplace=inplace, rows16=rows16)


def test_append_token_by_token(ctx):
    """A page filled token by token, its scale growing now and then."""
    say("append tokens")
    rng = np.random.default_rng(3)
    p = Paged(ctx, rng, [1, 1], [0, 0], 16, 2, 64, spare=4)
    p.maxpages, p.table = 3, np.array([[3, 0, 5], [1, 4, 2]], np.int32)
    for t in range(20):
        p.old[:] = [t, 3 * t // 2]
        p.upload()
        q, k, v = (rng.standard_normal((2, h, 64)).astype(np.float32) * (1 + t % 5) for h in (4, 2, 2))
        if t == 0:
            k[:] = v[:] = 0                                    # a scale of 0 first
        check_append(p, q, k, v)


def test_append_extremes(ctx):
    """Denormal scales, the largest values, ties between two codes, NaN and
    infinities (their page and head alone), far positions."""
    say("append extremes")
    rng = np.random.default_rng(4)
    lens, old = [16] * 9, [0, 0, 0, 0, 0, 0, 5, 40000 * 16, 0]
    p = Paged(ctx, rng, lens, [0] * 6 + [5, 0, 0], 16, 1, 64)
    # (one sequence at a far position, over a page of its own at that index)
    p.maxpages = 40001
    wide = np.full((9, p.maxpages), -1, np.int32)
    wide[:, :2] = p.table[:, :2]
    wide[7, 40000] = p.table[7, 0]
    p.table, p.old = wide, np.asarray(old, np.int32)
    p.upload()
    q, k, v = (rng.standard_normal((p.rows, h, 64)).astype(np.float32) for h in (2, 1, 1))
    q[:], at = np.abs(q) + 0.1, lambda i: slice(16 * i, 16 * i + 16)
    k[at(0)] *= 1e-38
    v[at(0)] *= 3e-41
    k[at(1)] *= 1e37
    v[at(1)] = np.float32(3.4e38)
    v[at(2)] = np.arange(16 * 64).reshape(16, 1, 64) % 255 - 127            # scale 1: exact
    v[at(3)] = (np.arange(16 * 64).reshape(16, 1, 64) % 253 - 126) + 0.5    # ties
    v[at(3)][0, 0, 0] = 127
    v[at(4)][3, 0, 9] = np.nan
    k[at(5)][3, 0, 9] = np.inf
    v[at(6)][0, 0, 0] = -np.inf
    k[at(8)] = 0
    check_append(p, q, k, v)


def test_append_missing_pages(ctx):
    """Rows without a page (ids out of range, positions past the table) store
    nothing; their rotated q and binary16 rows are there."""
    say("append missing")
    rng = np.random.default_rng(9)
    p = Paged(ctx, rng, [40, 20, 30], [0, 10, 50], 16, 2, 64)
    p.table[0, 1] = -1
    p.table[1, 0] = p.c.npages
    p.table[2, 3] = -2 ** 31
    p.table[2, 4] = 2 ** 31 - 1
    p.maxpages = 5
    p.table = np.ascontiguousarray(p.table[:, :5])
    p.old[2] = 70                                             # rows 70 .. 99, the table ends at 80
    p.upload()
    q, k, v = (rng.standard_normal((p.rows, h, 64)).astype(np.float32) for h in (4, 2, 2))
    check_append(p, q, k, v)


def run_cache(p, q, off=0, extra=0, ctx=None):
    T, nh, hd = q.shape
    ld = nh * hd + extra
    arena = np.full(off + T * ld + T * nh * hd + 8, 5, np.float32)
    arena[off:off + T * ld].reshape(T, ld)[:, :nh * hd] = q.reshape(T, -1)
    a, _ = dev(p.ctx, arena)
    q8hip.kv8_attention(ctx or p.ctx, a, off, off + T * ld, *p.where(T), nh, p.nkv, hd,
                        ldq=ld if extra else 0)
    now = a.download(arena.shape, np.float32)
    out = now[off + T * ld:off + T * ld + T * nh * hd].copy()
    arena[off + T * ld:off + T * ld + T * nh * hd] = out
    assert np.array_equal(now, arena, equal_nan=True)
    a.free()
    return out.reshape(T, nh, hd)


CACHES = [([1], [0]), ([1], [63]), ([1, 0, 1], [64, 9, 1000]), ([2, 5, 1, 3], [0, 17, 300, 129]),
          ([1] * 33, [37 * i % 200 for i in range(33)]), ([9, 0, 4], [2500, 100, 0]), ([70], [130])]


@pytest.mark.parametrize("lens,old", CACHES, ids=lambda x: "-".join(map(str, x[:4])))
@pytest.mark.parametrize("nh,nkv,hd,P", [(8, 2, 64, 16), (8, 2, 128, 64), (3, 3, 128, 32), (6, 1, 64, 128),
                                         (16, 2, 128, 16), (20, 1, 128, 64)])
def test_cache_attention(ctx, lens, old, nh, nkv, hd, P):
    say("cache attention", lens[:5], old[:5], nh, nkv, hd, P)
    rng = np.random.default_rng(sum(old) + nh)
    p = Paged(ctx, rng, lens, old, P, nkv, hd)
    q = rng.standard_normal((p.rows, nh, hd)).astype(np.float32)
    ref = p.c.attention(q, p.cu, p.old, p.table)
    off, extra = (0, 2 * nkv * hd) if P != 32 else (1, 5)
    assert max_rel_err(run_cache(p, q, off, extra), ref) <= 1e-5


def test_cache_attention_long(ctx):
    """One context of 20000 tokens (many splits) beside short ones, against the
    same in float64; dims and pages of very different sizes."""
    say("cache long")
    rng = np.random.default_rng(12)
    p = Paged(ctx, rng, [1, 2, 1], [20000, 3, 700], 64, 1, 128)
    p.c.s *= np.exp2(rng.integers(-3, 4, p.c.s.shape)).astype(np.float32)
    p.pool.upload(p.c.to_bytes())
    q = rng.standard_normal((4, 2, 128)).astype(np.float32) * np.exp2(rng.integers(-20, 1, 128))
    q = q.astype(np.float32)
    k, v = p.c.values(p.table[0], 20001)
    ref = np.concatenate([bo.attend(q[:1].astype(np.float64), k, v, 20000),
                          p.c.attention(q[1:], offsets([2, 1]), p.old[1:], p.table[1:])])
    assert max_rel_err(run_cache(p, q), ref) <= 1e-5


@pytest.mark.parametrize("nh,hd,P", [(2, 128, 128), (5, 64, 128), (20, 128, 32), (40, 64, 64)])
def test_cache_attention_splits(ctx, nh, hd, P):
    """Split contexts at every page size and column tile (16, 32, 64 columns), odd
    first units among them, some units of a wave's run in the next sequence."""
    say("cache splits", nh, hd, P)
    rng = np.random.default_rng(nh + P)
    lens, old = [1, 2, 1, 1], [1500, 700, 64 * 7, 3333]
    p = Paged(ctx, rng, lens, old, P, 1, hd)
    q = rng.standard_normal((p.rows, nh, hd)).astype(np.float32)
    assert max_rel_err(run_cache(p, q), p.c.attention(q, p.cu, p.old, p.table)) <= 1e-5


def test_cache_attention_many_sequences(ctx):
    """More sequences than one launch plans for."""
    say("cache many")
    rng = np.random.default_rng(50)
    n = 1100
    p = Paged(ctx, rng, [1 + i % 2 if i % 7 else 0 for i in range(n)], [i % 40 for i in range(n)], 16, 1, 64)
    q = rng.standard_normal((p.rows, 2, 64)).astype(np.float32)
    ref = p.c.attention(q, p.cu, p.old, p.table)
    assert max_rel_err(run_cache(p, q), ref) <= 1e-5
    q, k, v = (rng.standard_normal((p.rows, h, 64)).astype(np.float32) for h in (2, 1, 1))
    check_append(p, q, k, v)


def test_cache_attention_hidden(ctx):
    """A NaN scale reaches the rows that see a token of its page and head, no
    others; missing pages make NaN; rows past the table see what it holds; rows
    behind the last sequence are left alone."""
    say("cache hidden")
    rng = np.random.default_rng(13)
    p = Paged(ctx, rng, [3, 20, 2, 4], [30, 40, 200, 70], 16, 2, 64)
    p.c.s[p.table[1, 3], 0, 1] = np.nan                       # K of tokens 48 .. 63, head 1
    p.c.s[p.table[0, 2], 1, 0] = np.nan                       # V of tokens 32 .. 47
    p.table[2, 5] = -1
    p.maxpages, p.table = 13, np.ascontiguousarray(p.table[:, :13])
    p.old[3] = 206                                            # rows 206 .. 209; the table ends at 208
    p.table[3, 5:] = p.table[3, 0]
    p.pool.upload(p.c.to_bytes())
    p.upload()
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float32)
    ref = p.c.attention(q, p.cu, p.old, p.table)
    y = run_cache(p, q)
    assert np.array_equal(np.isnan(y), np.isnan(ref)) and np.isnan(y).any()
    f = np.isfinite(ref)
    assert f.any() and max_rel_err(y[f], ref[f]) <= 1e-5
    more = run_cache_dead(p, q)
    assert np.array_equal(more[:p.rows], y, equal_nan=True) and (more[p.rows:] == 5).all()


def run_cache_dead(p, q):
    """The same call told of 3 more rows than the sequences have."""
    T, nh, hd = q.shape
    arena = np.full(2 * (T + 3) * nh * hd, 5, np.float32)
    arena[:T * nh * hd] = q.reshape(-1)
    a, _ = dev(p.ctx, arena)
    q8hip.kv8_attention(p.ctx, a, 0, (T + 3) * nh * hd, *p.where(T + 3), nh, p.nkv, hd)
    out = a.download(arena.shape, np.float32)[(T + 3) * nh * hd:].reshape(T + 3, nh, hd)
    a.free()
    return out


# ---- pages ---------------------------------------------------------------------------------

class PageState:
    """The page state on the GPU beside the oracle's, with a pool of marked pages."""

    def __init__(self, ctx, nslots, maxpages, npages, P, layers=2, pb=48):
        self.ctx, self.o = ctx, bo.Pages(nslots, maxpages, npages, P)
        self.layers, self.pb, self.npages, self.maxpages, self.P, self.ns = layers, pb, npages, maxpages, P, nslots
        rng = np.random.default_rng(npages)
        self.data = rng.integers(0, 256, (layers, npages, pb), dtype=np.uint8)
        self.pool, _ = dev(ctx, self.data)
        arr = self.o.arrays()
        self.ix, o = dev(ctx, *arr.values(), np.zeros(nslots, np.int32), np.zeros(1, np.int32))
        self.at = dict(zip([*arr, "arg", "live"], [x // 4 for x in o]))

    def state(self):
        return (self.ix, *(self.at[n] for n in ("table", "len", "held", "ref")))

    def arg(self, v):
        self.ix.upload(np.asarray(v, np.int32), 4 * self.at["arg"])
        return self.at["arg"]

    def reserve(self, want):
        q8hip.pages_reserve(self.ctx, *self.state(), self.arg(want), self.ns, self.maxpages, self.npages,
                            self.P, self.pool, 0, self.pb, self.layers, self.npages * self.pb)
        for a, b in self.o.reserve(want):
            self.data[:, b] = self.data[:, a]

    def set_len(self, new):
        q8hip.pages_set_len(self.ctx, *self.state(), self.arg(new), self.ns, self.maxpages, self.npages, self.P)
        self.o.set_len(new)

    def fork(self, src):
        q8hip.pages_fork(self.ctx, *self.state(), self.arg(src), self.ns, self.maxpages, self.npages)
        self.o.fork(src)

    def compact(self):
        q8hip.pages_compact(self.ctx, self.ix, self.at["table"], self.at["held"], self.at["ref"],
                            self.at["live"], self.ns, self.maxpages, self.npages, self.pool, 0, self.pb,
                            self.layers, self.npages * self.pb)
        n, moves = self.o.compact()
        for a, b in moves:
            self.data[:, b] = self.data[:, a]
        assert self.ix.download((1,), np.int32, 4 * self.at["live"])[0] == n

    def check(self):
        for name, want in self.o.arrays().items():
            got = self.ix.download(want.shape, np.int32, 4 * self.at[name])
            assert np.array_equal(got, want), (name, got, want)
        assert np.array_equal(self.pool.download(self.data.shape, np.uint8), self.data)


@pytest.mark.parametrize("nslots,maxpages,npages,P,pb", [(1, 1, 1, 16, 16), (7, 9, 40, 16, 48),
                                                        (70, 67, 900, 64, 16400), (300, 5, 5000, 16, 16)])
def test_pages(ctx, nslots, maxpages, npages, P, pb):
    """Random runs of all page calls against the oracle, the pool too small at
    times, forks of forks, wants past the table."""
    say("pages", nslots, maxpages, npages)
    rng = np.random.default_rng(nslots)
    s = PageState(ctx, nslots, maxpages, npages, P, pb=pb)
    cap = maxpages * P
    for step in range(40):
        kind = rng.integers(0, 4) if step else 0
        if kind == 0:
            ln = np.array(s.o.len)
            want = ln + rng.integers(-3, 2 * P, nslots) * (rng.random(nslots) < 0.5)
            if rng.random() < 0.2:
                want[rng.integers(0, nslots)] = cap + 100
            s.reserve(want.tolist())
            if rng.random() < 0.3:               # fork slots that hold pages ahead, grow both
                src = np.where(rng.random(nslots) < 0.3, rng.integers(0, nslots, nslots), -1)
                s.fork(src.tolist())
                s.check()
                ln = np.array(s.o.len)
                want = ln + rng.integers(0, 3 * P, nslots)
                s.reserve(want.tolist())
                s.check()
            grown = np.minimum(np.maximum(ln, want), [len(r) * P for r in s.o.rows])
            s.set_len(np.where(rng.random(nslots) < 0.8, grown, -1).tolist())
        elif kind == 1:
            new = np.where(rng.random(nslots) < 0.3, rng.integers(0, cap + 1, nslots), -1)
            new[rng.random(nslots) < 0.1] = 0
            s.set_len(new.tolist())
        elif kind == 2:
            src = np.where(rng.random(nslots) < 0.3, rng.integers(-1, nslots + 1, nslots), -1)
            s.fork(src.tolist())
        else:
            s.compact()
        s.check()


def test_pages_many_slots(ctx):
    """The largest slot count: 4096 slots in one call each."""
    say("pages 4096")
    s = PageState(ctx, 4096, 3, 20000, 16, layers=1, pb=16)
    s.reserve([1 + i % 40 for i in range(4096)])
    s.set_len([1 + i % 40 for i in range(4096)])
    s.fork([i - i % 3 if i % 5 else -1 for i in range(4096)])
    s.check()
    s.reserve([n + 1 for n in s.o.len])
    s.set_len([n + 1 if i % 2 else 0 for i, n in enumerate(s.o.len)])
    s.compact()
    s.check()


# ---- together -------------------------------------------------------------------------------

def test_prompts_then_tokens(ctx):
    """Prompts of three sequences through append and packed attention, then token
    steps over the cache with forks, drafts and their return, one captured
    step replayed at every length."""
    say("prompts then tokens")
    rng = np.random.default_rng(21)
    nh, nkv, hd, P, ns, maxpages, npages = 4, 2, 64, 16, 4, 8, 40
    pb = bo.page_bytes(P, nkv, hd)
    s = PageState(ctx, ns, maxpages, npages, P, layers=1, pb=pb)
    c = bo.Cache(npages, P, nkv, hd)
    s.data[:] = c.to_bytes()[None]
    s.pool.upload(s.data)
    ld, Tmax = (nh + 2 * nkv) * hd, 80
    oinv, oy = Tmax * ld, Tmax * ld + 32
    a = ctx.alloc(4 * (oy + Tmax * nh * hd))
    a.upload(inv_freq(hd), 4 * oinv)
    kv = ctx.alloc(2 * 2 * Tmax * nkv * hd)
    # one arena for the calls' int32: cu, then the page state's arrays by copy
    flat = ctx.alloc(4 * (ns + 1 + ns + ns * maxpages))

    def ints(cu):
        st = s.o.arrays()
        flat.upload(np.concatenate([cu, st["len"], st["table"].reshape(-1)]).astype(np.int32))

    def issue(rows):
        where = (s.pool, 0, npages, P, flat, 0, ns + 1, 2 * ns + 1, ns, rows, maxpages)
        q8hip.kv8_append(ctx, a, 0, nh * hd, (nh + nkv) * hd, oinv, 0, *where, nh, nkv, hd, ld=ld, kv=kv,
                         okc_f16=0, ovc_f16=Tmax * nkv * hd)
        q8hip.kv8_attention(ctx, a, 0, oy, *where, nh, nkv, hd, ldq=ld)

    def step(lens, graph=None):
        cu = offsets(lens)
        T = int(cu[-1])
        s.reserve([n + m for n, m in zip(s.o.len, lens)])
        c2 = bo.Cache.from_bytes(s.data[0], P, nkv, hd)
        ints(cu)
        x = rng.standard_normal((Tmax, ld)).astype(np.float32)
        a.upload(x)
        if graph:
            graph.launch()
        else:
            issue(T)
        table, length = s.o.arrays()["table"], np.array(s.o.len)
        q = x[:T, :nh * hd].reshape(T, nh, hd)
        k = x[:T, nh * hd:(nh + nkv) * hd].reshape(T, nkv, hd)
        v = x[:T, (nh + nkv) * hd:].reshape(T, nkv, hd)
        qr, rows = c2.append(q, k, v, inv_freq(hd), cu, length, table)
        y = a.download((T, nh, hd), np.float32, 4 * oy)
        assert max_rel_err(y, c2.attention(qr, cu, length, table)) <= 1e-5
        s.data[0] = c2.to_bytes()
        assert np.array_equal(s.pool.download(s.data.shape, np.uint8), s.data)
        return cu, qr, rows, T

    lens = [37, 0, 5, 20]
    cu, qr, rows, T = step(lens)
    q8hip.attention_packed(ctx, a, 0, kv, 0, Tmax * nkv * hd, a, oy, flat, 0, ns, T, nh, nkv, hd, ldq=ld)
    y = a.download((T, nh, hd), np.float32, 4 * oy)
    assert max_rel_err(y, bo.attention_packed(qr, rows[0], rows[1], cu)) <= 1e-5
    s.set_len(lens)
    s.fork([-1, 0, -1, 0])                       # slots 1 and 3 continue slot 0
    s.check()
    ints(offsets([1, 2, 0, 1]))
    ctx.graph_begin()
    issue(Tmax)                                  # sized for every step below
    g = ctx.graph_end()
    for lens, keep in (([1, 2, 0, 1], [1, 2, 0, 1]), ([4, 4, 4, 4], [1, 4, 2, 3]), ([1, 0, 1, 40], [1, 0, 1, 9]),
                       ([2, 2, 2, 2], [0, 0, 1, 2])):
        for graph in (None, g):
            before = list(s.o.len)
            step(lens, graph)
            s.set_len([n + m for n, m in zip(before, keep)])
            s.check()
    s.set_len([0, -1, -1, 0])
    s.compact()
    s.check()
    g.destroy()


def test_captured_step(ctx):
    """A whole step captured -- pages taken and copied, append, attention, lengths
    advanced -- and replayed at lengths that grow over page ends, a fork among
    them, with eager work between: every replay as the oracle has it."""
    say("captured step")
    rng = np.random.default_rng(60)
    nh, nkv, hd, P, ns, maxpages, npages = 4, 2, 64, 16, 3, 6, 30
    pb, ld = bo.page_bytes(P, nkv, hd), (nh + 2 * nkv) * hd
    o, c = bo.Pages(ns, maxpages, npages, P), bo.Cache(npages, P, nkv, hd)
    pool, _ = dev(ctx, c.to_bytes())
    st = o.arrays()
    names = ["cu", "table", "len", "held", "ref", "want", "source"]
    ix, off = dev(ctx, np.arange(ns + 1, dtype=np.int32), *st.values(), np.zeros(ns, np.int32),
                  np.full(ns, -1, np.int32))
    at = {n: x // 4 for n, x in zip(names, off)}
    oinv, oy = ns * ld, ns * ld + 32
    a = ctx.alloc(4 * (oy + ns * nh * hd))
    a.upload(inv_freq(hd), 4 * oinv)
    state = (ix, at["table"], at["len"], at["held"], at["ref"])

    def issue():
        where = (pool, 0, npages, P, ix, at["cu"], at["len"], at["table"], ns, ns, maxpages)
        q8hip.pages_reserve(ctx, *state, at["want"], ns, maxpages, npages, P, pool, 0, pb)
        q8hip.kv8_append(ctx, a, 0, nh * hd, (nh + nkv) * hd, oinv, 0, *where, nh, nkv, hd, ld=ld)
        q8hip.kv8_attention(ctx, a, 0, oy, *where, nh, nkv, hd, ldq=ld)
        q8hip.pages_set_len(ctx, *state, at["want"], ns, maxpages, npages, P)

    ctx.graph_begin()
    issue()
    g = ctx.graph_end()
    for t in range(40):
        if t == 21:                                  # slots 0 and 2 continue slot 1
            ix.upload(np.array([1, -1, 1], np.int32), 4 * at["source"])
            q8hip.pages_fork(ctx, *state, at["source"], ns, maxpages, npages)
            o.fork([1, -1, 1])
        want = [n + 1 for n in o.len]
        ix.upload(np.array(want, np.int32), 4 * at["want"])
        x = rng.standard_normal((ns, ld)).astype(np.float32) * (1 + t % 3)
        a.upload(x)
        if t % 5 == 4:
            issue()                                  # eager between replays
        else:
            g.launch()
        for f, to in o.reserve(want):
            c.k[to], c.v[to], c.s[to] = c.k[f], c.v[f], c.s[f]
        table, length = o.arrays()["table"], np.array(o.len)
        q, k, v = (y.reshape(ns, -1, hd) for y in np.split(x, [nh * hd, (nh + nkv) * hd], 1))
        qr, _ = c.append(q, k, v, inv_freq(hd), [0, 1, 2, 3], length, table)
        y = a.download((ns, nh, hd), np.float32, 4 * oy)
        assert max_rel_err(y, c.attention(qr, [0, 1, 2, 3], length, table)) <= 1e-5, t
        o.set_len(want)
        for name, ref in o.arrays().items():
            assert np.array_equal(ix.download(ref.shape, np.int32, 4 * at[name]), ref), (t, name)
        assert np.array_equal(pool.download((npages, pb), np.uint8), c.to_bytes()), t
    g.destroy()


def test_far_pages(ctx):
    """Pages beyond 4 GiB: append, attention and compaction at 64-bit offsets."""
    say("far pages")
    rng = np.random.default_rng(61)
    P, nkv, hd, nh = 128, 8, 128, 8
    pb = bo.page_bytes(P, nkv, hd)
    npages = (5 << 30) // pb
    p = Paged(ctx, rng, [3, 1], [200, 500], P, nkv, hd)
    near = p.c.npages
    far = npages - near + np.arange(near)
    p.pool.free()
    p.pool = ctx.alloc(npages * pb)
    p.pool.upload(p.c.to_bytes(), int(far[0]) * pb)
    local = p.table.copy()
    p.table = np.where(local >= 0, local + far[0], -1).astype(np.int32)
    p.upload()
    where = (p.pool, 0, npages, P, p.ix, *p.at, 2, 4, p.maxpages)
    ld = (nh + 2 * nkv) * hd
    x = rng.standard_normal((4, ld)).astype(np.float32)
    a, (_, oinv, oy) = dev(ctx, x, inv_freq(hd), np.zeros((4, nh * hd), np.float32))
    q8hip.kv8_append(ctx, a, 0, nh * hd, (nh + nkv) * hd, oinv // 4, 0, *where, nh, nkv, hd, ld=ld)
    q8hip.kv8_attention(ctx, a, 0, oy // 4, *where, nh, nkv, hd, ldq=ld)
    q, k, v = (y.reshape(4, -1, hd) for y in np.split(x, [nh * hd, (nh + nkv) * hd], 1))
    qr, _ = p.c.append(q, k, v, inv_freq(hd), p.cu, p.old, local)
    ref = p.c.attention(qr, p.cu, p.old, local)
    assert max_rel_err(a.download((4, nh, hd), np.float32, oy), ref) <= 1e-5
    assert np.array_equal(p.pool.download((near, pb), np.uint8, int(far[0]) * pb), p.c.to_bytes())
    held = (local >= 0).sum(1).astype(np.int32)
    ref_counts = np.zeros(npages, np.int32)
    ref_counts[p.table[p.table >= 0]] = 1
    ix, off = dev(ctx, p.table, held, ref_counts, np.zeros(1, np.int32))
    q8hip.pages_compact(ctx, ix, *(x // 4 for x in off), 2, p.maxpages, npages, p.pool, 0, pb)
    n = int(held.sum())
    moved = ix.download(p.table.shape, np.int32)
    order = np.argsort(np.argsort(local[local >= 0]))
    assert np.array_equal(moved[moved >= 0], order)
    assert ix.download((1,), np.int32, off[3])[0] == n
    assert np.array_equal(p.pool.download((n, pb), np.uint8), p.c.to_bytes()[np.sort(local[local >= 0])])
    p.pool.free()


def test_graphs_share_scratch(ctx):
    """Two captured calls that split their keys, replayed in turn on two streams,
    with eager calls between: every replay as the eager result."""
    torch = pytest.importorskip("torch")
    say("graphs share scratch")
    rng = np.random.default_rng(30)
    ps = [Paged(ctx, rng, [1, 1], [5000, 400 + 100 * i], 64, 2, 64) for i in range(2)]
    arenas, eager, graphs = [], [], []
    nh, hd = 8, 64
    for p in ps:
        q = rng.standard_normal((2, nh, hd)).astype(np.float32)
        eager.append(run_cache(p, q))
        a, _ = dev(ctx, np.concatenate([q.reshape(-1), np.zeros(q.size, np.float32)]))
        arenas.append(a)
        ctx.graph_begin()
        q8hip.kv8_attention(ctx, a, 0, q.size, *p.where(2), nh, 2, hd)
        graphs.append(ctx.graph_end())
    streams = [torch.cuda.Stream() for _ in range(2)]
    n = 2 * nh * hd
    for i in range(12):
        for a in arenas:
            a.upload(np.zeros(n, np.float32), 4 * n)
        for st, g in zip(streams if i % 2 else streams[::-1], graphs):
            ctx.set_stream(st.cuda_stream)
            g.launch()
        torch.cuda.synchronize()
        ctx.set_stream(None)
        for a, y in zip(arenas, eager):
            assert np.array_equal(a.download((2, nh, hd), np.float32, 4 * n), y)
        assert np.array_equal(run_cache(ps[i % 2], arenas[i % 2].download((2, nh, hd), np.float32)), eager[i % 2])
    for g in graphs:
        g.destroy()


# ---- a model over several sequences ------------------------------------------------------

class OracleBatch:
    """The float64 model (oracle/model_oracle.py) over the slots of a Q8Batch.  Its
    attention reads the codes that the batch stored, after each has been checked
    against the float64 key or value (a code beside its border may fall either
    way by the linears' error, and would differ for good in a cache of its own)."""

    def __init__(self, spec, tensors, inv, batch):
        from oracle import model_oracle as mo
        self.mo, self.m = mo, mo.OracleModel(spec, tensors, inv, 1)
        self.sp, self.inv, self.b = spec, inv, batch
        self.kv = {}                          # slot -> [layer] -> (k, v) as computed

    def cache(self, L):
        p = self.b.pages
        raw = p.pool.download((p.npages, p.page_bytes), np.uint8, L * p.npages * p.page_bytes)
        return bo.Cache.from_bytes(raw, p.page, p.nkv, p.head_dim)

    def forward(self, slot, ids, packed):
        """Logits of every row of one slot, after the batch's call."""
        from oracle.q8_oracle import embed_gather_np
        sp, mo, lin, t, p = self.sp, self.mo, self.m.lin, self.m.tensors, self.b.pages
        s, hd = len(ids), sp.head_dim
        kv = self.kv.setdefault(slot, [(np.zeros((0, sp.n_kv, hd)),) * 2 for _ in range(sp.layers)])
        n = len(kv[0][0])
        assert p.length[slot] == n + s
        table = p.ix.download((p.slots, p.maxpages), np.int32, 4 * p.at["table"])[slot]
        x = embed_gather_np(t["model.embed_tokens.weight"], np.asarray(ids), sp.hidden, sp.G,
                            sp.scale).astype(np.float64)
        for L in range(sp.layers):
            w = f"model.layers.{L}."
            xn = mo.rmsnorm(x, t[w + "input_layernorm.weight"], sp.eps)
            q, k, v = (lin(w + f"self_attn.{y}_proj.weight", xn) for y in "qkv")
            if sp.qk_norm:
                q = mo.head_rmsnorm(q, t[w + "self_attn.q_norm.weight"], sp.n_heads, hd, sp.eps)
                k = mo.head_rmsnorm(k, t[w + "self_attn.k_norm.weight"], sp.n_kv, hd, sp.eps)
            q, k, v = (y.reshape(s, -1, hd) for y in (q, k, v))
            q, k = (bo.rotate(y, np.arange(n, n + s), self.inv) for y in (q, k))
            kv[L] = tuple(np.concatenate(y) for y in zip(kv[L], (k, v)))
            c = self.cache(L)
            stored = c.values(table, n + s)
            for which, (have, want) in enumerate(zip(stored, kv[L])):
                # half a step of the page's scale for the code, half for each time
                # the scale grew since (3 at most here), one for the border
                step = np.stack([c.s[table[i // p.page], which] for i in range(n + s)])[..., None]
                assert (np.abs(have - want) <= 3 * step + 1e-3 * np.abs(want).max()).all(), (L, which)
            if packed:
                ao = bo.attention_packed(q, k.astype(np.float16), v.astype(np.float16), [0, s])
            else:
                ao = bo.attend(q, *stored, n)
            h = x + lin(w + "self_attn.o_proj.weight", ao.reshape(s, -1))
            z = mo.rmsnorm(h, t[w + "post_attention_layernorm.weight"], sp.eps)
            g, u = lin(w + "mlp.gate_proj.weight", z), lin(w + "mlp.up_proj.weight", z)
            x = h + lin(w + "mlp.down_proj.weight", mo.swiglu(g, u))
        xn = mo.rmsnorm(x, t["model.norm.weight"], sp.eps)
        return lin("model.embed_tokens.weight" if sp.tied else "lm_head.weight", xn)

    def fork(self, dst, src):
        self.kv[dst] = list(self.kv[src])

    def truncate(self, slot, n):
        self.kv[slot] = [(k[:n], v[:n]) for k, v in self.kv[slot]]


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_model_batch(ctx, kind):
    """Prompts of three slots in one pass, token steps of all, a fork, drafts
    with their return, a late prompt beside running slots, release, compaction,
    against the float64 model.

    The bar: from 32 rows on a linear is within 2e-4 of its largest output
    (q8_linear), 4 * 2 + 1 of them follow each other, 1.8e-3; and a score s of q
    and k 2e-4 off each is 4e-4 |s| off, |s| up to 8 here, which a probability
    carries as a factor, 3.2e-3 in each of two layers: together 8.2e-3.  Fewer rows:
    linears within 1e-5, a twentieth of it.  A row at a wrong position, page, head
    or slot is off by its whole size."""
    import sys
    sys.path.insert(0, __file__.rsplit("/", 1)[0])
    from test_model_oracle import qwen_tiny, tiny_model
    from lama32_mojo_amd import batch, model as gm
    say("model batch", kind)
    spec, t, inv = tiny_model() if kind == "llama" else qwen_tiny()
    cfg = gm.Config(spec.hidden, spec.layers, spec.n_heads, spec.n_kv, spec.head_dim, spec.inter,
                    spec.vocab, spec.eps, 500000.0 if kind == "llama" else 1000000.0, 32.0, 1.0, 4.0,
                    8192.0, tied=spec.tied, qk_norm=spec.qk_norm,
                    rope="llama3" if kind == "llama" else "plain")
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    b = batch.Q8Batch(m, slots=4, npages=24, maxlen=160, page=16, max_rows=128)
    o = OracleBatch(spec, t, inv, b)
    rng = np.random.default_rng(1)

    def run(tokens, every=False):
        packed = all(b.pages.length[s] == 0 for s in tokens)
        rows = sum(len(x) for x in tokens.values())
        got = b.forward(tokens, every=every, logits=True)
        for s, ids in tokens.items():
            ref = o.forward(s, ids, packed)
            err = max_rel_err(got[s], ref if every else ref[-1])
            say("slot", s, "rows", len(ids), "of", rows, "err %.1e" % err)
            assert err <= (8.2e-3 if rows >= 32 else 4.1e-4), (s, len(ids))
    draw = lambda n: rng.integers(0, spec.vocab, n).tolist()
    run({0: draw(37), 1: draw(5), 3: draw(20)})              # packed prompts, 62 rows
    for _ in range(3):
        run({s: draw(1) for s in (0, 1, 3)})
    b.fork({2: 0})
    o.fork(2, 0)
    run({s: draw(1) for s in range(4)})
    run({0: draw(4), 2: draw(3), 3: draw(1)}, every=True)    # drafts; slot 0 keeps 2 of 4
    b.truncate({0: b.pages.length[0] - 2})
    o.truncate(0, b.pages.length[0])
    run({0: draw(2), 1: draw(30)})                           # a chunk beside a step
    b.truncate({1: 0})
    o.truncate(1, 0)
    live = b.compact()
    assert live == sum(-(-b.pages.length[s] // 16) for s in (0, 2, 3)) - 2    # two shared pages
    run({1: draw(40)})
    run({s: draw(1) for s in range(4)})
    # the ids are the argmax of the logits
    ids = b.forward({0: [3], 2: [5]})
    assert set(ids) == {0, 2} and all(0 <= x < spec.vocab for x in ids.values())
    with pytest.raises(RuntimeError, match="pages full"):
        b.forward({0: draw(120)})
    assert b.pages.length[0] == b.pages.ix.download((1,), np.int32, 4 * b.pages.at["len"])[0]
    with pytest.raises(ValueError):
        b.forward({0: draw(129)})
    with pytest.raises(ValueError):
        b.forward({0: []})
    b.close()
    m.close()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_packed_long(ctx, act):
    """A prompt long enough for the 8-wave blocks, beside 17 and more sequences."""
    say("packed long", act)
    rng = np.random.default_rng(40)
    for lens in ([4500], [1] * 20):
        q, k, v = packed_inputs(rng, lens, 2, 1, 128)
        q = bf16_to_f32(bf16_bits(q)) if act == "bf16" else q
        pick = np.unique(np.r_[0:3, 60:70, 2040:2050, 4490:4500]) if len(lens) == 1 else np.arange(20)
        y = run_packed(ctx, q, k, v, offsets(lens), act)
        for r in pick:
            a = 0 if len(lens) == 1 else r
            ref = bo.attend(q[r:r + 1].astype(np.float64), k[a:r + 1].astype(np.float64),
                            v[a:r + 1].astype(np.float64), r - a)[0]
            bar = 1e-5 * np.abs(ref).max() if act == "f32" else \
                2.0 ** -8 * np.abs(ref) + 2.0 ** -11 * np.abs(v.astype(np.float64)).max() + 1e-5
            assert (np.abs(y[r] - ref) <= bar).all(), r


def test_append_scale_rounding(ctx):
    """The scale is the f32 product of the largest value and f32(1 / 127), whose last
    bit differs from the quotient's for the values taken here: scales and codes equal
    the oracle's, codes beside a border of either among them."""
    say("append scale rounding")
    rng = np.random.default_rng(77)
    one = np.float32(1) / np.float32(127)
    top = rng.uniform(1, 8, 4000).astype(np.float32)
    top = top[top * one != top / np.float32(127)][:32]
    assert top.size == 32
    p = Paged(ctx, rng, [16] * 32, [0] * 32, 16, 1, 64)
    q, k, v = (rng.standard_normal((p.rows, 1, 64)).astype(np.float32) for _ in range(3))
    for i, t in enumerate(top):
        x = v[16 * i:16 * i + 16]
        s = t * one
        x[:] = ((rng.integers(-126, 126, x.shape) + 0.5) * float(s)).astype(np.float32)
        x[np.abs(x) > t] = 0
        x[0, 0, 0] = t
    check_append(p, q, k, v)


def test_pages_full_beside_shared(ctx):
    """A fork that would grow inside a shared page needs one of its own: with none
    free the reservation is refused, though the slot's held pages would do.  With
    one of the two slots released the other grows in place."""
    from lama32_mojo_amd.batch import Pages
    say("pages full beside shared")
    p = Pages(ctx, 2, 1, 1, 16, 1, 1, 64)
    p.reserve([10, 0])
    p.set_len([10, 0])
    p.fork([-1, 0])
    for want in ([11, 10], [10, 11], [11, 11]):
        with pytest.raises(RuntimeError, match="pages full"):
            p.reserve(want)
        assert p.length == [10, 10]
        assert p.ix.download((2,), np.int32, 4 * p.at["table"]).tolist() == [0, 0]
    p.reserve([10, 10])                                      # nothing grows
    p.set_len([0, -1])
    p.reserve([0, 16])
    p.set_len([-1, 16])
    assert p.ix.download((2,), np.int32, 4 * p.at["table"]).tolist() == [-1, 0]
    # room for one copy: slot 0 gets it, slot 1 then has the old page alone
    p2 = Pages(ctx, 2, 2, 2, 16, 1, 1, 64)
    p2.reserve([10, 0])
    p2.set_len([10, 0])
    p2.fork([-1, 0])
    p2.reserve([11, 10])
    p2.set_len([11, 10])
    p2.reserve([11, 11])
    assert sorted(p2.ix.download((2, 2), np.int32, 4 * p2.at["table"])[:, 0].tolist()) == [0, 1]
    p2.close()
    p.close()
