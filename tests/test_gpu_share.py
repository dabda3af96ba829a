"""q8_kv8_share and q8_kv8_attention_shared against the restatements in oracle/.

What is shared: equal.  The attention: 1e-5 of the largest output, the bar of
q8_kv8_attention -- operands' terms add up to the f32 values, so what is left are f32
sums of some thousand terms, one exp2 a probability, and one more factor of 1 + 2^-23
for each of the two parts that a row joins."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import batch_oracle as bo
from oracle import serving_oracle as so
from oracle.q8_oracle import max_rel_err

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


class Step:
    """Sequences over the first `shared[g]` pages of group g (-1: none) and pages of their
    own; lens rows each behind `tail` tokens of their own."""

    def __init__(self, rng, lens, group, shared, tail, P, nkv, hd, spare=3):
        self.lens, self.P, self.nkv, self.hd = lens, P, nkv, hd
        ns = len(lens)
        heads = {g: n for g, n in enumerate(shared)}
        self.old = np.array([heads.get(g, 0) * P + t for g, t in zip(group, tail)], np.int32)
        mine = [-(-(int(o) + n) // P) - heads.get(g, 0) for o, n, g in zip(self.old, lens, group)]
        npages = sum(shared) + sum(mine) + spare
        self.c = bo.Cache(npages, P, nkv, hd).random(rng)
        ids = rng.permutation(npages).tolist()
        take = lambda n: [ids.pop() for _ in range(n)]                         # noqa: E731
        first = {g: take(n) for g, n in heads.items()}
        rows = [first.get(g, []) + take(m) for g, m in zip(group, mine)]
        self.maxpages = max(len(r) for r in rows) + 1
        self.table = np.array([r + [-1] * (self.maxpages - len(r)) for r in rows], np.int32)
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.T = int(self.cu[-1])
        self.ns = ns

    def ints(self, rows):
        n = q8hip.kv8_share_ints(self.ns, rows)
        return np.concatenate([self.cu, self.old, self.table.reshape(-1), np.full(n + 1, -77, np.int32)]).astype(np.int32)

    def run(self, ctx, q, dead=0, off=0, extra=0, share=True, spoil=None, far=0):
        """far: pages in front of the ones in use."""
        T, nh, hd = q.shape
        rows, ld, ns = T + dead, nh * hd + extra, self.ns
        arena = np.full(off + rows * (ld + nh * hd) + 4, 5, np.float32)
        arena[off:off + T * ld].reshape(T, ld)[:, :nh * hd] = q.reshape(T, -1)
        ints = self.ints(rows)
        table = ints[2 * ns + 1:2 * ns + 1 + ns * self.maxpages]
        table[table >= 0] += far
        at = 2 * ns + 1 + ns * self.maxpages
        a, ix, pool = ctx.alloc(arena.nbytes), ctx.alloc(ints.nbytes), self.c.to_bytes()
        page_bytes, npages = pool.nbytes // self.c.npages, self.c.npages + far
        pages = ctx.alloc(npages * page_bytes)
        a.upload(arena)
        ix.upload(ints)
        pages.upload(pool, far * page_bytes)
        arrays = (ix, 0, ns + 1, 2 * ns + 1, ns, rows, self.maxpages)
        q8hip.kv8_share(ctx, *arrays, npages, self.P, at)
        now = ix.download(ints.shape, np.int32)
        assert np.array_equal(now[:at], ints[:at]) and now[-1] == -77
        self.found = now[at + 1:at + 1 + ns].tolist(), now[at + 1 + ns:at + 1 + 2 * ns].tolist()
        self.groups = int(now[at])
        if spoil is not None:
            ix.upload(spoil(now[at:-1]).astype(np.int32), 4 * at)
        oy = off + rows * ld
        args = (ctx, a, off, oy, pages, 0, npages, self.P, *arrays, nh, self.nkv, hd)
        if share:
            q8hip.kv8_attention_shared(*args, at, ldq=ld if extra else 0)
        else:
            q8hip.kv8_attention(*args, ldq=ld if extra else 0)
        got = a.download(arena.shape, np.float32)
        y = got[oy:oy + T * nh * hd].reshape(T, nh, hd).copy()
        got[oy:oy + T * nh * hd] = arena[oy:oy + T * nh * hd]
        assert np.array_equal(got, arena)                      # nothing else, nor rows behind the last
        for b in (a, ix, pages):
            b.free()
        return y

    def ref(self, q):
        return self.c.attention(q, self.cu, self.old, self.table)

    def check(self, ctx, q, **kw):
        y = self.run(ctx, q, **kw)
        group, tokens = so.share(self.cu, self.old, self.table, self.P, self.c.npages)
        assert self.found == (group, tokens) and self.groups == max(group, default=-1) + 1
        ref = self.ref(q)
        assert max_rel_err(y, ref) <= 1e-5
        return y


def queries(rng, T, nh, hd):
    return (rng.standard_normal((T, nh, hd)) * np.exp(rng.standard_normal((T, 1, 1)) * 0.5)).astype(np.float32)


HEADS = [(8, 2, 64), (8, 2, 128), (3, 3, 128), (5, 1, 64), (16, 1, 64), (2, 2, 64)]


@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_groups(ctx, P, nh, nkv, hd):
    """Two groups and sequences of their own, slots mixed, one to several rows, none."""
    say("shared", P, nh, nkv, hd)
    rng = np.random.default_rng(P + nh + hd)
    group = [0, 1, -1, 0, 0, 1, -1, 0, 1, 0]
    lens = [1, 2, 1, 5, 0, 1, 3, 1, 1, 2]
    tail = [0, 5, 40, 17, 3, 64, 0, 130, 1, P]
    s = Step(rng, lens, group, [5, 300 // P + 1], tail, P, nkv, hd)
    q = queries(rng, s.T, nh, hd)
    y = s.check(ctx, q, dead=2)
    assert np.array_equal(s.run(ctx, q, off=3, extra=7), y)
    assert np.array_equal(s.run(ctx, q), y)                   # the same bits again
    assert max_rel_err(y, s.run(ctx, q, share=False)) <= 1e-5


@pytest.mark.parametrize("ns", [2, 15, 16, 17, 33, 64, 100])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128)])
def test_group_sizes(ctx, ns, nh, nkv, hd):
    """One group over one to several row tiles, prefixes that end inside a unit of 64 keys."""
    say("shared sizes", ns, hd)
    rng = np.random.default_rng(ns)
    for pages in (1, 3, 21):
        s = Step(rng, [1] * ns, [0] * ns, [pages], rng.integers(0, 50, ns), 16, nkv, hd)
        s.check(ctx, queries(rng, s.T, nh, hd))


def test_long_prefix(ctx):
    say("shared long")
    rng = np.random.default_rng(2)
    for P, n in ((128, 40), (16, 300)):
        s = Step(rng, [1, 1, 2, 1], [0, 0, 0, -1], [n], [700, 0, 3, 900], P, 2, 64)
        s.check(ctx, queries(rng, s.T, 4, 64))


@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("hd", [64, 128])
def test_wide_tables(ctx, P, hd):
    """Tables with room for many more pages than are named, the groups' part a launch of its own."""
    say("shared wide", P, hd)
    rng = np.random.default_rng(P + hd)
    s = Step(rng, [1, 3, 1, 0, 1, 2], [0, 1, 0, 0, 1, -1], [9, 300 // P + 1], [70, 0, 3, 5, 200, 90], P, 2, hd)
    more = 64 * 9000 // P - s.maxpages
    s.table = np.concatenate([s.table, np.full((s.ns, more), -1, np.int32)], axis=1)
    s.maxpages += more
    s.check(ctx, queries(rng, s.T, 8, hd), dead=1, off=3, extra=7)


def test_far_pages(ctx):
    """Page ids whose bytes lie beyond 4 GiB: the bits of the same pages in front."""
    say("shared far")
    rng = np.random.default_rng(12)
    s = Step(rng, [1, 2, 1, 1], [0, 0, -1, 0], [5], [70, 3, 90, 0], 64, 2, 128)
    q = queries(rng, s.T, 8, 128)
    far = (1 << 32) // q8hip.kv8_page_bytes(64, 2, 128) + 1
    assert np.array_equal(s.run(ctx, q, far=far), s.check(ctx, q))


def test_drafts_in_wide_groups(ctx):
    """Row tiles of 32 and 64 columns for the sequences' own tokens."""
    say("shared drafts")
    rng = np.random.default_rng(3)
    for lens in ([6] * 9, [20, 1, 30, 9], [70, 70]):
        ns = len(lens)
        s = Step(rng, lens, [0] * ns, [9], rng.integers(0, 90, ns), 16, 2, 64)
        s.check(ctx, queries(rng, s.T, 8, 64))


def test_which_pages(ctx):
    """Chains of forks, prefixes of other lengths, leaders without rows, missing pages,
    lengths inside the shared pages."""
    say("shared which")
    rng = np.random.default_rng(4)
    s = Step(rng, [1] * 12, [-1] * 12, [], [100] * 12, 16, 2, 64)
    tab = s.table
    for i in (1, 2, 3):
        tab[i, :6] = tab[0, :6]                    # four with all six whole pages
    tab[4, :2] = tab[0, :2]                        # one that left early
    tab[6, :3] = tab[5, :3]
    tab[7, :3] = tab[5, :3]                        # three with three
    tab[8, :] = tab[9, :]
    s.old[9] = 40                                  # two whole pages of the shared ones
    tab[10, 0] = tab[11, 0] = -1                   # equal, and missing
    q = queries(rng, s.T, 4, 64)
    y = s.run(ctx, q)
    group, tokens = so.share(s.cu, s.old, tab, 16, s.c.npages)
    assert s.found == (group, tokens)
    assert group[:4] == [0] * 4 and tokens[0] == 96 and group[4] == -1 and group[5:8] == [1] * 3
    assert tokens[5] == 48 and group[8:10] == [2, 2] and tokens[8] == 32 and group[10:] == [-1, -1]
    ref = s.ref(q)
    assert np.array_equal(np.isnan(y), np.isnan(ref)) and np.isnan(y[10:]).all()
    assert max_rel_err(y[:10], ref[:10]) <= 1e-5
    s.lens[0], s.cu = 0, np.concatenate([[0, 0], np.arange(1, 12)]).astype(np.int32)
    s.T = 11
    tab[3, 3] = s.c.npages                         # a missing page inside what three have in common
    tab[1, 3] = tab[2, 3] = s.c.npages
    y = s.run(ctx, q[1:])
    assert s.found == so.share(s.cu, s.old, tab, 16, s.c.npages) and s.found[0][0] == -1
    ref = s.ref(q[1:])
    assert np.array_equal(np.isnan(y), np.isnan(ref)) and np.isnan(y[:3]).all()
    f = ~np.isnan(ref)
    assert max_rel_err(y[f], ref[f]) <= 1e-5


def test_many(ctx):
    """1024 sequences in one group, in more groups than are taken, each for itself."""
    say("shared many")
    rng = np.random.default_rng(5)
    s = Step(rng, [1] * 1024, [0] * 1024, [2], [i % 9 for i in range(1024)], 16, 1, 64)
    s.check(ctx, queries(rng, s.T, 1, 64))
    s = Step(rng, [1] * 300, [i % 100 for i in range(300)], [1 + i % 3 for i in range(100)], [1] * 300, 16, 1, 64)
    s.check(ctx, queries(rng, s.T, 1, 64))
    assert s.groups == 64
    s = Step(rng, [1] * 70, [-1] * 70, [], [i % 90 for i in range(70)], 16, 1, 64)
    s.check(ctx, queries(rng, s.T, 2, 64))
    assert s.groups == 0


def test_more_rows_than_records(ctx):
    """Where the groups' records do not fit, the sequences read their own tokens."""
    say("shared no room")
    rng = np.random.default_rng(6)
    s = Step(rng, [1500, 1500], [0, 0], [2], [3, 5], 16, 2, 128)
    q = queries(rng, s.T, 32, 128)
    y = s.run(ctx, q)
    assert s.groups == 1
    assert np.array_equal(y, s.run(ctx, q, share=False))


def test_spans_and_nan(ctx):
    """q whose dims span many powers of two; a page of NaN scale among the shared ones and
    among a sequence's own; infinite q."""
    say("shared spans")
    rng = np.random.default_rng(7)
    s = Step(rng, [1] * 6, [0, 0, 0, 0, 1, 1], [4, 5], [20, 3, 0, 40, 5, 6], 16, 2, 64)
    q = queries(rng, s.T, 4, 64)
    q[:, :, 7] *= 2.0 ** 40
    s.c.k[:, :, :, 7] = 0
    s.check(ctx, q)
    q = queries(rng, s.T, 4, 64)
    s.c.s[s.table[0, 2], 0, 1] = np.nan            # a shared page of group 0, head 1
    s.c.s[s.table[4, 5], 1, 0] = np.nan            # sequence 4's own page
    q[5, 0, 3] = np.inf
    y, ref = s.run(ctx, q), s.ref(q)
    assert np.isnan(y[:4, 2:]).all() and not np.isnan(y[:4, :2]).any()
    assert np.isnan(y[4, :2]).all() and np.isnan(y[5, 0]).all()
    f = np.isfinite(ref) & np.isfinite(y)
    f[5, 0] = False
    assert max_rel_err(y[f], ref[f]) <= 1e-5 and f[4, 2:].all() and f[5, 1:].all()


def test_nonsense(ctx):
    """Whatever cu, lengths, tables and what is shared hold, only out is written."""
    say("shared nonsense")
    rng = np.random.default_rng(8)
    big = lambda n: rng.integers(-2 ** 31, 2 ** 31 - 1, n)                     # noqa: E731
    s = Step(rng, [1] * 20, [0] * 20, [4], [9] * 20, 16, 2, 64)
    q = queries(rng, s.T, 4, 64)
    s.run(ctx, q, spoil=lambda v: big(len(v)))
    s.run(ctx, q, spoil=lambda v: np.concatenate([[2 ** 31 - 1], rng.integers(0, 20, len(v) - 1)]))
    s.run(ctx, q, spoil=lambda v: np.where(rng.random(len(v)) < 0.3, rng.integers(-3, 300, len(v)), v))
    s.old = big(20).astype(np.int32)
    s.run(ctx, q)
    s.table = rng.integers(-1, s.c.npages + 1, s.table.shape).astype(np.int32)
    s.run(ctx, q)
    s.cu = np.array([0, 20] * 10 + [0], np.int32)
    s.run(ctx, q)
    s.cu = big(21).astype(np.int32)
    s.run(ctx, q)


def test_captured(ctx):
    """A captured step finds what is shared anew at every replay."""
    say("shared captured")
    rng = np.random.default_rng(9)
    P, nkv, hd, nh, ns = 16, 2, 64, 8, 12
    steps = []
    for groups in ([0] * 12, [0, 1] * 6, [-1] * 12, [0, 0, 0, -1, -1, -1, 1, 1, 1, 1, 1, 1]):
        steps.append(Step(rng, [1] * ns, groups, [6, 3][:max(groups) + 1], rng.integers(0, 60, ns), P, nkv, hd, spare=0))
    npages, maxpages = max(s.c.npages for s in steps), max(s.maxpages for s in steps)
    pb = q8hip.kv8_page_bytes(P, nkv, hd)
    at = 2 * ns + 1 + ns * maxpages
    a, pages, ix = ctx.alloc(8 * ns * nh * hd), ctx.alloc(npages * pb), ctx.alloc(4 * (at + q8hip.kv8_share_ints(ns, ns)))
    arrays = (ix, 0, ns + 1, 2 * ns + 1, ns, ns, maxpages)
    ctx.graph_begin()
    q8hip.kv8_share(ctx, *arrays, npages, P, at)
    for _ in range(2):
        q8hip.kv8_attention_shared(ctx, a, 0, ns * nh * hd, pages, 0, npages, P, *arrays, nh, nkv, hd, at)
    g = ctx.graph_end()
    for s in steps * 2:
        q = queries(rng, ns, nh, hd)
        tab = np.full((ns, maxpages), -1, np.int32)
        tab[:, :s.maxpages] = s.table
        a.upload(q)
        pages.upload(s.c.to_bytes())
        ix.upload(np.concatenate([s.cu, s.old, tab.reshape(-1)]).astype(np.int32))
        g.launch()
        y = a.download((ns, nh, hd), np.float32, 4 * ns * nh * hd)
        assert max_rel_err(y, s.ref(q)) <= 1e-5
        steps[0].run(ctx, queries(rng, ns, nh, hd))            # the same scratch, eagerly
    g.destroy()
    for b in (a, pages, ix):
        b.free()
