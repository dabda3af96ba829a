"""q8_kv8_attention_shared where the groups' records are large beside the scratch: many KV
heads, many groups, many sequences.

That a group's tokens are read by way of its leader is seen by hiding them: after
q8_kv8_share the table entries of the other members' shared pages name no page, so a sequence
that read its own table would be NaN.  The bar is that of tests/test_gpu_share.py, 1e-5."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import serving_oracle as so
from oracle.q8_oracle import max_rel_err
from test_gpu_share import Step, queries, say

pytestmark = pytest.mark.gpu


def hidden(ctx, monkeypatch, s, q):
    """(outputs with the members' shared pages hidden, members behind the first of each group
    by group)."""
    group, tokens = so.share(s.cu, s.old, s.table, s.P, s.c.npages)
    table, members, seen = s.table.copy(), {}, set()
    for i, g in enumerate(group):
        if g in seen:
            table[i, :tokens[i] // s.P] = -1
            members.setdefault(g, []).append(i)
        elif g >= 0:
            seen.add(g)
    call = q8hip.kv8_attention_shared

    def hide(ctx, a, oq, oy, pages, opages, npages, page, ix, ocu, olen, otab, *rest, **kw):
        ix.upload(table, 4 * otab)
        call(ctx, a, oq, oy, pages, opages, npages, page, ix, ocu, olen, otab, *rest, **kw)
    with monkeypatch.context() as m:
        m.setattr(q8hip, "kv8_attention_shared", hide)
        y = s.run(ctx, q)
    assert s.found == (group, tokens)
    return y, members


@pytest.mark.parametrize("ns", [64, 77, 78, 128])
@pytest.mark.parametrize("nh,nkv", [(32, 32), (64, 32), (40, 40)])
def test_many_kv_heads(ctx, monkeypatch, ns, nh, nkv):
    """One group of a step's sequences is read once whatever the number of KV heads."""
    say("shared KV heads", ns, nh, nkv)
    rng = np.random.default_rng(ns + nh)
    s = Step(rng, [1] * ns, [0] * ns, [21], rng.integers(0, 40, ns), 16, nkv, 128)
    q = queries(rng, s.T, nh, 128)
    y, members = hidden(ctx, monkeypatch, s, q)
    assert len(members[0]) == ns - 1
    ref = s.ref(q)
    assert max_rel_err(y, ref) <= 1e-5
    assert max_rel_err(s.run(ctx, q), ref) <= 1e-5


@pytest.mark.parametrize("P,nkv,hd,ns,most", [(128, 32, 128, 90, 1), (64, 32, 128, 60, 5), (16, 32, 64, 700, 3)])
def test_pages_and_rows(ctx, monkeypatch, P, nkv, hd, ns, most):
    """The same with other pages and heads, several rows a sequence, tables with room to spare,
    rows behind the last sequence and q inside wider rows."""
    say("shared limit", P, hd, ns)
    rng = np.random.default_rng(ns)
    lens = rng.integers(1, most + 1, ns).tolist()
    s = Step(rng, lens, [0 if i % 5 else -1 for i in range(ns)], [2], rng.integers(0, 20, ns), P, nkv, hd)
    s.table = np.concatenate([s.table, np.full((ns, 300), -1, np.int32)], axis=1)
    s.maxpages += 300
    q = queries(rng, s.T, nkv, hd)
    y, members = hidden(ctx, monkeypatch, s, q)
    ref = s.ref(q)
    assert members and max_rel_err(y, ref) <= 1e-5
    assert np.array_equal(s.check(ctx, q, dead=3, off=3, extra=7), s.run(ctx, q, dead=3))


def outside(y, members, groups):
    """The groups whose members read their own tables; every other group is read by its leader."""
    nan = np.isnan(y).any((1, 2))
    out = [g for g in range(groups) if nan[members[g]].any()]
    assert np.array_equal(np.flatnonzero(nan), sorted(i for g in out for i in members[g]))
    return out, nan


def test_groups_that_have_room(ctx, monkeypatch):
    """More groups than there is room for: the first ones are read once, the members of the
    others read their own tokens."""
    say("shared room for some")
    rng = np.random.default_rng(1)
    groups, ns = 14, 14 * 12
    s = Step(rng, [1] * ns, [i % groups for i in range(ns)], [40] * groups, [2] * ns, 16, 128, 128)
    q = queries(rng, s.T, 128, 128)
    y, members = hidden(ctx, monkeypatch, s, q)
    out, nan = outside(y, members, groups)
    assert 0 < len(out) < groups and out == list(range(groups - len(out), groups))
    ref = s.ref(q)
    assert max_rel_err(y[~nan], ref[~nan]) <= 1e-5
    assert max_rel_err(s.run(ctx, q), ref) <= 1e-5


def test_groups_that_save_enough(ctx, monkeypatch):
    """Where there is not room for whatever groups there may be, small ones are left out: a row
    tile of 64 columns costs as much as four sequences."""
    say("shared groups that save")
    rng = np.random.default_rng(2)
    sizes, pages = (3, 20, 4, 40, 5, 11), (90, 4, 60, 21, 100, 30)
    group = [g for g, n in enumerate(sizes) for _ in range(n)]
    ns = len(group)
    s = Step(rng, [1] * ns, group, list(pages), rng.integers(0, 20, ns), 16, 32, 128)
    q = queries(rng, s.T, 32, 128)
    y, members = hidden(ctx, monkeypatch, s, q)
    out, nan = outside(y, members, len(sizes))
    assert out == [g for g, n in enumerate(sizes) if n <= 4]
    assert 0 < len(out) < len(sizes)
    ref = s.ref(q)
    assert max_rel_err(y[~nan], ref[~nan]) <= 1e-5
    assert max_rel_err(s.run(ctx, q), ref) <= 1e-5


def test_nonsense(ctx):
    """Whatever is found shared, only out is written, with a limit on the groups' blocks too."""
    say("shared room nonsense")
    rng = np.random.default_rng(3)
    ns = 90
    s = Step(rng, [1] * ns, [i % 7 for i in range(ns)], [30, 2, 9, 40, 1, 5, 7], rng.integers(0, 20, ns), 16, 32, 128)
    q = queries(rng, s.T, 32, 128)
    big = lambda n: rng.integers(-2 ** 31, 2 ** 31 - 1, n)                     # noqa: E731
    for spoil in (lambda v: big(len(v)), lambda v: np.concatenate([[64], rng.integers(0, ns, len(v) - 1)]),
                  lambda v: np.concatenate([[7], rng.integers(0, 2000, len(v) - 1)]),
                  lambda v: np.where(rng.random(len(v)) < 0.3, rng.integers(-3, 700, len(v)), v)):
        s.run(ctx, q, spoil=spoil)
    s.check(ctx, q)


def test_captured(ctx):
    """A captured call with a limit, replayed with other groups: as the eager one."""
    say("shared room captured")
    rng = np.random.default_rng(4)
    P, nkv, hd, nh, ns = 16, 32, 128, 32, 80
    steps = [Step(rng, [1] * ns, [i % g for i in range(ns)], [6 + 3 * i for i in range(g)], rng.integers(0, 30, ns), P, nkv,
                  hd, spare=0) for g in (1, 3, 16, 40)]
    npages, maxpages = max(s.c.npages for s in steps), max(s.maxpages for s in steps)
    at = 2 * ns + 1 + ns * maxpages
    a, ix = ctx.alloc(8 * ns * nh * hd), ctx.alloc(4 * (at + q8hip.kv8_share_ints(ns, ns)))
    pages = ctx.alloc(npages * q8hip.kv8_page_bytes(P, nkv, hd))
    arrays = (ix, 0, ns + 1, 2 * ns + 1, ns, ns, maxpages)

    def call():
        q8hip.kv8_share(ctx, *arrays, npages, P, at)
        q8hip.kv8_attention_shared(ctx, a, 0, ns * nh * hd, pages, 0, npages, P, *arrays, nh, nkv, hd, at)
    ctx.graph_begin()
    call()
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
        a.upload(np.zeros(ns * nh * hd, np.float32), 4 * ns * nh * hd)
        call()
        assert np.array_equal(y, a.download((ns, nh, hd), np.float32, 4 * ns * nh * hd))
        assert max_rel_err(y, s.ref(q)) <= 1e-5
    g.destroy()
    for b in (a, pages, ix):
        b.free()


@pytest.mark.parametrize("nkv", [253, 500, 512])
def test_most_kv_heads(ctx, nkv):
    """As many KV heads as a call may have, in two and three sequences."""
    say("shared most KV heads", nkv)
    rng = np.random.default_rng(nkv)
    for ns in (2, 3):
        s = Step(rng, [1] * ns, [0] * ns, [2], [3, 20, 0][:ns], 16, nkv, 128)
        q = queries(rng, s.T, nkv, 128)
        y = s.run(ctx, q)
        assert max_rel_err(y, s.ref(q)) <= 1e-5
        assert max_rel_err(y, s.run(ctx, q, share=False)) <= 1e-5


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("ns", [700, 1024])
def test_many_sequences(ctx, ns, wide):
    """Heads of 128 with as many sequences as may share, both parts in one launch and (wide
    tables) in two."""
    say("shared many sequences", ns, wide)
    rng = np.random.default_rng(ns)
    s = Step(rng, [1] * ns, [i % 3 - 1 for i in range(ns)], [2, 5], rng.integers(0, 20, ns), 16, 1, 128)
    if wide:
        more = 64 * 400 // 16 - s.maxpages
        s.table = np.concatenate([s.table, np.full((ns, more), -1, np.int32)], axis=1)
        s.maxpages += more
    s.check(ctx, queries(rng, s.T, 2, 128))
