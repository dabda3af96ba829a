"""Tokens that are returned (drafts that were rejected): what they leave in the page
they shared, and the fork that avoids it."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import batch_oracle as bo
from oracle.q8_oracle import max_rel_err
from test_gpu_batch import PageState, dev, inv_freq, offsets, say

pytestmark = pytest.mark.gpu

NH, NKV, HD, P, NS, MAXPAGES, NPAGES = 4, 2, 64, 16, 2, 4, 8


class Slots:
    """Two slots of one layer, beside the oracle's."""

    def __init__(self, ctx):
        self.ctx = ctx
        self.s = PageState(ctx, NS, MAXPAGES, NPAGES, P, layers=1, pb=bo.page_bytes(P, NKV, HD))
        self.s.data[:] = bo.Cache(NPAGES, P, NKV, HD).to_bytes()[None]
        self.s.pool.upload(self.s.data)

    def append(self, x, slot=0):
        """Rows x [n, NH + 2 NKV, HD] behind a slot: its outputs over the cache."""
        s, n = self.s, len(x)
        lens = [n if i == slot else 0 for i in range(NS)]
        s.reserve([a + b for a, b in zip(s.o.len, lens)])
        st, cu = s.o.arrays(), offsets(lens)
        ix, _ = dev(self.ctx, cu, st["len"], st["table"])
        a, (_, oinv, oy) = dev(self.ctx, x, inv_freq(HD), np.zeros((n, NH, HD), np.float32))
        where = (s.pool, 0, NPAGES, P, ix, 0, NS + 1, 2 * NS + 1, NS, n, MAXPAGES)
        ld = (NH + 2 * NKV) * HD
        q8hip.kv8_append(self.ctx, a, 0, NH * HD, (NH + NKV) * HD, oinv // 4, 0, *where, NH, NKV, HD, ld=ld)
        q8hip.kv8_attention(self.ctx, a, 0, oy // 4, *where, NH, NKV, HD, ldq=ld)
        c = bo.Cache.from_bytes(s.data[0], P, NKV, HD)
        q, k, v = np.split(x, [NH, NH + NKV], 1)
        qr, _ = c.append(q, k, v, inv_freq(HD), cu, st["len"], st["table"])
        ref = c.attention(qr, cu, st["len"], st["table"])
        y = a.download((n, NH, HD), np.float32, oy)
        assert np.array_equal(np.isnan(y), np.isnan(ref))
        if np.isfinite(ref).any():
            assert max_rel_err(y[np.isfinite(ref)], ref[np.isfinite(ref)]) <= 1e-5
        got = bo.Cache.from_bytes(s.pool.download(s.data.shape, np.uint8)[0], P, NKV, HD)
        for name in ("k", "v", "s"):
            assert np.array_equal(getattr(got, name), getattr(c, name), equal_nan=True), name
        s.data[0] = c.to_bytes()
        s.set_len([a + b for a, b in zip(s.o.len, lens)])
        return y

    def scales(self, slot=0):
        """The scales of the page that the slot's last token is in."""
        s = self.s
        return bo.Cache.from_bytes(s.data[0], P, NKV, HD).s[s.o.rows[slot][(s.o.len[slot] - 1) // P]]


@pytest.mark.parametrize("kind", ["outlier", "nan", "inf"])
def test_returned_tokens(ctx, kind):
    """Returned by length alone, a draft leaves the page at its own scale: an outlier's
    coarse one, or NaN, for as long as the page holds older tokens.  A slot forked
    before the draft and continued from the fork is as if there had been none."""
    say("returned tokens", kind)
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, NH + 2 * NKV, HD)).astype(np.float32)
    bad = rng.standard_normal((2, NH + 2 * NKV, HD)).astype(np.float32)
    bad[1, NH:] = {"outlier": 1000.0, "nan": np.nan, "inf": np.inf}[kind]
    plain, back, fork = (Slots(ctx) for _ in range(3))
    for c in (plain, back, fork):
        c.append(x[:5])
    fork.s.fork([-1, 0])
    for c in (back, fork):
        c.append(bad)
    back.s.set_len([5, -1])
    fork.s.fork([1, -1])
    fork.s.set_len([-1, 0])
    want = [plain.append(x[5 + i:6 + i]) for i in range(2)]
    for i in range(2):
        assert np.array_equal(fork.append(x[5 + i:6 + i]), want[i])
    assert np.array_equal(fork.scales(), plain.scales())
    y = back.append(x[5:6])
    if kind == "outlier":
        assert (back.scales() > 100 * plain.scales()).all() and np.isfinite(y).all()
    else:
        assert np.isnan(back.scales()).all() and np.isnan(y).all()
    # a page that holds no older token starts anew
    back.s.set_len([0, -1])
    assert np.isfinite(back.append(x[:5])).all()
    back.append(x[5:7])
    assert np.array_equal(back.scales(), plain.scales())
