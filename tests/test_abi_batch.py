"""Argument checks of the calls over several sequences on a host-only context:
what each refuses and with which status; valid calls reach the device step."""

import pytest

from lama32_mojo_amd import q8hip
from lama32_mojo_amd.q8hip import (Q8_ERR_ARG, Q8_ERR_NODEVICE, Q8_ERR_RANGE, Q8_ERR_SHAPE,
                                   Q8_ERR_UNSUPPORTED, Q8Error)


@pytest.fixture
def hctx():
    c = q8hip.Context(q8hip.Q8_DEVICE_NONE)
    yield c
    c.close()


def code(fn, *args, **kw):
    try:
        fn(*args, **kw)
    except Q8Error as e:
        return e.code
    return 0


def test_page_bytes():
    assert q8hip.kv8_page_bytes(64, 8, 128) == 2 * 8 * 64 * 128 + 64
    assert q8hip.kv8_page_bytes(16, 1, 64) == 2 * 16 * 64 + 16
    for bad in ((8, 8, 128), (64, 0, 128), (64, 8, 96), (48, 8, 64)):
        with pytest.raises(Q8Error):
            q8hip.kv8_page_bytes(*bad)


def test_attention_packed(hctx):
    T, nh, nkv, hd = 40, 8, 2, 64
    q, out = hctx.alloc(4 * T * nh * hd), hctx.alloc(4 * T * nh * hd)
    kv, ix = hctx.alloc(2 * 2 * T * nkv * hd), hctx.alloc(4 * 8)

    def call(oq=0, okc=0, ovc=T * nkv * hd, o=out, oy=0, ocu=0, nseq=7, rows=T, nh=nh, nkv=nkv, hd=hd,
             act="f32", ldq=0):
        return code(q8hip.attention_packed, hctx, q, oq, kv, okc, ovc, o, oy, ix, ocu, nseq, rows, nh,
                    nkv, hd, act, ldq)
    assert call() == Q8_ERR_NODEVICE
    assert call(nseq=0) == call(rows=0) == Q8_ERR_NODEVICE
    assert call(act=3) == Q8_ERR_ARG
    assert call(act="bf16", oy=0, o=q, oq=T * nh * hd) == Q8_ERR_NODEVICE      # halves of one buffer
    assert call(act="bf16", oy=8, o=q, oq=T * nh * hd - 8) == Q8_ERR_ARG
    assert call(o=q) == call(o=kv, rows=4) == Q8_ERR_ARG
    assert call(oq=4) == call(oy=4) == call(okc=8, ovc=T * nkv * hd + 8) == Q8_ERR_RANGE
    assert call(nseq=8) == call(ocu=1) == Q8_ERR_RANGE
    assert call(ldq=nh * hd - 4) == call(rows=-1) == call(nseq=-1) == Q8_ERR_SHAPE
    assert call(rows=1, ldq=nh * hd + 2) == call(rows=1, oq=1) == call(rows=1, okc=4) == Q8_ERR_UNSUPPORTED
    assert call(nh=7) == Q8_ERR_SHAPE
    assert call(hd=96, rows=4) == call(hd=32) == Q8_ERR_UNSUPPORTED
    assert call(nh=129, nkv=1, rows=1) == Q8_ERR_UNSUPPORTED
    assert call(rows=1 << 25) == Q8_ERR_SHAPE
    # more row tiles than a launch has blocks
    q, out, kv = (hctx.alloc(1 << 41) for _ in range(3))
    T = 1 << 24
    assert call(nh=8, nkv=1, rows=T, ovc=T * 64, o=out) == Q8_ERR_NODEVICE
    assert call(nh=128, nkv=1, rows=T, ovc=T * 64, o=out) == Q8_ERR_SHAPE


def cache(hctx, npages=5, page=16, nkv=2, hd=64, nseq=3, maxpages=4, rows=9):
    pages = hctx.alloc(npages * q8hip.kv8_page_bytes(page, nkv, hd))
    ix = hctx.alloc(4 * (nseq + 1 + nseq + nseq * maxpages))
    return pages, ix


def test_kv8_append(hctx):
    T, nh, nkv, hd = 9, 4, 2, 64
    ld = (nh + 2 * nkv) * hd
    pages, ix = cache(hctx)
    a, kv = hctx.alloc(4 * (T * (ld + nh * hd) + 32)), hctx.alloc(2 * 2 * T * nkv * hd)

    def call(oq=0, ok=nh * hd, ov=(nh + nkv) * hd, oinv=T * (ld + nh * hd), oqr=T * ld, p=pages, op=0,
             npages=5, page=16, ocu=0, olen=4, otab=7, nseq=3, rows=T, maxpages=4, nh=nh, nkv=nkv,
             hd=hd, ld=ld, ldr=None, kv=None, okc=0, ovc=T * nkv * hd):
        return code(q8hip.kv8_append, hctx, a, oq, ok, ov, oinv, oqr, p, op, npages, page, ix, ocu,
                    olen, otab, nseq, rows, maxpages, nh, nkv, hd, ld, ldr, kv, okc, ovc)
    assert call() == call(oqr=0) == call(kv=kv) == Q8_ERR_NODEVICE
    assert call(rows=0) == call(nseq=0) == Q8_ERR_NODEVICE
    assert call(oqr=4) == call(oqr=0, ldr=ld + 4, rows=8) == Q8_ERR_ARG        # over q at another stride
    assert call(oqr=0, ok=64) == Q8_ERR_ARG                                    # k inside q's columns
    assert call(oinv=T * ld + 8) == call(oqr=0, oinv=8) == Q8_ERR_ARG
    assert call(kv=kv, ovc=8) == call(kv=pages, ovc=4 * T * hd) == Q8_ERR_ARG
    assert call(p=a, npages=1, nseq=1) == Q8_ERR_ARG                           # pages over the arena
    assert call(kv=kv, ovc=T * nkv * hd + 1) == call(oinv=T * (ld + nh * hd) + 1) == Q8_ERR_RANGE
    assert call(npages=6) == call(op=16) == call(otab=8) == Q8_ERR_RANGE
    assert call(page=48) == call(hd=96, ld=0) == Q8_ERR_UNSUPPORTED
    assert call(nseq=5000) == Q8_ERR_UNSUPPORTED
    assert call(npages=0) == call(maxpages=0) == call(ld=8) == call(nh=3) == call(rows=-1) == Q8_ERR_SHAPE
    assert call(maxpages=1 << 27) == Q8_ERR_SHAPE


def test_kv8_attention(hctx):
    T, nh, nkv, hd = 9, 4, 2, 64
    pages, ix = cache(hctx)
    a = hctx.alloc(4 * 2 * T * nh * hd)

    def call(oq=0, oy=T * nh * hd, p=pages, op=0, npages=5, page=16, ocu=0, olen=4, otab=7, nseq=3,
             rows=T, maxpages=4, nh=nh, nkv=nkv, hd=hd, ldq=0, ix=ix):
        return code(q8hip.kv8_attention, hctx, a, oq, oy, p, op, npages, page, ix, ocu, olen, otab,
                    nseq, rows, maxpages, nh, nkv, hd, ldq)
    assert call() == call(rows=0) == call(nseq=0) == Q8_ERR_NODEVICE
    assert call(oy=T * nh * hd - 4) == call(oy=0) == call(p=a, op=4 * T * nh * hd, npages=1) == Q8_ERR_ARG
    assert call(ix=a, ocu=T * nh * hd) == Q8_ERR_ARG
    assert call(oy=T * nh * hd + 4) == Q8_ERR_RANGE
    assert call(npages=6) == call(olen=19) == Q8_ERR_RANGE
    assert call(page=8) == call(nseq=4097) == call(hd=32) == Q8_ERR_UNSUPPORTED
    assert call(npages=0) == call(nh=5) == call(ldq=8) == Q8_ERR_SHAPE
    assert call(rows=(1 << 22) + 1) == Q8_ERR_SHAPE
    assert call(nkv=513, nh=513, p=hctx.alloc(1 << 30)) == Q8_ERR_UNSUPPORTED
    # more units of work than an int32 counts
    big = hctx.alloc(8 << 32)
    assert call(ix=big, maxpages=1 << 26, nseq=50, otab=100, olen=52, ocu=0) == Q8_ERR_NODEVICE
    assert call(ix=big, maxpages=1 << 26, nseq=64, otab=200, olen=100, ocu=0) == Q8_ERR_SHAPE


def test_pages(hctx):
    ns, mp, npg, pb = 3, 4, 6, 64
    ix, pool = hctx.alloc(4 * 64), hctx.alloc(2 * npg * pb)
    o = dict(otab=0, olen=12, oheld=15, oref=18, ox=24)

    def state(kw):
        s = {**o, **kw}
        return [s[k] for k in ("otab", "olen", "oheld", "oref", "ox")]

    def reserve(ns=ns, mp=mp, npg=npg, page=16, pool=pool, op=0, pb=pb, layers=2, ls=npg * pb, **kw):
        return code(q8hip.pages_reserve, hctx, ix, *state(kw), ns, mp, npg, page, pool, op, pb, layers, ls)

    def set_len(ns=ns, mp=mp, npg=npg, page=16, **kw):
        return code(q8hip.pages_set_len, hctx, ix, *state(kw), ns, mp, npg, page)

    def fork(ns=ns, mp=mp, npg=npg, **kw):
        return code(q8hip.pages_fork, hctx, ix, *state(kw), ns, mp, npg)

    def compact(ns=ns, mp=mp, npg=npg, pool=pool, op=0, pb=pb, layers=2, ls=npg * pb, **kw):
        s = {**o, **kw}
        return code(q8hip.pages_compact, hctx, ix, s["otab"], s["oheld"], s["oref"], s["ox"], ns, mp, npg,
                    pool, op, pb, layers, ls)
    for f in (reserve, set_len, fork, compact):
        assert f() == f(ns=0) == Q8_ERR_NODEVICE, f
        assert f(ns=-1) == f(mp=0) == f(npg=0) == Q8_ERR_SHAPE, f
        assert f(ns=5000) == Q8_ERR_UNSUPPORTED, f
        assert f(oref=60) == f(otab=60) == f(ox=64) == Q8_ERR_RANGE, f
        assert f(oref=14) == f(ox=18) == Q8_ERR_ARG, f               # arrays over one another
    for f in (reserve, compact):
        assert f(layers=3) == f(op=16) == Q8_ERR_RANGE, f
        assert f(layers=0) == f(pb=0) == f(ls=npg * pb - 16) == Q8_ERR_SHAPE, f
        assert f(pb=24, ls=npg * 32) == f(layers=1, op=8) == Q8_ERR_UNSUPPORTED, f
        assert f(pool=ix, pb=16, layers=1, npg=2) == Q8_ERR_ARG, f   # the pool over the state
        assert f(layers=1, ls=0) == Q8_ERR_NODEVICE, f
    assert reserve(page=0) == set_len(page=-1) == set_len(mp=1 << 25) == Q8_ERR_SHAPE
    ix = hctx.alloc(1 << 30)
    assert reserve(npg=6 << 20, ox=7 << 20) == compact(npg=6 << 20, ox=7 << 20) == Q8_ERR_UNSUPPORTED
