"""Argument checks of the calls for requests that differ, on a host-only context:
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


def test_sample(hctx):
    R, n = 4, 100
    a, ids = hctx.alloc(4 * (R * n + 5 * R)), hctx.alloc(4 * 2 * R)

    def call(ox=0, rows=R, n=n, op=R * n, k=0, oid=R, lp=a, olp=R * n + 4 * R, ldx=0, a=a, ids=ids):
        return code(q8hip.sample, hctx, a, ox, rows, n, op, ids, k, oid, lp, olp, ldx)
    assert call() == call(lp=None, olp=1 << 40) == call(rows=0) == call(ldx=n) == Q8_ERR_NODEVICE
    assert call(rows=-1) == call(n=0) == call(rows=1, n=(1 << 22) + 1) == call(ldx=n - 1) == Q8_ERR_SHAPE
    assert call(rows=(1 << 24) + 1) == call(ldx=1 << 31) == Q8_ERR_SHAPE
    assert call(ox=6 * R) == call(op=R * n + R + 1) == call(k=R + 1) == call(oid=R + 1) == Q8_ERR_RANGE
    assert call(olp=R * n + 4 * R + 1) == call(ldx=n + 10) == call(ox=1 << 62) == Q8_ERR_RANGE
    assert call(oid=0) == call(oid=3) == call(olp=0) == call(olp=R * n) == Q8_ERR_ARG    # outputs over inputs
    big = hctx.alloc(4 * (R * n + 8 * R))
    assert call(a=big, ids=big, k=R * n + 5 * R, oid=R * n + 6 * R, lp=big, olp=R * n + 4 * R) == Q8_ERR_NODEVICE
    assert code(q8hip.sample, hctx, big, 0, R, n, R * n, big, R * n + 5 * R, 2) == Q8_ERR_ARG
    rc = hctx._lib.q8_sample(hctx.h, None, 0, 0, R, n, 0, ids.h, 0, R, None, 0)
    assert rc == Q8_ERR_ARG
    assert hctx._lib.q8_sample(None, a.h, 0, 0, R, n, R * n, ids.h, 0, R, None, 0) == Q8_ERR_ARG


def test_lora(hctx):
    T, m, na, R, widths = 9, 64, 3, 16, [40, 8]
    n = sum(widths)
    sa, sb = 2 * R * m, n * R
    a, w, ix = hctx.alloc(4 * (T * (m + 2 * n) + na)), hctx.alloc(2 * na * (sa + sb)), hctx.alloc(4 * (4 + 3 + na))

    def call(oa=0, sa=sa, ob=na * sa, sb=sb, na=na, R=R, ox=0, obase=T * m, oy=T * (m + n), osc=T * (m + 2 * n),
             ocu=0, oid=4, orank=7, nseq=3, rows=T, m=m, widths=widths, dtype="bf16", ldx=0, ldy=0, w=w, a=a):
        return code(q8hip.lora, hctx, w, oa, sa, ob, sb, na, R, a, ox, obase, oy, osc, ix, ocu, oid, orank, nseq, rows,
                    m, widths, dtype, ldx, ldy)
    assert call() == call(obase=T * (m + n)) == call(rows=0) == call(nseq=0) == call(R=13) == Q8_ERR_NODEVICE
    assert call(dtype=3) == Q8_ERR_ARG
    assert call(m=60) == call(m=0) == call(na=0) == call(R=0) == call(widths=[0]) == Q8_ERR_SHAPE
    assert call(widths=[40, 0, 8]) == call(sa=sa - 8) == call(sb=sb - 8) == call(rows=-1) == Q8_ERR_SHAPE
    assert call(R=24) == call(ldx=m - 1) == call(ldy=n - 1) == call(widths=[40, 16]) == Q8_ERR_SHAPE
    assert call(R=257) == call(na=4097) == call(nseq=4097) == Q8_ERR_UNSUPPORTED
    assert call(dtype="f32") == call(na=4) == call(ob=na * sa + 8) == call(oa=1 << 62) == Q8_ERR_RANGE
    assert call(osc=T * (m + 2 * n) + 1) == call(rows=10) == call(ldx=m + 300) == call(ldy=n + 9) == Q8_ERR_RANGE
    assert call(orank=8) == call(nseq=7) == call(ocu=9) == Q8_ERR_RANGE
    assert call(oy=0) == call(ldx=m + 100) == call(oy=T * m + 1) == call(oy=T * (m + n) - n) == Q8_ERR_ARG
    small = hctx.alloc(2 * na * (sa + sb) + 4)
    assert call(oa=1, w=small, ob=na * sa + 2) == call(ob=na * sa + 1, w=small) == Q8_ERR_UNSUPPORTED
    with pytest.raises(ValueError):
        call(widths=[8, 8, 8, 8])
    with pytest.raises(ValueError):
        call(widths=[])


def test_share(hctx):
    ns, T, maxpages, npages, page, nh, nkv, hd = 3, 9, 4, 5, 16, 4, 2, 64
    n = q8hip.kv8_share_ints(ns, T)
    assert q8hip.kv8_share_ints(1024, 1 << 22) > 1 << 22
    for bad in ((1025, 1), (-1, 1), (1, -1), (1, (1 << 22) + 1)):
        with pytest.raises(Q8Error):
            q8hip.kv8_share_ints(*bad)
    at = 2 * ns + 1 + ns * maxpages
    ix, a = hctx.alloc(4 * (at + n)), hctx.alloc(4 * 2 * T * nh * hd)
    pages = hctx.alloc(npages * q8hip.kv8_page_bytes(page, nkv, hd))

    def find(ocu=0, olen=ns + 1, otab=2 * ns + 1, ns=ns, rows=T, maxpages=maxpages, npages=npages, page=page, at=at):
        return code(q8hip.kv8_share, hctx, ix, ocu, olen, otab, ns, rows, maxpages, npages, page, at)
    assert find() == find(rows=0) == find(ns=0) == Q8_ERR_NODEVICE
    assert find(page=24) == find(ns=1025) == Q8_ERR_UNSUPPORTED
    assert find(ns=-1) == find(rows=-1) == find(maxpages=0) == find(npages=0) == Q8_ERR_SHAPE
    assert find(rows=(1 << 22) + 1) == find(maxpages=1 << 27) == Q8_ERR_SHAPE
    assert find(at=at + 1) == find(rows=T + 1) == find(otab=at + n) == Q8_ERR_RANGE
    assert find(at=at - 1) == find(at=0) == find(ocu=at + 2) == Q8_ERR_ARG

    def call(oy=T * nh * hd, ns=ns, at=at, rows=T, a=a, hd=hd, ix=ix):
        return code(q8hip.kv8_attention_shared, hctx, a, 0, oy, pages, 0, npages, page, ix, 0, ns + 1, 2 * ns + 1, ns,
                    rows, maxpages, nh, nkv, hd, at)
    assert call() == call(rows=0) == Q8_ERR_NODEVICE
    assert call(at=at + 1) == call(at=1 << 62) == Q8_ERR_RANGE
    assert call(oy=0) == Q8_ERR_ARG
    assert call(hd=96) == Q8_ERR_UNSUPPORTED
    many = hctx.alloc(1 << 24)
    assert call(ns=1025, ix=many, at=100000) == Q8_ERR_UNSUPPORTED and call(ns=1024, ix=many, at=100000) == Q8_ERR_NODEVICE
    assert call(a=many, ix=many, oy=(1 << 20), at=(1 << 20) + 5) == Q8_ERR_ARG
