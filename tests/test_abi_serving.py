"""Argument checks of the calls for requests that differ, on a host-only context:
what each refuses and with which status; valid calls reach the device step."""

import pytest

from lama32_mojo_amd import q8hip
from lama32_mojo_amd.q8hip import (Q8_ERR_ARG, Q8_ERR_NODEVICE, Q8_ERR_RANGE, Q8_ERR_SHAPE, Q8Error)


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
