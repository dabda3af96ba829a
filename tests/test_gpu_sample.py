"""q8_sample against the float64 restatement in oracle/serving_oracle.py.

Ids are equal: the kernel's running sums differ from float64's by about 2^-41 of a
weight each, so an id could differ only where u or a border lies within some 1e-12 of a
running sum; the borders that are met exactly here (equal logits at T = 1, whose weights
are 1) are exact in both.  Log-probabilities: half a step of f32, 2^-24 of the value,
and 1e-11 for those sums."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle.serving_oracle import sample_row

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def run(ctx, x, temp, k, top_p, min_p, u, pad=0, extra=0, lp=True):
    """x [R, n]; settings per row; logits at element `pad`, rows `extra` floats apart."""
    R, n = x.shape
    ld = n + extra
    arena = np.full(pad + R * ld + 5 * R, np.nan, np.float32)
    rows = np.full((R, ld), 1e30, np.float32)
    rows[:, :n] = x
    arena[pad:pad + R * ld] = rows.reshape(-1)
    at = pad + R * ld
    for i, v in enumerate((temp, top_p, min_p, u)):
        arena[at + i * R:at + (i + 1) * R] = v
    ints = np.concatenate([np.broadcast_to(np.asarray(k, np.int32), R), np.full(R + 1, -7, np.int32)])
    a, ib = ctx.alloc(arena.nbytes), ctx.alloc(ints.nbytes)
    a.upload(arena)
    ib.upload(ints)
    q8hip.sample(ctx, a, pad, R, n, at, ib, 0, R, lp=a if lp else None, olp=at + 4 * R,
                 ldx=ld if extra else 0)
    got = ib.download(ints.shape, np.int32)
    now = a.download(arena.shape, np.float32)
    a.free()
    ib.free()
    assert np.array_equal(now[:at + 4 * R], arena[:at + 4 * R], equal_nan=True) and got[-1] == -7
    assert np.array_equal(got[:R], ints[:R])
    return got[R:2 * R], now[at + 4 * R:]


def check(ctx, x, temp=1.0, k=0, top_p=1.0, min_p=0.0, u=0.5, **kw):
    R = len(x)
    full = [np.broadcast_to(np.asarray(v), R) for v in (temp, k, top_p, min_p, u)]
    ids, lp = run(ctx, x, full[0], full[1], *full[2:], **kw)
    for r in range(R):
        want, wlp = sample_row(x[r], *(v[r] for v in full))
        assert ids[r] == want, (r, ids[r], want, [v[r] for v in full])
        if np.isinf(wlp):
            assert lp[r] == wlp
        else:
            assert abs(float(lp[r]) - wlp) <= 2.0 ** -24 * abs(wlp) + 1e-11, (r, lp[r], wlp)
    return ids


SETS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05),
        (0.6, 20, 0.95, 0.01), (1.3, 1000, 1.0, 0.0), (2.0, 3, 0.3, 0.4), (0.05, 0, 0.999, 0.0), (1.0, 1, 1.0, 0.0),
        (30.0, 0, 0.5, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 10 ** 9, 1.5, -1.0), (-1.0, 5, 0.5, 0.5)]


@pytest.mark.parametrize("n", [1, 2, 5, 63, 64, 1000, 4097, 8192, 8193, 32003, 128256])
def test_sizes(ctx, n):
    say("sample", n)
    rng = np.random.default_rng(n)
    R = 2 * len(SETS)
    x = (rng.standard_normal((R, n)) * rng.uniform(0.5, 4, (R, 1))).astype(np.float32)
    for r in range(R):
        x[r, rng.integers(0, n, 5)] += rng.uniform(0, 8, 5).astype(np.float32)
        if r % 3 == 2 and n > 1:
            x[r, rng.random(n) < 0.5] = -np.inf
    sets = [SETS[r % len(SETS)] for r in range(R)]
    cols = [np.array([s[i] for s in sets]) for i in range(4)]
    u = rng.random(R).astype(np.float32)
    check(ctx, x, *cols, u=u)
    check(ctx, x, *cols, u=rng.random(R).astype(np.float32), pad=3, extra=5)


@pytest.mark.parametrize("rows", [1, 2, 37, 300])
def test_rows(ctx, rows):
    """One row takes many blocks, many rows one each: the same ids either way."""
    say("sample rows", rows)
    rng = np.random.default_rng(rows)
    n = 40000 if rows < 300 else 9000
    x = (rng.standard_normal((rows, n)) * 2).astype(np.float32)
    sets = [SETS[r % len(SETS)] for r in range(rows)]
    u = rng.random(rows).astype(np.float32)
    ids = check(ctx, x, *(np.array([s[i] for s in sets]) for i in range(4)), u=u)
    one = [run(ctx, x[r:r + 1], *(np.array([v]) for v in (sets[r][0], sets[r][1], *sets[r][2:], u[r])))[0][0]
           for r in range(min(rows, 15))]
    assert one == ids[:15].tolist()


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.25, 0.5, 0.999, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, np.nan])
def test_ends_of_u(ctx, u):
    say("sample u", u)
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((len(SETS), 700)) * 2).astype(np.float32)
    check(ctx, x, *(np.array([s[i] for s in SETS]) for i in range(4)), u=u)


@pytest.mark.parametrize("n", [4, 4096, 20000, 70000])
def test_equal_logits(ctx, n):
    """All tokens alike: lowest indices first, borders met exactly; more members of one
    bin than LDS holds."""
    say("sample equal", n)
    x = np.full((7, n), 1.0, np.float32)
    ids = check(ctx, x, k=[0, 3, 0, n // 2, 0, n - 1, 0], top_p=[1, 1, 0.5, 0.5, 1, 1, 0.25], min_p=[0, 0, 0, 0, 1, 0, 0],
                u=[0.0, 0.5, 0.75, 0.5, 1 - 2.0 ** -24, 0.25, 0.0])
    assert ids[0] == 0 and ids[1] == 1
    x[3, n // 2:] = 0.0
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0                                # zeros of both signs are equal
    check(ctx, x, k=[0, 3, 0, n // 2 + 1, 0, n - 1, 0], u=0.77)


def test_two_values(ctx):
    """Many ties at the border of top-k and of the mass."""
    say("sample ties")
    rng = np.random.default_rng(8)
    x = rng.integers(0, 3, (30, 9000)).astype(np.float32)
    k = rng.integers(1, 9000, 30)
    check(ctx, x, k=k, u=rng.random(30).astype(np.float32))
    check(ctx, x, k=k, top_p=rng.random(30).astype(np.float32), u=rng.random(30).astype(np.float32))


def test_infinities_and_nan(ctx):
    say("sample infinities")
    n = 9000
    rng = np.random.default_rng(4)
    x = rng.standard_normal((12, n)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = np.nan
    x[2, 17] = -3.0
    x[3, [5, 100, 8999]] = np.inf
    x[4, ::2] = np.nan
    x[5] = -np.inf
    x[5, 8500] = -3e38
    x[6, 8999] = 3e38
    x[7] = np.float32(np.finfo(np.float32).min)
    x[8, [0, 8191, 8192]] = np.inf
    x[9, 1:] = -np.inf
    u = np.full(12, 0.6, np.float32)
    for kw in (dict(), dict(k=2), dict(top_p=0.5), dict(min_p=0.1), dict(temp=0.0), dict(k=2, top_p=0.9, min_p=0.2)):
        ids = check(ctx, x, u=u, **kw)
        assert ids[0] == ids[1] == -1 and ids[2] == 17 and ids[5] == 8500 and ids[6] == 8999 and ids[9] == 0


@pytest.mark.parametrize("temp", [1e-45, 1e-30, 1e-3, 1e3, 1e30, np.inf, np.nan])
def test_temperatures(ctx, temp):
    say("sample temperature", temp)
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((6, 9000)) * 3).astype(np.float32)
    x[1] *= 1e30
    x[2, 4000] = -np.inf
    x[3, 10:20] = np.inf
    u = rng.random(6).astype(np.float32)
    check(ctx, x, temp=temp, u=u)
    check(ctx, x, temp=temp, k=7, top_p=0.8, u=u)


def test_far_tail(ctx):
    """Tokens whose weight underflows are as if they were not there."""
    say("sample tail")
    x = np.full((3, 10000), -500.0, np.float32)
    x[:, 9000:9003] = [1.0, 2.0, 0.0]
    check(ctx, x, k=[0, 1000, 2], top_p=[1, 0.999, 1], u=[1 - 2.0 ** -24, 0.99, 0.9])


def test_frequencies(ctx):
    """Over even u the ids come as often as their probabilities say, within one."""
    say("sample frequencies")
    rng = np.random.default_rng(9)
    row = rng.standard_normal(50).astype(np.float32)
    R = 4096
    u = ((np.arange(R) + 0.5) / R).astype(np.float32)
    ids, lp = run(ctx, np.tile(row, (R, 1)), 1.0, 0, 1.0, 0.0, u)
    p = np.exp(row.astype(np.float64))
    p /= p.sum()
    assert (np.abs(np.bincount(ids, minlength=50) - R * p) <= 1.0).all()
    assert np.allclose(np.exp(lp.astype(np.float64)), p[ids], rtol=1e-6)


def test_captured(ctx):
    """Replayed with new logits, settings and random numbers, beside other work of the
    context's scratch, and without log-probabilities."""
    say("sample captured")
    rng = np.random.default_rng(10)
    R, n = 5, 9001
    a, ib = ctx.alloc(4 * (R * n + 4 * R)), ctx.alloc(8 * R)
    ib.upload(np.array([0, 50, 0, 3, 0] + [0] * R, np.int32))

    def fill():
        x = (rng.standard_normal((R, n)) * 2).astype(np.float32)
        par = np.array([[1.0, 0.8, 0.7, 1.0, 0.0], [1, 0.9, 0.8, 1, 1], [0, 0, 0, 0, 0.1], rng.random(R)], np.float32)
        a.upload(np.concatenate([x.reshape(-1), par.reshape(-1)]))
        return x, par
    fill()
    ctx.graph_begin()
    q8hip.sample(ctx, a, 0, R, n, R * n, ib, 0, R)
    g = ctx.graph_end()
    for _ in range(4):
        x, par = fill()
        g.launch()
        got = ib.download((R,), np.int32, 4 * R)
        for r, k in enumerate([0, 50, 0, 3, 0]):
            assert got[r] == sample_row(x[r], par[0, r], k, *par[1:, r])[0]
        run(ctx, x, *par[0:1], 0, *par[1:])                     # the same scratch, eagerly
    g.destroy()
    a.free()
    ib.free()


def test_largest_row(ctx):
    """2^22 logits, spread and all alike."""
    say("sample largest")
    rng = np.random.default_rng(15)
    x = (rng.standard_normal((2, 1 << 22)) * 3).astype(np.float32)
    x[1] = 0.5
    for kw in (dict(), dict(k=40, top_p=0.9), dict(top_p=0.95)):
        check(ctx, x, u=np.array([0.3, 0.7], np.float32), **kw)


def test_far_rows(ctx):
    """Rows whose bytes lie beyond 4 GiB: the ids of the same rows side by side."""
    say("sample far")
    rng = np.random.default_rng(14)
    R, n, ld = 3, 20001, (1 << 29) + 3
    x = (rng.standard_normal((R, n)) * 3).astype(np.float32)
    par = np.array([[1.0, 0.7, 1.3], [0.9, 1.0, 0.95], [0, 0.01, 0], rng.random(R)], np.float32)
    k = np.array([0, 0, 500], np.int32)
    a, near, ids = ctx.alloc(4 * (2 * ld + n)), ctx.alloc(4 * (R * n + 4 * R)), ctx.alloc(4 * 3 * R)
    near.upload(np.concatenate([x.reshape(-1), par.reshape(-1)]))
    for r in range(R):
        a.upload(x[r], 4 * r * ld)
    a.upload(par.reshape(-1), 4 * (n + 5))                   # (between the rows)
    ids.upload(k)
    q8hip.sample(ctx, near, 0, R, n, R * n, ids, 0, R)
    q8hip.sample(ctx, a, 0, R, n, n + 5, ids, 0, 2 * R, ldx=ld)
    got = ids.download((3, R), np.int32)
    assert np.array_equal(got[1], got[2]) and (got[1] >= 0).all()
    for b in (a, near, ids):
        b.free()


def test_many_rows(ctx):
    """More rows than a launch's grid holds."""
    say("sample many rows")
    rng = np.random.default_rng(11)
    R = 70000
    x = rng.standard_normal((R, 3)).astype(np.float32)
    u = rng.random(R).astype(np.float32)
    ids, _ = run(ctx, x, 1.0, 2, 1.0, 0.0, u)
    order = np.argsort(-x, kind="stable")
    v = np.take_along_axis(x, order, 1).astype(np.float64)
    p = 1 / (1 + np.exp(v[:, 1] - v[:, 0]))
    assert np.array_equal(ids, np.where(u < p, order[:, 0], order[:, 1]))
