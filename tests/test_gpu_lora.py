"""q8_lora against the float64 restatement in oracle/serving_oracle.py.

Bar of an element: S, the sum of the magnitudes that it is made of, times 2^-24 times the
f32 additions that one value passes through.  Those are at most 3 per step of 32 of m
(three bf16 terms, six for f32 adapters), the parts of K that are joined (16 at most),
3 (6) per 32 of the rank, and a dozen around them; the terms of x, A x and f32 weights add
up to the f32 values, and products below 2^-24 that f32 adapters leave out are 3 more."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle.serving_oracle import lora

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def up8(r):
    return (r + 7) // 8 * 8


class Setup:
    def __init__(self, rng, lens, ids, ranks, m, widths, dtype="bf16", max_rank=None, gap=0, dead=0):
        self.lens, self.ids, self.ranks, self.m, self.widths, self.dtype = lens, ids, ranks, m, widths, dtype
        n, parts, self.max_rank = sum(widths), len(widths), max_rank or max(max(ranks), 1)
        R, na = up8(self.max_rank), len(ranks)
        align = 8
        self.sa, self.sb = parts * R * m + align * gap, (n * R + align * gap + 7) // 8 * 8
        w = np.full(na * (self.sa + self.sb), 1e4, np.float32)       # what nothing should read
        self.A, self.B = [], []
        for i, r in enumerate(ranks):
            if r <= 0:
                self.A.append(None)
                self.B.append(None)
                continue
            A = np.zeros((parts, up8(r), m), np.float32)
            B = np.zeros((n, up8(r)), np.float32)
            A[:, :r] = rng.standard_normal((parts, r, m)) / np.sqrt(m)
            B[:, :r] = rng.standard_normal((n, r)) * 0.3
            if dtype == "bf16":
                A, B = ((bf16(v).astype(np.uint32) << 16).view(np.float32) for v in (A, B))
            w[i * self.sa:i * self.sa + A.size] = A.reshape(-1)
            at = na * self.sa + i * self.sb
            w[at:at + B.size] = B.reshape(-1)
            self.A.append(A[:, :r].reshape(-1, m))
            self.B.append(B[:, :r])
        self.w = bf16(w) if dtype == "bf16" else w
        self.T = sum(lens)
        self.rows = self.T + dead
        self.x = (rng.standard_normal((self.rows, m)) * np.exp(rng.standard_normal((self.rows, 1)))).astype(np.float32)
        self.base = rng.standard_normal((self.rows, n)).astype(np.float32)
        self.scale = rng.uniform(0.5, 2, na).astype(np.float32)
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)

    def run(self, ctx, in_place=False, pad=0, ex=0, ey=0):
        m, n, rows, na = self.m, sum(self.widths), self.rows, len(self.ranks)
        lx, ly = m + ex, n + ey
        arena = np.full(pad + rows * (lx + 2 * ly) + na, 123.0, np.float32)
        ox, ob = pad, pad + rows * lx
        oy, osc = ob + rows * ly, ob + 2 * rows * ly
        arena[ox:ob].reshape(rows, lx)[:, :m] = self.x
        arena[ob:oy].reshape(rows, ly)[:, :n] = self.base
        arena[osc:] = self.scale
        ints = np.concatenate([self.cu, self.ids, self.ranks]).astype(np.int32)
        a, w, ix = ctx.alloc(arena.nbytes), ctx.alloc(self.w.nbytes), ctx.alloc(ints.nbytes)
        a.upload(arena)
        w.upload(self.w)
        ix.upload(ints)
        ns = len(self.lens)
        q8hip.lora(ctx, w, 0, self.sa, na * self.sa, self.sb, na, self.max_rank, a, ox, ob, ob if in_place else oy,
                   osc, ix, 0, ns + 1, 2 * ns + 1, ns, rows, m, self.widths, dtype=self.dtype,
                   ldx=lx if ex else 0, ldy=ly if ey else 0)
        now = a.download(arena.shape, np.float32)
        for b in (a, w, ix):
            b.free()
        out = ob if in_place else oy
        y = now[out:out + rows * ly].reshape(rows, ly)[:, :n].copy()
        # nothing else is written, nor rows behind the last sequence
        now[out:out + rows * ly].reshape(rows, ly)[:self.T, :n] = arena[out:out + rows * ly].reshape(rows, ly)[:self.T, :n]
        assert np.array_equal(now, arena, equal_nan=True)
        return y[:self.T]

    def ref(self):
        y, size = lora(self.x, self.base, self.cu, self.ids, self.A, self.B, self.scale, self.widths)
        adds = (3 if self.dtype == "bf16" else 6) * (self.m / 32 + 1 + self.max_rank / 32 + 1) + 16 + 12 + 3
        return y[:self.T], (size * adds * 2.0 ** -24)[:self.T]

    def check(self, ctx, **kw):
        y = self.run(ctx, **kw)
        ref, bar = self.ref()
        assert (np.abs(y - ref) <= bar).all(), np.max(np.abs(y - ref) / bar)
        return y


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("widths", [[64], [1], [17], [130, 31, 31], [1000, 513], [4096, 1024, 1024]],
                         ids=lambda w: "-".join(map(str, w)))
def test_token_step(ctx, widths, dtype):
    """A row each, adapters of several ranks, requests that share one, requests without."""
    say("lora step", widths, dtype)
    rng = np.random.default_rng(sum(widths))
    ids = [0, 3, 3, -1, 2, 4, 1, 0, 3, 99, 5, -7]
    s = Setup(rng, [1] * 12, ids, [8, 5, 16, 33, 0, 64], 320, widths, dtype)
    y = s.check(ctx)
    assert np.array_equal(y[[3, 9, 5, 11]], s.base[[3, 9, 5, 11]])
    assert np.array_equal(s.run(ctx, in_place=True), y)
    assert np.array_equal(s.run(ctx, pad=3, ex=5, ey=7), y)


@pytest.mark.parametrize("m", [8, 16, 24, 32, 40, 512, 1600, 4104, 14336])
def test_input_sizes(ctx, m):
    say("lora m", m)
    rng = np.random.default_rng(m)
    for dtype in ("bf16", "f32"):
        Setup(rng, [1, 3, 2], [1, 0, 1], [8, 12], m, [70], dtype).check(ctx)


@pytest.mark.parametrize("rank", [1, 7, 8, 9, 24, 32, 40, 96, 128, 136, 256])
@pytest.mark.parametrize("rows", [2, 200])
def test_ranks(ctx, rank, rows):
    say("lora rank", rank, rows)
    rng = np.random.default_rng(rank)
    for dtype in ("bf16", "f32"):
        Setup(rng, [rows - 1, 1], [1, 0], [rank, max(1, rank // 2)], 160, [48, 20, 33], dtype).check(ctx)


@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [16], [17], [64], [65, 1], [300, 1, 2, 77], [1, 2, 3, 500, 0, 260],
                                  [33] * 20], ids=lambda v: "-".join(map(str, v[:6])))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompts(ctx, lens, dtype):
    """Rows of an adapter scattered over sequences, tiles that end inside one, in place."""
    say("lora prompts", lens, dtype)
    rng = np.random.default_rng(len(lens))
    ids = [(i * 2) % 3 if i % 5 != 4 else -1 for i in range(len(lens))]
    s = Setup(rng, lens, ids, [16, 40, 8], 192, [96, 45], dtype, dead=3, gap=1)
    y = s.check(ctx)
    assert np.array_equal(s.run(ctx, in_place=True), y)
    assert np.array_equal(s.run(ctx, pad=1, ex=9, ey=2), y)


def test_many(ctx):
    """4096 sequences, 4096 adapters, most of them not in use."""
    say("lora many")
    rng = np.random.default_rng(1)
    ids = rng.integers(-1, 40, 4096) * 100
    Setup(rng, [1] * 4096, ids.tolist(), [4] * 4096, 16, [8], "bf16").check(ctx)
    ids = np.where(rng.random(4096) < 0.5, 4095, 7)
    Setup(rng, (rng.random(4096) < 0.7).astype(int).tolist(), ids.tolist(), [4] * 4096, 16, [8], "bf16").check(ctx)


@pytest.mark.parametrize("rank", [1, 8, 9, 24, 40, 128])
@pytest.mark.parametrize("lens", [[257], [500, 270, 0, 1, 63], [1024]])
def test_tiles_of_64_rows(ctx, rank, lens):
    say("lora tiles", rank, lens)
    rng = np.random.default_rng(rank + lens[0])
    s = Setup(rng, lens, [0, 1, 0, -1, 1][:len(lens)], [rank, 8][:len(lens)], 264, [300, 17], gap=1, dead=3)
    y = s.check(ctx, pad=1, ex=5, ey=3)
    assert np.array_equal(s.run(ctx, in_place=True), y)


def test_more_columns_than_blocks(ctx):
    """More blocks of 128 columns than a grid has places in y."""
    say("lora wide")
    rng = np.random.default_rng(11)
    Setup(rng, [1], [0], [1], 8, [65535 * 128 + 130]).check(ctx)


@pytest.mark.parametrize("rows", [1, 70])
def test_far_adapters(ctx, rows):
    """The second adapter's A and B begin more than 2^31 elements behind the first's."""
    say("lora far", rows)
    rng = np.random.default_rng(13)
    s = Setup(rng, [rows], [0], [9], 64, [40])
    y = s.check(ctx)
    n, m, stride, ns = 40, 64, (1 << 31) + 64, 1
    w, a, ix = ctx.alloc(2 * (4 * stride)), ctx.alloc(4 * (rows * (m + 2 * n) + 2)), ctx.alloc(4 * 5)
    w.upload(s.w[:s.sa], 2 * stride)
    w.upload(s.w[s.sa:], 2 * 3 * stride)
    a.upload(np.concatenate([s.x.reshape(-1), s.base.reshape(-1), np.zeros(rows * n + 1, np.float32), s.scale]))
    ix.upload(np.array([0, rows, 1, 0, 9], np.int32))
    q8hip.lora(ctx, w, 0, stride, 2 * stride, stride, 2, 9, a, 0, rows * m, rows * (m + n), rows * (m + 2 * n), ix, 0, 2,
               3, ns, rows, m, [n])
    assert np.array_equal(a.download((rows, n), np.float32, 4 * rows * (m + n)), y)
    for b in (w, a, ix):
        b.free()


def test_scratch_in_parts(ctx):
    """More rows than the scratch holds parts of A x for: the tiles go in several runs."""
    say("lora scratch")
    rng = np.random.default_rng(2)
    s = Setup(rng, [9000, 60000, 1], [0, 1, 0], [128, 100], 16, [8, 8, 8])
    s.check(ctx)


def test_hidden_values(ctx):
    """Infinities and NaN in x stay in their rows."""
    say("lora hidden")
    rng = np.random.default_rng(3)
    for lens in ([1] * 9, [5, 70, 2]):
        s = Setup(rng, lens, [0, 1, 0] * (len(lens) // 3), [8, 24], 96, [50, 20])
        clean = s.run(ctx)
        bad = [2, s.T - 2]
        s.x[bad[0], 5] = np.nan
        s.x[bad[1], 40] = np.inf
        y = s.run(ctx)
        keep = np.ones(s.T, bool)
        keep[bad] = False
        assert np.array_equal(y[keep], clean[keep]) and np.isnan(y[bad]).all()
    s.x[:] = 0
    assert np.array_equal(s.run(ctx), s.base[:s.T])


def test_large_and_small(ctx):
    """x beside values many times larger keeps its bits (every term is carried)."""
    say("lora spans")
    rng = np.random.default_rng(4)
    s = Setup(rng, [3, 80], [0, 0], [8], 64, [33], "f32")
    s.x[:, 0] *= 2.0 ** 60
    A = s.A[0]
    A[:, 0] = 0                                        # the large one meets zeros
    s.w[:s.sa].reshape(-1)[:8 * 64].reshape(8, 64)[:, 0] = 0
    s.check(ctx)


def test_nonsense_arrays(ctx):
    """Whatever cu, ids and ranks hold, only y is written."""
    say("lora nonsense")
    rng = np.random.default_rng(5)
    s = Setup(rng, [3] * 12, [0, 1] * 6, [8, 24], 96, [50, 20])
    s.cu = rng.integers(-2 ** 31, 2 ** 31 - 1, 13).astype(np.int32)
    s.ids = rng.integers(-5, 5, 12).tolist()
    s.run(ctx)
    s.cu = np.array([0, 36] * 6 + [0], np.int32)
    s.run(ctx)
    s.ranks = [2 ** 31 - 1, -5]
    s.run(ctx)


def test_captured(ctx):
    """A captured call serves other rows, adapters and lengths; the scratch is used by
    other calls between the replays."""
    say("lora captured")
    rng = np.random.default_rng(6)
    m, widths, ranks, ns, T = 256, [90, 40], [8, 30, 64], 6, 130
    n, R, na = sum(widths), 64, 3
    proto = Setup(rng, [T] + [0] * 5, [0] * 6, ranks, m, widths)
    a, w, ix = ctx.alloc(4 * (T * (m + 2 * n) + na)), ctx.alloc(proto.w.nbytes), ctx.alloc(4 * (2 * ns + 1 + na))
    w.upload(proto.w)
    ctx.graph_begin()
    q8hip.lora(ctx, w, 0, proto.sa, na * proto.sa, proto.sb, na, R, a, 0, T * m, T * (m + n), T * (m + 2 * n), ix, 0,
               ns + 1, 2 * ns + 1, ns, T, m, widths)
    g = ctx.graph_end()
    for lens, ids in (([1] * 6, [0, 1, 2, -1, 1, 0]), ([100, 0, 5, 25, 0, 0], [2, 0, 1, 2, 0, 0]), ([0] * 6, [0] * 6),
                      ([20, 20, 20, 20, 20, 30], [1, 1, 2, 2, -1, 0])):
        proto.lens, proto.ids, proto.T = lens, ids, sum(lens)
        proto.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        proto.x = rng.standard_normal((T, m)).astype(np.float32)
        proto.base = rng.standard_normal((T, n)).astype(np.float32)
        mark = np.full((T, n), 9, np.float32)
        a.upload(np.concatenate([proto.x.reshape(-1), proto.base.reshape(-1), mark.reshape(-1), proto.scale]))
        ix.upload(np.concatenate([proto.cu, ids, ranks]).astype(np.int32))
        g.launch()
        y = a.download((T, n), np.float32, 4 * T * (m + n))
        ref, bar = proto.ref()
        assert (np.abs(y[:proto.T] - ref) <= bar).all() and (y[proto.T:] == 9).all()
        Setup(rng, [40, 40], [0, 0], [16], 64, [64]).check(ctx)
    g.destroy()
    for b in (a, w, ix):
        b.free()
