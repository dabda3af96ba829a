"""The longest-first search for a block's row tile (up to 16 sequences of a packed
call), restated with its 64 lanes as arrays: every row tile belongs to one block,
tiles come in descending order of their place, and offsets that hold nonsense name
no row outside the call."""

import numpy as np

LANE = np.arange(64)


def packed_tile(cu, nseq, rows, PB, nb, b):
    """(first row, end, tile) of block b of nb; tile -1: none."""
    x = np.minimum(LANE, nseq - 1)
    c0, c1 = np.clip(cu[x], 0, rows), np.clip(cu[x + 1], 0, rows)
    tiles = np.where((LANE < nseq) & (c1 > c0), (c1 - c0 + PB - 1) // PB, 0)
    k0, step, first = 0, nb, 0
    while True:
        step = (step + 63) // 64
        k = k0 + LANE * step
        c = np.maximum(tiles[:nseq, None] - k, 0).sum(0)         # tiles with a place from k on
        z = np.nonzero(c > b)[0]
        if z.size == 0:
            return 0, 0, -1
        k0 += int(z[-1]) * step
        first = int(c[z[-1]])
        if step <= 1:
            break
    have = np.nonzero(tiles > k0)[0]                             # sequences that have a tile k0
    r = b - (first - have.size)
    if not 0 <= r < have.size:
        return 0, 0, -1
    i = have[r]
    return int(c0[i]), int(c1[i]), k0


def blocks(rows, nseq, PB):
    return rows // PB + nseq


def test_every_tile_once_and_longest_first():
    rng = np.random.default_rng(3)
    for step in range(150):
        nseq, PB = int(rng.integers(1, 17)), int(rng.choice([1, 3, 32, 42, 128]))
        lens = rng.integers(0, 3 + PB * rng.integers(0, 30), nseq) * (rng.random(nseq) < 0.8)
        cu = np.concatenate([[0], np.cumsum(lens)])
        rows = int(cu[-1]) + int(rng.integers(0, 20))
        seen, places = [], []
        nb = blocks(rows, nseq, PB)
        for b in range(nb):
            r0, r1, t = packed_tile(cu, nseq, rows, PB, nb, b)
            if t >= 0:
                seen.append((r0 + t * PB, min(r0 + (t + 1) * PB, r1)))
                places.append(t)
        want = [(a + t, min(a + t + PB, z)) for a, z in zip(cu[:-1], cu[1:]) for t in range(0, z - a, PB)]
        assert sorted(seen) == sorted(want)
        assert places == sorted(places, reverse=True)


def test_long_and_nonsense():
    # more tiles than 64 * 64, so the search takes three steps
    cu, PB = np.array([0, 9000, 9000, 9010, 14000]), 1
    nb = blocks(14000, 4, PB)
    got = [packed_tile(cu, 4, 14000, PB, nb, b) for b in range(nb)]
    rows = sorted(r0 + t for r0, r1, t in got if t >= 0)
    assert rows == list(range(14000))
    rng = np.random.default_rng(4)
    for _ in range(100):
        nseq, n = int(rng.integers(1, 17)), int(rng.integers(1, 400))
        cu = rng.integers(-2 ** 31, 2 ** 31, nseq + 1)
        mix = rng.random(nseq + 1) < 0.6
        cu[mix] = rng.integers(0, n + 1, int(mix.sum()))
        nb = blocks(n, nseq, 3)
        for b in range(nb):
            r0, r1, t = packed_tile(cu, nseq, n, 3, nb, b)
            assert t < 0 or 0 <= r0 <= r0 + 3 * t < r1 <= n
