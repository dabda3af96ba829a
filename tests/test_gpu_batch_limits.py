"""GPU checks of the calls over several sequences at the edges of what they take
(the bars are those of test_gpu_batch.py)."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import batch_oracle as bo
from oracle.q8_oracle import max_rel_err
from test_gpu_batch import (Paged, bf16_bits, bf16_to_f32, offsets, packed_inputs, run_append,
                            run_cache, run_packed, say)

pytestmark = pytest.mark.gpu


def test_cache_nonsense_offsets(ctx):
    """Offsets out of order or out of range: append and cache attention stay inside
    their buffers (nothing beside the outputs is written), and a well-formed
    sequence whose rows no other names has its rows right."""
    say("cache nonsense")
    rng = np.random.default_rng(70)
    for cu in ([-5, 10, 10, 4, 1 << 30], [20, 0, 20, 0, 20], [7, 9, 1 << 30, -1 << 30, 3]):
        p = Paged(ctx, rng, [16] * 4, [0, 30, 0, 700], 16, 1, 64)
        p.cu = np.asarray(cu, np.int32)
        p.old = np.array([0, 30, -9, 1 << 30], np.int32)
        p.rows = 20
        p.upload()
        q, k, v = (rng.standard_normal((20, h, 64)).astype(np.float32) for h in (2, 1, 1))
        y = run_cache(p, q)
        if cu[0] == -5:                                # rows 0 .. 9, of which 4 .. are named again
            ref = p.c.attention(q, [0, 10], p.old[:1], p.table[:1])
            assert max_rel_err(y[:4], ref[:4]) <= 1e-5
        if cu[0] == 7:
            ref = p.c.attention(q, [7, 9], p.old[:1], p.table[:1])
            assert max_rel_err(y[7:9], ref[7:9]) <= 1e-5
        run_append(p, q, k, v)
        for b in (p.pool, p.ix):
            b.free()


@pytest.mark.parametrize("large", [2.0 ** 14, 2.0 ** 20, 2.0 ** 23, 2.0 ** 34, 2.0 ** 60, 2.0 ** 126])
@pytest.mark.parametrize("nh,nkv,hd,P,lens,old", [
    (8, 2, 128, 64, [1, 1], [500, 90]),                # whole row tiles
    (6, 2, 64, 16, [2, 1, 3], [40, 300, 0]),
    (8, 2, 128, 64, [1, 2, 1], [1500, 700, 64 * 20]),  # runs of split contexts
    (5, 1, 64, 128, [1, 1], [3000, 1000]),
    (20, 1, 128, 32, [1, 1], [1500, 900]),             # 32 columns
    (40, 1, 64, 128, [2, 2], [1100, 1500]),            # 64 columns
])
def test_cache_carries_q_beside_a_large_dim(ctx, nh, nkv, hd, P, lens, old, large):
    """q counts as f32: beside dims many times the others, whose K codes are 0, the
    scores of the others stay within 1e-5 (every second row; the others ordinary)."""
    say("cache large q", nh, hd, P, lens, large)
    rng = np.random.default_rng(nh + hd)
    p = Paged(ctx, rng, lens, old, P, nkv, hd)
    p.c.k[..., 5] = 0
    p.c.k[..., hd - 3] = 0
    p.pool.upload(p.c.to_bytes())
    q = rng.standard_normal((p.rows, nh, hd)).astype(np.float32)
    q[::2, :, 5] = large
    q[::2, 1::2, hd - 3] = -large / 3
    y, ref = run_cache(p, q), p.c.attention(q, p.cu, p.old, p.table)
    for r in range(p.rows):
        assert max_rel_err(y[r], ref[r]) <= 1e-5, r
    # K that sees them: the scores' own size decides, here one key takes all
    p.c.k[..., 5] = rng.integers(-127, 128, p.c.k.shape[:-1])
    p.pool.upload(p.c.to_bytes())
    y = run_cache(p, q)
    assert np.isfinite(y).all()
    for b in (p.pool, p.ix):
        b.free()


def bf16_bar(ref, v):
    """Half a bf16 step of the output, half a binary16 step of the largest |v| for the
    probabilities, the f32 bar."""
    return 2.0 ** -8 * np.abs(ref) + 2.0 ** -11 * np.abs(v.astype(np.float64)).max() + 1e-5


@pytest.mark.parametrize("large", [2.0 ** 14, 2.0 ** 20, 2.0 ** 23, 2.0 ** 34, 2.0 ** 43, 2.0 ** 60, 2.0 ** 126])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,lens", [(8, 2, 64, [1, 130, 7]), (8, 2, 128, [1, 130, 7]), (2, 1, 128, [4200])])
def test_packed_carries_q_beside_a_large_dim(ctx, nh, nkv, hd, lens, act, large):
    """q counts as it stands: beside dims many times the others, which K does not
    have, the scores of the others stay as exact (every second row; the others
    ordinary)."""
    say("packed large q", nh, hd, lens, act, large)
    rng = np.random.default_rng(nh + hd)
    q, k, v = packed_inputs(rng, lens, nh, nkv, hd)
    k[..., 5] = 0
    k[..., hd - 3] = 0
    q[::2, :, 5] = large
    q[::2, 1::2, hd - 3] = -large / 3
    if act == "bf16":
        q = bf16_to_f32(bf16_bits(q))
    y = run_packed(ctx, q, k, v, offsets(lens), act)
    cu = offsets(lens)
    rows = range(len(q)) if len(q) < 500 else [0, 1, 2, 63, 64, 255, 256, 2047, 2048, 4198, 4199]
    for r in rows:
        a = cu[np.searchsorted(cu, r, "right") - 1]
        ref = bo.attend(q[r:r + 1].astype(np.float64), k[a:r + 1].astype(np.float64),
                        v[a:r + 1].astype(np.float64), r - a)[0]
        bar = 1e-5 * np.abs(ref).max() if act == "f32" else bf16_bar(ref, v)
        assert (np.abs(y[r] - ref) <= bar).all(), r


@pytest.mark.parametrize("nh,nkv,hd,nseq,most", [
    (8, 2, 64, 128, 1), (8, 2, 64, 129, 1),       # 256 and 258 row tiles over the KV heads
    (32, 2, 128, 65, 1), (40, 1, 64, 100, 3), (6, 2, 128, 40, 9), (20, 4, 64, 66, 2)])
def test_cache_tiles_of_many_sequences(ctx, nh, nkv, hd, nseq, most):
    """Every row tile has its block, whole or split, where tiles are about as many as
    the card has CUs: sequences of one row, of none, and of several that end inside
    a tile."""
    say("cache tiles", nh, nkv, hd, nseq, most)
    rng = np.random.default_rng(nseq)
    lens = [1] * nseq if most == 1 else rng.integers(0, most + 1, nseq).tolist()
    p = Paged(ctx, rng, lens, rng.integers(0, 120, nseq).tolist(), 32, nkv, hd)
    q = rng.standard_normal((p.rows, nh, hd)).astype(np.float32)
    assert max_rel_err(run_cache(p, q), p.c.attention(q, p.cu, p.old, p.table)) <= 1e-5
    for b in (p.pool, p.ix):
        b.free()
