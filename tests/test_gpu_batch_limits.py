"""GPU checks of the calls over several sequences at the edges of what they take
(the bars are those of test_gpu_batch.py)."""

import numpy as np
import pytest

from oracle import batch_oracle as bo
from oracle.q8_oracle import max_rel_err
from test_gpu_batch import (PageState, Paged, bf16_bits, bf16_to_f32, offsets, packed_inputs, run_append,
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


def packed_errors(ctx, lens, nh, nkv, hd, act, seed, rows=None):
    """Rows of a packed call against float64; the bars of test_gpu_batch.py."""
    rng = np.random.default_rng(seed)
    q, k, v = packed_inputs(rng, lens, nh, nkv, hd)
    if act == "bf16":
        q = bf16_to_f32(bf16_bits(q))
    cu = offsets(lens)
    y = run_packed(ctx, q, k, v, cu, act, dead=2)
    for r in range(len(q)) if rows is None else rows:
        a = cu[np.searchsorted(cu, r, "right") - 1]
        ref = bo.attend(q[r:r + 1].astype(np.float64), k[a:r + 1].astype(np.float64),
                        v[a:r + 1].astype(np.float64), r - a)[0]
        bar = 1e-5 * np.abs(ref).max() if act == "f32" else bf16_bar(ref, v)
        assert (np.abs(y[r] - ref) <= bar).all(), r


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd", [(33, 1, 64), (66, 2, 128), (100, 1, 128), (128, 1, 64), (128, 1, 128)])
def test_packed_wide_groups(ctx, nh, nkv, hd, act):
    """Groups whose heads take several waves, with columns left over in one."""
    say("packed groups", nh, nkv, hd, act)
    packed_errors(ctx, [1, 0, 5, 70], nh, nkv, hd, act, nh)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("grp", [3, 5, 7])
def test_packed_long_odd_groups(ctx, grp, act):
    """The 8-wave blocks of long prompts, at groups that leave columns over."""
    say("packed long groups", grp, act)
    n = 4097 + 4200
    rows = np.unique(np.r_[0:3, 36:38, 84:87, 4094:4099, 4180:4184, n - 90:n - 86, n - 3:n])
    packed_errors(ctx, [4097, 4200], grp, 1, 128, act, grp, rows)


@pytest.mark.parametrize("nseq", [15, 16, 17])
def test_packed_sequence_counts(ctx, nseq):
    """Either side of the count up to which tiles go longest first."""
    say("packed sequences", nseq)
    lens = [(37 * i * i + 11 * i) % 150 for i in range(nseq)]
    packed_errors(ctx, lens, 4, 2, 64, "f32", nseq)
    packed_errors(ctx, lens[::-1], 6, 2, 128, "bf16", nseq)


def test_reserve_over_many_pages(ctx):
    """Pools of more pages than one go of the search: free pages that begin behind the
    first go, runs that cross from one to the next, and too few of them."""
    say("pages 60000")
    s = PageState(ctx, 24, 3000, 60000, 16, layers=1, pb=16)
    s.reserve([16 * (1500 + 37 * i % 200) for i in range(22)] + [0, 0])    # past 32768
    s.set_len([16 * len(r) for r in s.o.rows])
    s.check()
    s.set_len([-1, 160, -1, 0] + [-1] * 20)                                 # holes in the first go
    s.fork([-1, -1, -1, 4] + [-1] * 20)
    s.reserve([n + (16 * 2900 - n if 12 < i < 24 else i % 3) for i, n in enumerate(s.o.len)])
    s.check()
    s.set_len([16 * len(r) if i % 2 else -1 for i, r in enumerate(s.o.rows)])
    s.reserve([16 * 3000] * 24)                                             # 72000: the pool ends
    s.check()
    s.reserve([16 * 3000 if i % 5 == 0 else n for i, n in enumerate(s.o.len)])
    s.compact()
    s.check()


@pytest.mark.parametrize("kind", ["llama", "qwen"])
def test_greedy_ids_are_the_largest_logits(ctx, kind):
    """forward's ids, one a slot and one a row, are the argmax of the logits that the
    same calls return."""
    from lama32_mojo_amd import batch, model as gm
    from test_model_oracle import qwen_tiny, tiny_model
    say("greedy ids", kind)
    spec, t, inv = tiny_model() if kind == "llama" else qwen_tiny()
    cfg = gm.Config(spec.hidden, spec.layers, spec.n_heads, spec.n_kv, spec.head_dim, spec.inter,
                    spec.vocab, spec.eps, 500000.0 if kind == "llama" else 1000000.0, 32.0, 1.0, 4.0,
                    8192.0, tied=spec.tied, qk_norm=spec.qk_norm,
                    rope="llama3" if kind == "llama" else "plain")
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    two = [batch.Q8Batch(m, slots=4, npages=24, maxlen=160, page=16, max_rows=128) for _ in range(2)]
    rng = np.random.default_rng(2)
    draw = lambda n: rng.integers(0, spec.vocab, n).tolist()
    for tokens, every in (({0: draw(37), 1: draw(5), 3: draw(20)}, False), ({0: draw(1), 1: draw(1), 3: draw(1)}, False),
                          ({0: draw(4), 3: draw(3)}, True), ({2: draw(7)}, True), ({1: draw(33), 2: draw(1)}, False),
                          ({2: draw(1)}, False)):
        lg, ids = two[0].forward(tokens, every=every, logits=True), two[1].forward(tokens, every=every)
        assert set(ids) == set(lg) == set(tokens)
        for s in tokens:
            want = np.argmax(lg[s], -1)
            assert ids[s] == (want.tolist() if every else int(want)), (s, tokens)
            assert not every or len(ids[s]) == len(tokens[s])
    for b in two:
        b.close()
    m.close()
