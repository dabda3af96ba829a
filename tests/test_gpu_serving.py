"""Requests that differ on one Q8Batch: adapters of each slot, drawn ids, prefixes that
forks share, against the float64 model of tests/test_gpu_batch.py."""

import os
import sys

import numpy as np
import pytest

from lama32_mojo_amd import batch, model as gm
from lama32_mojo_amd.adapters import CALLS, Adapters
from oracle.q8_oracle import max_rel_err
from oracle.serving_oracle import sample_row

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def tiny(kind):
    from test_model_oracle import qwen_tiny, tiny_model
    spec, t, inv = tiny_model() if kind == "llama" else qwen_tiny()
    cfg = gm.Config(spec.hidden, spec.layers, spec.n_heads, spec.n_kv, spec.head_dim, spec.inter, spec.vocab,
                    spec.eps, 500000.0 if kind == "llama" else 1000000.0, 32.0, 1.0, 4.0, 8192.0, tied=spec.tied,
                    qk_norm=spec.qk_norm, rope="llama3" if kind == "llama" else "plain")
    return spec, t, inv, cfg


def matrices(rng, cfg, ad, rank, linears, bits):
    """lora_A, lora_B of the given linears in every layer, values as the device holds them."""
    out = {}
    for L in range(cfg.layers):
        for call, ls in CALLS.items():
            m, widths = ad.shape[call]
            for linear, n in zip(ls, widths):
                if linear not in linears:
                    continue
                for name, shape in (("lora_A", (rank, m)), ("lora_B", (n, rank))):
                    x = (rng.standard_normal(shape) / np.sqrt(shape[1])).astype(np.float32)
                    x = (x.view(np.uint32) & 0xffff0000).view(np.float32) if bits else x
                    out[f"base_model.model.model.layers.{L}.{linear}.{name}.weight"] = x
    return out


@pytest.mark.parametrize("kind,dtype", [("llama", "bf16"), ("qwen", "f32")])
def test_adapters(ctx, kind, dtype):
    """Slots with different adapters, one with none, prompts, token steps, a fork that keeps
    its adapter, a slot that gets another, an adapter loaded anew.

    The bar is that of the model without adapters (see test_model_batch), whose linears
    here have another term of their own size: twice it."""
    from test_gpu_batch import OracleBatch
    say("serving adapters", kind, dtype)
    spec, t, inv, cfg = tiny(kind)
    rng = np.random.default_rng(1)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    ad = Adapters(ctx, cfg, 3, 20, dtype)
    everything = [x for ls in CALLS.values() for x in ls]
    mats = [matrices(rng, cfg, ad, r, ls, dtype == "bf16")
            for r, ls in ((8, everything), (20, ["self_attn.q_proj", "self_attn.v_proj"]), (5, ["mlp.down_proj"]))]
    alpha = [8.0, 30.0, 5.0]
    for i in range(3):
        ad.load(i, mats[i], alpha[i])
    b = batch.Q8Batch(m, slots=4, npages=40, maxlen=160, page=16, max_rows=128, adapters=ad)
    o = OracleBatch(spec, t, inv, b)
    plain, now = o.m.lin, [-1]

    def lin(name, x):
        y, i = plain(name, x), now[0]
        A = mats[i].get("base_model.model." + name[:-6] + "lora_A.weight") if i >= 0 else None
        if A is None:
            return y
        B = mats[i]["base_model.model." + name[:-6] + "lora_B.weight"]
        return y + alpha[i] / max(x.shape[0] for k, x in mats[i].items() if "lora_A" in k) * \
            (np.asarray(x, np.float64) @ A.T.astype(np.float64)) @ B.T.astype(np.float64)
    o.m.lin = lin

    def run(tokens, every=False):
        packed = all(b.pages.length[s] == 0 for s in tokens)
        rows = sum(len(x) for x in tokens.values())
        got = b.forward(tokens, every=every, logits=True)
        for s, ids in tokens.items():
            now[0] = b.adapter[s]
            ref = o.forward(s, ids, packed)
            err = max_rel_err(got[s], ref if every else ref[-1])
            say("slot", s, "rows", len(ids), "of", rows, "err %.1e" % err)
            assert err <= 2 * (8.2e-3 if rows >= 32 else 4.1e-4), (s, len(ids))
    draw = lambda n: rng.integers(0, spec.vocab, n).tolist()                   # noqa: E731
    b.use({0: 0, 1: 1, 3: 2})
    run({0: draw(37), 1: draw(5), 2: draw(9), 3: draw(20)})
    for _ in range(2):
        run({s: draw(1) for s in range(4)})
    b.fork({2: 0})
    o.fork(2, 0)
    assert b.adapter == [0, 1, 0, 2]
    b.use({0: -1, 1: 0})
    run({s: draw(1 + s) for s in range(4)}, every=True)
    mats[2] = matrices(rng, cfg, ad, 16, ["mlp.up_proj", "self_attn.o_proj"], dtype == "bf16")
    ad.load(2, mats[2], alpha[2])
    run({3: draw(3), 0: draw(1)})
    with pytest.raises(ValueError):
        b.use({0: 3})
    with pytest.raises(ValueError):
        b.use({4: 0})
    with pytest.raises(KeyError):
        ad.load(0, {"model.layers.0.self_attn.x_proj.lora_A.weight": np.zeros((1, 1))}, 1.0)
    with pytest.raises(KeyError):
        ad.load(0, {"model.layers.0.self_attn.q_proj.lora_A.weight": np.zeros((1, cfg.hidden))}, 1.0)
    with pytest.raises(ValueError):
        ad.load(0, {"model.layers.0.self_attn.q_proj.lora_A.weight": np.zeros((25, cfg.hidden)),
                    "model.layers.0.self_attn.q_proj.lora_B.weight": np.zeros((cfg.q_dim(), 25))}, 1.0)
    b.close()
    ad.close()
    m.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_adapters_of_other_linears(ctx, dtype):
    """In one call with an adapter of all linears, one that changes few of them is the same
    as alone, whatever its place held before.

    The bits do not depend on the place.  Alone, the prompt takes calls of other row counts
    (9 and 18), each within the bar of test_adapters (2 * 4.1e-4) of one float64 model, so
    the two are within twice that; the token step reads 8-bit codes of which some may have
    been rounded the other way, and is compared by its bits only."""
    say("serving adapters of other linears", dtype)
    spec, t, inv, cfg = tiny("llama")
    rng = np.random.default_rng(9)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    ad = Adapters(ctx, cfg, 2, 16, dtype)
    everything = [x for ls in CALLS.values() for x in ls]
    few = matrices(rng, cfg, ad, 3, ["self_attn.o_proj"], dtype == "bf16")
    ad.load(0, matrices(rng, cfg, ad, 16, everything, dtype == "bf16"), 16.0)
    prompt = rng.integers(0, spec.vocab, 9).tolist()

    def logits(both):
        b = batch.Q8Batch(m, slots=2, npages=8, maxlen=64, page=16, max_rows=64, adapters=ad)
        b.use({0: 0, 1: 1})
        return [b.forward({s: prompt if len(x) else [7] for s in ((0, 1) if both else (1,))}, logits=True)[1]
                for x in (prompt, [])]
    ad.load(1, few, 3.0)
    alone, both = logits(False), logits(True)
    ad.load(1, {k: np.full_like(v, np.inf) for k, v in
                matrices(rng, cfg, ad, 16, everything, dtype == "bf16").items()}, 1.0)
    ad.load(1, few, 3.0)
    again = logits(True)
    assert np.array_equal(again[0], both[0]) and np.array_equal(again[1], both[1])
    assert max_rel_err(both[0], alone[0]) <= 2 * 2 * 4.1e-4


def test_without_adapters_in_use(ctx):
    """A batch that could have adapters, and one that draws, give the ids of one that
    cannot, bit for bit."""
    say("serving none in use")
    spec, t, inv, cfg = tiny("llama")
    rng = np.random.default_rng(2)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    ad = Adapters(ctx, cfg, 1, 8)
    one = batch.Q8Batch(m, slots=3, npages=40, maxlen=160, page=16, max_rows=128)
    two = batch.Q8Batch(m, slots=3, npages=40, maxlen=160, page=16, max_rows=128, adapters=ad, share=True)
    two.use({0: 0})                                     # (nothing loaded: no change)
    for n in (40, 1, 3):
        tokens = {s: rng.integers(0, spec.vocab, n + s).tolist() for s in range(3)}
        a, b = (x.forward(tokens, every=n < 40, logits=True) for x in (one, two))
        for s in range(3):
            assert np.array_equal(a[s], b[s])
    for x in (one, two, ad, m):
        x.close()


@pytest.mark.parametrize("page", [16, 64])
def test_shared_prefix(ctx, page):
    """Forks of a long prompt: token steps and drafts over the shared pages, growth into
    pages of their own, rollback into the shared part, a slot of another origin."""
    from test_gpu_batch import OracleBatch
    say("serving shared", page)
    spec, t, inv, cfg = tiny("llama")
    rng = np.random.default_rng(3)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    b = batch.Q8Batch(m, slots=6, npages=80, maxlen=320, page=page, max_rows=160, share=True)
    o = OracleBatch(spec, t, inv, b)
    draw = lambda n: rng.integers(0, spec.vocab, n).tolist()                   # noqa: E731

    def run(tokens, every=False):
        packed = all(b.pages.length[s] == 0 for s in tokens)
        rows = sum(len(x) for x in tokens.values())
        got = b.forward(tokens, every=every, logits=True)
        for s, ids in tokens.items():
            ref = o.forward(s, ids, packed)
            err = max_rel_err(got[s], ref if every else ref[-1])
            assert err <= (8.2e-3 if rows >= 32 else 4.1e-4), (s, len(ids), err)
        return b.pages.ix.download((13,), np.int32, 4 * b.pages.at["share"])
    run({0: draw(150)})
    b.fork({s: 0 for s in (1, 2, 3, 4)})
    for s in (1, 2, 3, 4):
        o.fork(s, 0)
    at = 150 // page * page
    found = run({s: draw(1) for s in range(5)})
    assert found[0] == 1 and found[1:7].tolist() == [0] * 5 + [-1] and found[7:12].tolist() == [at] * 5
    run({5: draw(20)})
    for n in (1, 4):
        found = run({s: draw(n) for s in range(6)}, every=True)
        assert found[1:7].tolist() == [0] * 5 + [-1]
    b.truncate({2: 50})                                 # back into the shared pages
    o.truncate(2, 50)
    found = run({s: draw(2) for s in (0, 1, 2, 3)})
    saves = {at // page: 2, 50 // page: 3}
    take = max(saves, key=lambda p: (saves[p] * p, p))
    assert found[1:7].tolist() == [0, 0, 0 if take == 50 // page else -1, 0, -1, -1]
    b.truncate({s: 0 for s in range(6)})
    for s in range(6):
        o.truncate(s, 0)
    run({1: draw(9), 2: draw(5)})
    b.close()
    m.close()


def test_drawn_ids(ctx):
    """Ids and log-probabilities are those of the logits, by each slot's settings."""
    say("serving draws")
    spec, t, inv, cfg = tiny("qwen")
    rng = np.random.default_rng(4)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    one, two = (batch.Q8Batch(m, slots=4, npages=40, maxlen=160, page=16, max_rows=128) for _ in range(2))
    how = {0: batch.Sampling(0.7, 20, 0.9), 1: batch.Sampling(1.5, min_p=0.1), 3: batch.Sampling()}
    for n, every in ((12, False), (1, False), (3, True), (1, False)):
        tokens = {s: rng.integers(0, spec.vocab, n).tolist() for s in range(4)}
        u = rng.random(4 * (n if every else 1)).astype(np.float32)
        logits = one.forward(tokens, every=every, logits=True)
        got = two.forward(tokens, every=every, sample=how, u=u)
        k = 0
        for s in range(4):
            h = how.get(s, batch.Sampling(0.0))
            for row, (i, lp) in zip(np.atleast_2d(logits[s]), got[s] if every else [got[s]]):
                want, wlp = sample_row(row, h.temperature, h.top_k, h.top_p, h.min_p, u[k])
                assert i == want and abs(lp - wlp) <= 2.0 ** -24 * abs(wlp) + 1e-11
                k += 1
    for bad in (dict(sample=how), dict(u=[0.5]), dict(sample=how, u=[0.5] * 3), dict(sample=how, u=[0.5] * 4, logits=True),
                dict(sample={9: how[0]}, u=[0.5] * 4)):
        before = list(two.pages.length)
        with pytest.raises(ValueError):
            two.forward({s: [1] for s in range(4)}, **bad)
        assert two.pages.length == before
    for x in (one, two, m):
        x.close()


def test_all_together(ctx):
    """A shared prompt, an adapter and settings for each request, several steps: what a
    step draws follows from its own logits, and a captured run's settings stay apart."""
    say("serving together")
    spec, t, inv, cfg = tiny("llama")
    rng = np.random.default_rng(5)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    ad = Adapters(ctx, cfg, 2, 8)
    everything = [x for ls in CALLS.values() for x in ls]
    for i in range(2):
        ad.load(i, matrices(rng, cfg, ad, 8, everything, True), 8.0)
    pair = [batch.Q8Batch(m, slots=4, npages=60, maxlen=160, page=16, max_rows=128, adapters=ad, share=True)
            for _ in range(2)]
    how = {s: batch.Sampling(0.9, 40, 0.95) for s in range(4)}
    prompt = rng.integers(0, spec.vocab, 70).tolist()
    for b in pair:
        b.forward({0: prompt})
        b.fork({1: 0, 2: 0, 3: 0})
        b.use({1: 0, 2: 1, 3: 0})
    ids = {s: 7 for s in range(4)}
    for _ in range(5):
        u = rng.random(4).astype(np.float32)
        logits = pair[0].forward({s: [i] for s, i in ids.items()}, logits=True)
        got = pair[1].forward({s: [i] for s, i in ids.items()}, sample=how, u=u)
        for s in range(4):
            assert got[s][0] == sample_row(logits[s], 0.9, 40, 0.95, 0.0, u[s])[0]
        ids = {s: got[s][0] for s in range(4)}
    assert pair[0].pages.ix.download((1,), np.int32, 4 * pair[0].pages.at["share"])[0] == 1
    assert not np.array_equal(logits[0], logits[1])
    for x in (*pair, ad, m):
        x.close()


def test_graphs_share_scratch(ctx):
    """Captured draws, adapters and shared attention of one context, replayed in turn on three
    streams beside eager calls: every replay as the eager result."""
    torch = pytest.importorskip("torch")
    from lama32_mojo_amd import q8hip
    from test_gpu_lora import Setup
    from test_gpu_share import Step, queries
    say("serving graphs share scratch")
    rng = np.random.default_rng(21)
    # (arrays, the call on them, where the result lies): buffers stay as long as the graphs
    R, n = 5, 20001
    logits = (rng.standard_normal((R, n)) * 2).astype(np.float32)
    par = np.array([[1.0] * R, [0.9, 1, 1, 0.99, 1], [0, 0.1, 0, 0, 0], rng.random(R)], np.float32)
    sa, sids = ctx.alloc(4 * (R * n + 4 * R)), ctx.alloc(8 * R)
    sa.upload(np.concatenate([logits.reshape(-1), par.reshape(-1)]))
    sids.upload(np.array([0, 0, 50, 0, 0], np.int32))

    su = Setup(rng, [300, 1, 40], [0, 1, 0], [40, 8], 512, [600], dtype="bf16")
    m, w = 512, 600
    la, lw, lx = ctx.alloc(4 * (su.rows * (m + 2 * w) + 2)), ctx.alloc(su.w.nbytes), ctx.alloc(4 * 9)
    la.upload(np.concatenate([su.x.reshape(-1), su.base.reshape(-1), np.zeros(su.rows * w, np.float32), su.scale]))
    lw.upload(su.w)
    lx.upload(np.concatenate([su.cu, su.ids, su.ranks]).astype(np.int32))

    st = Step(rng, [1] * 9, [0] * 7 + [-1, -1], [30], rng.integers(0, 200, 9), 16, 2, 64)
    q = queries(rng, 9, 8, 64)
    at = 2 * 9 + 1 + 9 * st.maxpages
    aa, ap, ax = ctx.alloc(2 * q.nbytes), ctx.alloc(st.c.to_bytes().nbytes), ctx.alloc(4 * (at + q8hip.kv8_share_ints(9, 9)))
    aa.upload(q)
    ap.upload(st.c.to_bytes())
    ax.upload(np.concatenate([st.cu, st.old, st.table.reshape(-1)]).astype(np.int32))
    where = (ax, 0, 10, 19, 9, 9, st.maxpages)

    def share():
        q8hip.kv8_share(ctx, *where, st.c.npages, 16, at)
        q8hip.kv8_attention_shared(ctx, aa, 0, q.size, ap, 0, st.c.npages, 16, *where, 8, 2, 64, at)
    calls = [
        (lambda: q8hip.sample(ctx, sa, 0, R, n, R * n, sids, 0, R), sids, (R,), np.int32, 4 * R),
        (lambda: q8hip.lora(ctx, lw, 0, su.sa, 2 * su.sa, su.sb, 2, 40, la, 0, su.rows * m, su.rows * (m + w),
                            su.rows * (m + 2 * w), lx, 0, 4, 7, 3, su.rows, m, [w]), la, (su.rows, w), np.float32,
         4 * su.rows * (m + w)),
        (share, aa, q.shape, np.float32, q.nbytes)]
    eager, graphs = [], []
    for call, buf, shape, dtype, off in calls:
        call()
        eager.append(buf.download(shape, dtype, off))
        ctx.graph_begin()
        call()
        graphs.append(ctx.graph_end())
    streams = [torch.cuda.Stream() for _ in calls]
    for i in range(9):
        for _, buf, shape, dtype, off in calls:
            buf.upload(np.full(shape, -3, dtype), off)
        for k in range(3):
            ctx.set_stream(streams[(i + k) % 3].cuda_stream)
            graphs[(k + i // 3) % 3].launch()
        torch.cuda.synchronize()
        ctx.set_stream(None)
        for (call, buf, shape, dtype, off), y in zip(calls, eager):
            assert np.array_equal(buf.download(shape, dtype, off), y), i
        calls[i % 3][0]()
    for g in graphs:
        g.destroy()
    for b in (sa, sids, la, lw, lx, aa, ap, ax):
        b.free()
