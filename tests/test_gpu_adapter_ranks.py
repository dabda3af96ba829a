"""An adapter whose linears differ in rank, on a Q8Batch, against the float64 model with
alpha over each linear's own rank.

The bar is that of test_gpu_serving.test_adapters below 32 rows, 2 * 4.1e-4: B is multiplied
by a quotient of ranks, which is a power of two in bf16 and off by 2^-23 in f32.  Calls have
fewer than 32 rows: scores reach 33 with these updates, and a linear of 32 rows or more, within
2e-4, moves a probability by 4e-4 of them, 1.3e-2, where the bars of such calls and of the
codes that they store count scores of 8."""

import numpy as np
import pytest

from lama32_mojo_amd import batch, model as gm
from lama32_mojo_amd.adapters import CALLS, Adapters
from oracle.q8_oracle import max_rel_err
from test_gpu_serving import matrices, say, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,ranks", [("f32", (16, 5, 12, 3, 7, 9, 1)), ("bf16", (8, 16, 4, 2, 16, 1, 8))])
def test_ranks(ctx, dtype, ranks):
    from test_gpu_batch import OracleBatch
    say("adapter ranks", dtype)
    spec, t, inv, cfg = tiny("llama")
    rng = np.random.default_rng(12)
    m = gm.Q8Llama(ctx, cfg, 16, weights=t)
    ad = Adapters(ctx, cfg, 2, 16, dtype)
    mats = {}
    for linear, r in zip([x for ls in CALLS.values() for x in ls], ranks):
        mats |= matrices(rng, cfg, ad, r, [linear], dtype == "bf16")
    alpha = 20.0
    ad.load(1, mats, alpha)
    b = batch.Q8Batch(m, slots=2, npages=20, maxlen=100, page=16, max_rows=31, adapters=ad)
    b.use({0: 1})
    o = OracleBatch(spec, t, inv, b)
    plain, now = o.m.lin, [-1]

    def lin(name, x):
        y = plain(name, x)
        A = mats.get("base_model.model." + name[:-6] + "lora_A.weight")
        if now[0] < 0 or A is None:
            return y
        B = mats["base_model.model." + name[:-6] + "lora_B.weight"].astype(np.float64)
        return y + alpha / len(A) * (np.asarray(x, np.float64) @ A.T.astype(np.float64)) @ B.T
    o.m.lin = lin
    for n in (9, 1, 13, 1):
        tokens = {s: rng.integers(0, spec.vocab, n).tolist() for s in range(2)}
        packed = all(x == 0 for x in b.pages.length)
        got = b.forward(tokens, logits=True)
        for s in range(2):
            now[0] = b.adapter[s]
            err = max_rel_err(got[s], o.forward(s, tokens[s], packed)[-1])
            say("slot", s, "rows", n, "err %.1e" % err)
            assert err <= 2 * 4.1e-4
    for x in (b, ad, m):
        x.close()
