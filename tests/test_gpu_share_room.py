"""q8_kv8_attention_shared where the groups' records are large beside the scratch: many KV
heads, many groups, many sequences.

The bar is that of tests/test_gpu_share.py, 1e-5."""

import numpy as np
import pytest

from oracle.q8_oracle import max_rel_err
from test_gpu_share import Step, queries, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nkv", [253, 500, 512])
def test_most_kv_heads(ctx, nkv):
    """As many KV heads as a call may have, in two and three sequences."""
    say("shared most KV heads", nkv)
    rng = np.random.default_rng(nkv)
    for ns in (2, 3):
        s = Step(rng, [1] * ns, [0] * ns, [2], [3, 20, 0][:ns], 16, nkv, 128)
        q = queries(rng, s.T, nkv, 128)
        y = s.run(ctx, q)
        assert max_rel_err(y, s.ref(q)) <= 1e-5
        assert max_rel_err(y, s.run(ctx, q, share=False)) <= 1e-5


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("ns", [700, 1024])
def test_many_sequences(ctx, ns, wide):
    """Heads of 128 with as many sequences as may share, both parts in one launch and (wide
    tables) in two."""
    say("shared many sequences", ns, wide)
    rng = np.random.default_rng(ns)
    s = Step(rng, [1] * ns, [i % 3 - 1 for i in range(ns)], [2, 5], rng.integers(0, 20, ns), 16, 1, 128)
    if wide:
        more = 64 * 400 // 16 - s.maxpages
        s.table = np.concatenate([s.table, np.full((ns, more), -1, np.int32)], axis=1)
        s.maxpages += more
    s.check(ctx, queries(rng, s.T, 2, 128))
