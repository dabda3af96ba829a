"""GPU checks of the calls over several sequences at the edges of what they take
(the bars are those of test_gpu_batch.py)."""

import numpy as np
import pytest

from lama32_mojo_amd import q8hip
from oracle import batch_oracle as bo
from oracle.q8_oracle import max_rel_err
from test_gpu_batch import Paged, inv_freq, run_append, run_cache, say

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
