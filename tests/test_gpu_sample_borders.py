"""q8_sample where running sums meet their borders, at logits and temperatures that no
binary fraction of a bin describes, against oracle/serving_oracle.py.

Equal logits weigh 1 each in float64, so their sums are whole numbers, and borders at
1/4, 1/2 and 3/4 of them are met exactly: the ids are those of the definition whatever
the logits' value.  Log-probabilities: half a step of f32, 2^-24 of the value, and 1e-11
for sums that are held to 2^-39."""

import numpy as np
import pytest

from test_gpu_sample import check, say

pytestmark = pytest.mark.gpu

VALUES = [0.3, 3.14, -4.3, 0.765625, 5.5, 1e-3, 77.7]


@pytest.mark.parametrize("temp", [1.0, 0.7, 1.25])
@pytest.mark.parametrize("n", [2, 4, 64, 960, 5000])
def test_equal_logits(ctx, n, temp):
    """n equal logits among tokens that are ruled out, far below, or not there."""
    say("sample borders", n, temp)
    N = 9001
    rows, top_p, u = [], [], []
    for v in VALUES:
        for p in (0.25, 0.5, 0.75):
            for z in (0.0, 0.25, 0.75, 0.999):
                rows.append(v)
                top_p.append(p)
                u.append(z)
    v = np.array(rows, np.float32)
    at = np.sort(np.random.default_rng(n).permutation(N)[:n])
    for fill in (-np.inf, -60.0, None):
        x = np.repeat(v[:, None], n, 1)
        if fill is not None:
            x = np.full((len(v), N), np.float32(fill)) + (v[:, None] if np.isfinite(fill) else 0)
            x[:, at] = v[:, None]
        x = x.astype(np.float32)
        check(ctx, x, temp=temp, top_p=top_p, u=u)
        check(ctx, x, temp=temp, k=n + 3, top_p=top_p, u=u)
        check(ctx, x, temp=temp, k=max(1, n // 2), top_p=top_p, u=u)


@pytest.mark.parametrize("temp", [1.0, 0.7])
def test_tokens_behind_the_border(ctx, temp):
    """Equal logits with a tail that counts: the border lies behind the half of them."""
    say("sample tails", temp)
    v = np.array(VALUES, np.float32)
    for n, gap in ((4, 8.0), (64, 12.0), (4, 20.0)):
        x = np.repeat((v - np.float32(gap))[:, None], 3000, 1)
        x[:, 100:100 + n] = v[:, None]
        for u in (0.0, 0.5, 0.999):
            check(ctx, x, temp=temp, top_p=0.5, u=u)
            check(ctx, x, temp=temp, top_p=0.5, min_p=0.5, u=u)


@pytest.mark.parametrize("temp", [0.75, 1.25, 1.5, 0.7, 3.0])
@pytest.mark.parametrize("n", [40, 5000, 20000])
def test_half_bins(ctx, n, temp):
    """Logits halfway between two bins' middles, the largest among them."""
    say("sample half bins", n, temp)
    rng = np.random.default_rng(n)
    j = rng.integers(-200, 100, (12, n))
    x = (np.float64(np.float32(temp)) * (2 * j + 1) / 32).astype(np.float32)
    for r in range(12):
        x[r, rng.integers(0, n)] = np.float32(np.float64(np.float32(temp)) * (2 * (100 + 7 * r) + 1) / 32)
    u = rng.random(12).astype(np.float32)
    for kw in (dict(), dict(top_p=0.9), dict(k=30, top_p=0.8), dict(min_p=0.03), dict(k=n // 2)):
        check(ctx, x, temp=temp, u=u, **kw)
