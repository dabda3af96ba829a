"""Adapters.load: what lies on the device for an adapter whose linears differ in rank, in
host memory."""

import numpy as np
import pytest

from lama32_mojo_amd import adapters, model
from lama32_mojo_amd.adapters import CALLS, Adapters
from test_batch_pages import Memory

CFG = model.Config(64, 2, 4, 2, 16, 96, 50, 1e-5, 10000.0, 32.0, 1.0, 4.0, 8192.0, tied=True, qk_norm=False, rope="plain")
RANKS = {"self_attn.q_proj": 16, "self_attn.k_proj": 5, "self_attn.v_proj": 8, "self_attn.o_proj": 12, "mlp.gate_proj": 4,
         "mlp.up_proj": 16, "mlp.down_proj": 1}


def up8(r):
    return (r + 7) // 8 * 8


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(adapters, "Buffer", Memory)


def tensors(rng, ad, rank_of):
    out = {}
    for L in range(CFG.layers):
        for call, linears in CALLS.items():
            m, widths = ad.shape[call]
            for linear, n in zip(linears, widths):
                r = rank_of(L, linear)
                if r:
                    for name, shape in (("lora_A", (r, m)), ("lora_B", (n, r))):
                        out[f"model.layers.{L}.{linear}.{name}.weight"] = rng.standard_normal(shape).astype(np.float32)
    return out


def held(ad, i, L, call):
    """(A [parts, p, m], B [n, p]) of adapter i, p its largest rank rounded up."""
    m, widths = ad.shape[call]
    p, dtype = up8(ad.rank[i]), np.uint16 if ad.dtype == "bf16" else np.float32
    oa, sa, ob, sb = ad.at[L, call]
    out = []
    for off, shape in ((oa + i * sa, (len(widths), p, m)), (ob + i * sb, (sum(widths), p))):
        x = ad.w.download(shape, dtype, off * ad.elem)
        out.append(x if dtype == np.float32 else (x.astype(np.uint32) << 16).view(np.float32))
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["linears", "layers", "one"])
def test_scale_of_each_linear(host, dtype, which):
    """scale B is alpha / r of the linear's own rank times its lora_B: within the rounding of
    the quotient, the product and the scale (2^-24 each) and to bf16 (2^-8); exact where the
    ranks are alike."""
    rng = np.random.default_rng(3)
    ad = Adapters(None, CFG, 2, 16, dtype)
    rank_of = {"linears": lambda L, x: RANKS[x], "layers": lambda L, x: (16, 6)[L],
               "one": lambda L, x: 12 if x != "mlp.up_proj" else 0}[which]
    t, alpha = tensors(rng, ad, rank_of), 24.0
    ad.load(1, t, alpha)
    half = 0.0 if dtype == "f32" else 2.0 ** -8
    for L in range(CFG.layers):
        for call, linears in CALLS.items():
            if call not in ad.has[1]:
                continue
            first, (A, B) = 0, held(ad, 1, L, call)
            for z, (linear, n) in enumerate(zip(linears, ad.shape[call][1])):
                a = t[f"model.layers.{L}.{linear}.lora_A.weight"]
                b = t[f"model.layers.{L}.{linear}.lora_B.weight"].astype(np.float64)
                r = len(a)
                assert np.all(np.abs(A[z, :r] - a) <= half * np.abs(a)) and not A[z, r:].any()
                got = np.float64(np.float32(ad.scale[1])) * B[first:first + n]
                want = alpha / r * b
                assert np.all(np.abs(got[:, :r] - want) <= (half + 3.1 * 2.0 ** -24) * np.abs(want)), (L, linear)
                assert not got[:, r:].any()
                if r == ad.rank[1] and dtype == "f32":
                    assert np.array_equal(B[first:first + n, :r], b.astype(np.float32))
                first += n
