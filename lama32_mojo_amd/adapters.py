"""Low-rank adapters of a model, many at once: y += scale B (A x) beside each Q8
linear, with the adapter of each request (q8_lora).

  Adapters   room for `count` adapters of ranks up to max_rank for a Config's linears;
             load() takes a dict of lora_A / lora_B matrices by name

The reference has one set of weights; the names are those of its linears
(qwen3_mojo/src/qwen_q8.mojo:35-52) with .lora_A.weight and .lora_B.weight.
"""

from __future__ import annotations

from typing import Mapping

import numpy as np

from . import q8hip
from .model import Config
from .q8hip import Buffer, Context

# calls of one layer: the stacked linears of each (q|k|v share x and lie in one row)
CALLS = {"qkv": ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), "o": ("self_attn.o_proj",),
         "gate": ("mlp.gate_proj",), "up": ("mlp.up_proj",), "down": ("mlp.down_proj",)}


def _bf16_bits(x: np.ndarray) -> np.ndarray:
    """f32 values rounded to bf16 (nearest, ties to even; NaN stays NaN)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


class Adapters:
    """`count` places for adapters of ranks up to max_rank, held as "bf16" or "f32"."""

    def __init__(self, ctx: Context, cfg: Config, count: int, max_rank: int, dtype: str = "bf16"):
        if not 1 <= count <= 4096 or not 1 <= max_rank <= 256 or dtype not in q8hip.ACT:
            raise ValueError(f"Adapters: count={count}, max_rank={max_rank}, dtype={dtype}")
        self.ctx, self.cfg, self.count, self.dtype = ctx, cfg, int(count), dtype
        self.max_rank = (int(max_rank) + 7) // 8 * 8
        H, QD, KVD, I = cfg.hidden, cfg.q_dim(), cfg.kv_dim(), cfg.inter
        self.shape = {"qkv": (H, (QD, KVD, KVD)), "o": (QD, (H,)), "gate": (H, (I,)), "up": (H, (I,)),
                      "down": (I, (H,))}
        self.at, top = {}, 0                   # (layer, call) -> (oa, a_stride, ob, b_stride)
        for L in range(cfg.layers):
            for call, (m, widths) in self.shape.items():
                sa, sb = len(widths) * self.max_rank * m, sum(widths) * self.max_rank
                self.at[L, call] = (top, sa, top + self.count * sa, sb)
                top += self.count * (sa + sb)
        self.elem = 2 if dtype == "bf16" else 4
        self.w = Buffer.alloc(ctx, top * self.elem)
        self.rank = [0] * self.count
        self.scale = [0.0] * self.count
        self.has = [frozenset()] * self.count  # the calls that each adapter changes
        self.version = 0

    def load(self, i: int, tensors: Mapping[str, np.ndarray], alpha: float) -> None:
        """Adapter i from its lora_A [rank, m] and lora_B [n, rank] matrices (floating
        values, or bf16 bits as uint16) by name; linears that are not named are left
        alone.  The scale of a linear is alpha / its own rank.  (The device has one scale an
        adapter, that of the largest rank; the B of others are multiplied by the quotient of
        the two ranks before they are rounded to `dtype`, so in bf16 an update of another rank
        is off by up to half a step of bf16, 2^-8, unless the quotient is a power of two.)"""
        if not 0 <= i < self.count:
            raise ValueError(f"load: adapter {i} of {self.count}")
        found: dict[tuple, dict] = {}
        for name, x in tensors.items():
            at = name.rfind("model.layers.")
            part = name[at:].split(".") if at >= 0 else []
            if len(part) != 7 or part[5] not in ("lora_A", "lora_B") or part[6] != "weight" \
                    or not part[2].isdigit() or int(part[2]) >= self.cfg.layers:
                raise KeyError(f"load: {name} is no adapter matrix of this model")
            x = np.asarray(x)
            if x.dtype == np.uint16:
                x = (x.astype(np.uint32) << 16).view(np.float32)
            found.setdefault((int(part[2]), ".".join(part[3:5])), {})[part[5]] = x.astype(np.float32)
        rank = 0
        for (L, linear), ab in found.items():
            call = next((c for c, ls in CALLS.items() if linear in ls), None)
            if call is None or set(ab) != {"lora_A", "lora_B"}:
                raise KeyError(f"load: layer {L} {linear} needs lora_A and lora_B of a linear of this model")
            m, widths = self.shape[call]
            n, r = widths[CALLS[call].index(linear)], ab["lora_A"].shape[0]
            if ab["lora_A"].shape != (r, m) or ab["lora_B"].shape != (n, r) or not 1 <= r <= self.max_rank:
                raise ValueError(f"load: layer {L} {linear}: lora_A {ab['lora_A'].shape}, lora_B "
                                 f"{ab['lora_B'].shape}, expected [r, {m}], [{n}, r], r at most {self.max_rank}")
            rank = max(rank, r)
        p = (rank + 7) // 8 * 8
        has = frozenset(c for c, ls in CALLS.items() if any(linear in ls for _, linear in found))
        for (L, call), (oa, sa, ob, sb) in self.at.items():
            if call not in has:
                continue
            m, widths = self.shape[call]
            A = np.zeros((len(widths), p, m), np.float32)
            B = np.zeros((sum(widths), p), np.float32)
            first = 0
            for z, (linear, n) in enumerate(zip(CALLS[call], widths)):
                ab = found.get((L, linear))
                if ab is not None:
                    r = ab["lora_A"].shape[0]
                    A[z, :r] = ab["lora_A"]
                    B[first:first + n, :r] = ab["lora_B"] * np.float32(rank / r)
                first += n
            for off, x in ((oa + i * sa, A), (ob + i * sb, B)):
                x = _bf16_bits(x) if self.dtype == "bf16" else x
                self.w.upload(x.reshape(-1), off * self.elem)
        self.rank[i], self.scale[i], self.has[i] = rank, (alpha / rank if rank else 0.0), has
        self.version += 1

    def close(self) -> None:
        self.w.free()
