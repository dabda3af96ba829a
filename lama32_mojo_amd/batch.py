"""Many sequences on one Q8 model: packed prompts and token steps over an 8-bit
paged KV cache.

  Pages    the page state (tables, lengths, reference counts) and the pool of
           pages of all layers, over the q8_pages_* calls
  Q8Batch  a Q8Llama's weights run over the slots of a Pages: prompts of several
           slots in one pass (q8_kv8_append, q8_attention_packed), token steps
           with one row a slot or several (q8_kv8_append, q8_kv8_attention),
           forks, rollback, release, compaction; an adapter a slot (q8_lora), drawn
           ids (q8_sample), prefixes that forks share read once (q8_kv8_share)
  Sampling how a slot's ids are drawn

The reference serves one sequence at a time (qwen3_mojo/src/qwen_q8.mojo:110-162);
the layers are the ones of Q8Llama.layer (run_layer_q8, src/llama_q8.mojo:144-230)
with every row at its own sequence's position.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping, Sequence

import numpy as np

from . import q8hip
from .adapters import CALLS, Adapters
from .model import Q8Llama, rope_inv_freq
from .q8 import PAD, Acts, q8_rowstride
from .q8hip import Buffer, Context


@dataclass(frozen=True)
class Sampling:
    """Settings of q8_sample: temperature 0 takes the most likely token; top_k 0, top_p 1
    and min_p 0 leave all."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


class Pages:
    """`slots` sequences over `npages` pages of `page` tokens, in `layers` layers.
    extra: more int32 arrays, by name, behind the state in `ix`."""

    def __init__(self, ctx: Context, slots: int, npages: int, maxpages: int, page: int, layers: int,
                 nkv: int, head_dim: int, extra: Mapping[str, int] | None = None):
        self.ctx, self.slots, self.npages, self.maxpages = ctx, slots, npages, maxpages
        self.page, self.layers, self.nkv, self.head_dim = page, layers, nkv, head_dim
        self.page_bytes = q8hip.kv8_page_bytes(page, nkv, head_dim)
        self.pool = Buffer.alloc(ctx, layers * npages * self.page_bytes)
        sizes = dict(cu=slots + 1, len=slots, held=slots, arg=slots, live=1, table=slots * maxpages,
                     ref=npages)
        self.at, top = {}, 0
        for name, n in sizes.items():
            self.at[name] = top
            top += n
        start = np.zeros(top, np.int32)
        start[self.at["table"]:self.at["table"] + slots * maxpages] = -1
        self.ints = top
        for name, n in (extra or {}).items():
            self.at[name] = top
            top += n
        self.ix = Buffer.alloc(ctx, 4 * top)
        self.ix.upload(start)
        self.length = [0] * slots              # the lengths, as the host knows them
        self.held = [0] * slots                # the pages held, likewise
        self.forked = set()                    # slots that may share pages

    def _state(self):
        return (self.ix, *(self.at[n] for n in ("table", "len", "held", "ref")))

    def _arg(self, values) -> int:
        if len(values) != self.slots:
            raise ValueError(f"{len(values)} values for {self.slots} slots")
        self.ix.upload(np.asarray(values, np.int32), 4 * self.at["arg"])
        return self.at["arg"]

    def _pool(self):
        return (self.pool, 0, self.page_bytes, self.layers, self.npages * self.page_bytes)

    def reserve(self, want: Sequence[int]) -> None:
        """Pages for want[s] tokens in every slot; raises (and gives back what it
        took) when the free pages do not reach."""
        shape = (self.slots, self.maxpages, self.npages)
        # a refused call's copies of shared pages cannot be told from the others, and
        # pages held ahead not from what it took: then the state as it was goes back
        keep = any(h > self._pages_of(n) for h, n in zip(self.held, self.length)) or \
            any(w > n for s, (w, n) in enumerate(zip(want, self.length)) if s in self.forked)
        before = self.ix.download((self.ints,), np.int32) if keep else None
        q8hip.pages_reserve(self.ctx, *self._state(), self._arg(want), *shape, self.page, *self._pool())
        if self._short(want):
            if keep:
                self.ix.upload(before)
            else:
                self.set_len(self.length)
            raise RuntimeError("KV pages full")
        self.held = [max(h, self._pages_of(w)) for h, w in zip(self.held, want)]

    def _pages_of(self, n: int) -> int:
        return -(-int(n) // self.page)

    def _short(self, want) -> bool:
        """Whether a slot lacks pages for want tokens, or is to write to a page that
        another slot names: one that found no free page for its copy keeps it, with
        its held pages as they were."""
        held = self.ix.download((self.slots,), np.int32, 4 * self.at["held"])
        if any(w > int(h) * self.page for w, h in zip(want, held)):
            return True
        grow = [s for s in self.forked if want[s] > self.length[s]]
        if not grow:
            return False
        table = self.ix.download((self.slots, self.maxpages), np.int32, 4 * self.at["table"])
        ref = self.ix.download((self.npages,), np.int32, 4 * self.at["ref"])
        return any((ref[table[s, self.length[s] // self.page:-(-want[s] // self.page)]] > 1).any()
                   for s in grow)

    def set_len(self, new: Sequence[int]) -> None:
        """The slots' lengths (-1: unchanged; at most what the slot's pages hold); pages
        behind them are released."""
        for s, (n, h) in enumerate(zip(new, self.held)):
            if n > h * self.page:
                raise ValueError(f"set_len: slot {s} holds pages for {h * self.page} tokens, not {n}")
        q8hip.pages_set_len(self.ctx, *self._state(), self._arg(new), self.slots, self.maxpages,
                            self.npages, self.page)
        self.length = [int(n) if n >= 0 else old for n, old in zip(new, self.length)]
        self.held = [self._pages_of(n) if n >= 0 else h for n, h in zip(new, self.held)]
        self.forked -= {s for s, n in enumerate(new) if n == 0}    # (these hold no pages now)

    def fork(self, source: Sequence[int]) -> None:
        """Slot s continues slot source[s] (-1: unchanged)."""
        q8hip.pages_fork(self.ctx, *self._state(), self._arg(source), self.slots, self.maxpages,
                         self.npages)
        pairs = [(s, f) for s, f in enumerate(source) if 0 <= f < self.slots and f != s]
        old = list(zip(self.length, self.held))
        for s, f in pairs:
            self.length[s], self.held[s] = old[f]
            self.forked |= {s, f}

    def compact(self) -> int:
        """The pages in use moved to the lowest ids; how many there are."""
        q8hip.pages_compact(self.ctx, self.ix, self.at["table"], self.at["held"], self.at["ref"],
                            self.at["live"], self.slots, self.maxpages, self.npages, *self._pool())
        return int(self.ix.download((1,), np.int32, 4 * self.at["live"])[0])

    def layer(self, L: int, rows: int):
        """The cache arguments of q8hip.kv8_append and kv8_attention for layer L."""
        return (self.pool, L * self.npages * self.page_bytes, self.npages, self.page, self.ix,
                self.at["cu"], self.at["len"], self.at["table"], self.slots, rows, self.maxpages)

    def close(self) -> None:
        self.pool.free()
        self.ix.free()


class Q8Batch:
    """`slots` sequences decoded together on the weights of `model` (its own cache
    and arena are not used): at most max_rows rows a call.  adapters: low-rank ones
    that slots may be given (use); share: attention reads the whole pages that forks
    share once for all of them."""

    def __init__(self, model: Q8Llama, slots: int, npages: int, maxlen: int, page: int = 64,
                 max_rows: int = 2048, adapters: Adapters | None = None, share: bool = False):
        cfg = model.cfg
        self.m, self.ctx, self.slots, self.max_rows = model, model.ctx, slots, int(max_rows)
        self.adapters, self.share = adapters, bool(share)
        if adapters is not None and (adapters.cfg is not cfg and adapters.cfg != cfg or adapters.ctx is not model.ctx):
            raise ValueError("Q8Batch: the adapters are of another model or context")
        most = max(slots, min(self.max_rows, 64))            # rows of logits
        extra = dict(k=most, drawn=most)
        if share:
            extra["share"] = q8hip.kv8_share_ints(slots, self.max_rows)
        if adapters is not None:
            extra |= dict(adapter=slots, rank=len(CALLS) * adapters.count)
        self.pages = Pages(self.ctx, slots, npages, -(-maxlen // page), page, cfg.layers, cfg.n_kv,
                           cfg.head_dim, extra)
        H, QD, KVD, I = cfg.hidden, cfg.q_dim(), cfg.kv_dim(), cfg.inter
        rs = q8_rowstride(H, model.G, model.scale)
        if any(lo.k != lo.q + QD * rs or lo.v != lo.k + KVD * rs or lo.up != lo.gate + I * rs
               for lo in model.lo):
            raise ValueError("Q8Batch needs stacked q|k|v and gate|up rows")
        s = self.max_rows
        self.a = Acts(self.ctx, PAD + cfg.half() + s * (6 * H + 2 * QD + 2 * KVD + 2 * I)
                      + max(slots, min(s, 64)) * (H + cfg.vocab + 5) + 256
                      + (adapters.count if adapters is not None else 0))
        self.oinv = self.a.alloc(cfg.half())
        self.a.write(self.oinv, rope_inv_freq(cfg))
        self.adapter = [-1] * slots            # the slots' adapters
        self.loaded = None                     # what of them is on the device
        if adapters is not None:
            self.oscale = self.a.alloc(adapters.count)
        self.rows16 = Buffer.alloc(self.ctx, 2 * 2 * s * KVD)
        self.ids = Buffer.alloc(self.ctx, 4 * max(s, slots))

    # ---- one layer over the rows of several slots --------------------------------
    def _adapt(self, L: int, call: str, ox: int, oy: int, s: int, lora: frozenset) -> None:
        """Adds the slots' adapters to the s rows at oy, the linear's outputs for those
        at ox."""
        if call not in lora:
            return
        ad, p = self.adapters, self.pages
        m, widths = ad.shape[call]
        oa, sa, ob, sb = ad.at[L, call]
        q8hip.lora(self.ctx, ad.w, oa, sa, ob, sb, ad.count, ad.max_rank, self.a.buf, ox, oy, oy, self.oscale,
                   p.ix, p.at["cu"], p.at["adapter"], p.at["rank"] + list(CALLS).index(call) * ad.count, self.slots, s,
                   m, widths, dtype=ad.dtype)

    def _layer(self, L: int, ox: int, s: int, packed: bool, lora: frozenset, shared: bool) -> None:
        """One block on the s rows at ox, in place.  (Adapters need the linears' inputs:
        no norm or swiglu in a GEMM's pre-pass.)"""
        m, ctx, a, w, cfg = self.m, self.ctx, self.a, self.m.w, self.m.cfg
        lo, G, sc = m.lo[L], m.G, m.scale
        H, QD, KVD, I = cfg.hidden, cfg.q_dim(), cfg.kv_dim(), cfg.inter
        ld = QD + 2 * KVD
        gemm = s >= 32 and H <= 16384 and not lora
        a.align(4)
        oq = a.alloc(s * ld)
        if gemm:
            q8hip.linear_rmsnorm(ctx, w.buf, lo.q, lo.in_norm, cfg.eps, a.buf, ox, oq, s, H, ld, G, sc)
        else:
            xn = a.alloc(s * H)
            q8hip.rmsnorm(ctx, w.buf, lo.in_norm, a.buf, ox, xn, s, H, cfg.eps)
            q8hip.linear(ctx, w.buf, lo.q, a.buf, xn, oq, s, H, ld, G, sc)
            self._adapt(L, "qkv", xn, oq, s, lora)
        if cfg.qk_norm:
            q8hip.head_rmsnorm(ctx, w.buf, lo.q_norm, a.buf, oq, oq, s, cfg.n_heads, cfg.head_dim, ld,
                               cfg.eps)
            q8hip.head_rmsnorm(ctx, w.buf, lo.k_norm, a.buf, oq + QD, oq + QD, s, cfg.n_kv,
                               cfg.head_dim, ld, cfg.eps)
        heads = (cfg.n_heads, cfg.n_kv, cfg.head_dim)
        p = self.pages
        q8hip.kv8_append(ctx, a.buf, oq, oq + QD, oq + QD + KVD, self.oinv, oq, *p.layer(L, s), *heads,
                         ld=ld, kv=self.rows16 if packed else None, okc_f16=0,
                         ovc_f16=self.max_rows * KVD)
        a.align(4)
        oao = a.alloc(s * QD)
        if packed:
            q8hip.attention_packed(ctx, a.buf, oq, self.rows16, 0, self.max_rows * KVD, a.buf, oao, p.ix,
                                   p.at["cu"], self.slots, s, *heads, ldq=ld)
        elif shared:
            q8hip.kv8_attention_shared(ctx, a.buf, oq, oao, *p.layer(L, s), *heads, p.at["share"], ldq=ld)
        else:
            q8hip.kv8_attention(ctx, a.buf, oq, oao, *p.layer(L, s), *heads, ldq=ld)
        a.align(4)
        oo = a.alloc(s * H)
        q8hip.linear(ctx, w.buf, lo.o, a.buf, oao, oo, s, QD, H, G, sc)
        self._adapt(L, "o", oao, oo, s, lora)
        og = a.alloc(s * 2 * I)
        if gemm:
            q8hip.linear_rmsnorm(ctx, w.buf, lo.gate, lo.post_norm, cfg.eps, a.buf, ox, og, s, H, 2 * I,
                                 G, sc, ores_f32=oo, oh_f32=ox)
            q8hip.linear_swiglu(ctx, w.buf, lo.down, a.buf, og, og + I, oo, s, I, H, G, sc, ld=2 * I)
        else:
            oz = a.alloc(s * H)
            q8hip.add_rmsnorm(ctx, w.buf, lo.post_norm, a.buf, ox, oo, ox, oz, s, H, cfg.eps)
            q8hip.linear(ctx, w.buf, lo.gate, a.buf, oz, og, s, H, I, G, sc)
            q8hip.linear(ctx, w.buf, lo.up, a.buf, oz, og + s * I, s, H, I, G, sc)
            self._adapt(L, "gate", oz, og, s, lora)
            self._adapt(L, "up", oz, og + s * I, s, lora)
            q8hip.swiglu(ctx, a.buf, og, og + s * I, s * I)
            q8hip.linear(ctx, w.buf, lo.down, a.buf, og, oo, s, I, H, G, sc)
            self._adapt(L, "down", og, oo, s, lora)
        q8hip.add(ctx, a.buf, oo, ox, s * H)

    def _head(self, ox: int, rows: Sequence[int]) -> int:
        """Logits [len(rows), vocab] of the given rows of ox."""
        m, cfg = self.m, self.m.cfg
        w, n, H = m.w, len(rows), cfg.hidden
        self.a.align(4)
        oz = self.a.alloc(n * H)
        norm = w.o("model.norm.weight")
        if list(rows) == list(range(rows[0], rows[0] + n)):
            q8hip.rmsnorm(self.ctx, w.buf, norm, self.a.buf, ox + rows[0] * H, oz, n, H, cfg.eps)
        else:
            for i, r in enumerate(rows):
                q8hip.rmsnorm(self.ctx, w.buf, norm, self.a.buf, ox + r * H, oz + i * H, 1, H, cfg.eps)
        self.a.align(4)
        olg = self.a.alloc(n * cfg.vocab)
        q8hip.linear(self.ctx, w.buf, w.o(m._head_name()), self.a.buf, oz, olg, n, H, cfg.vocab, m.G, m.scale)
        return olg

    # ---- calls -----------------------------------------------------------------------
    def forward(self, tokens: Mapping[int, Sequence[int]], every: bool = False,
                logits: bool = False, sample: Mapping[int, Sampling] | None = None,
                u: Sequence[float] | None = None):
        """Appends tokens[slot] to each slot named and returns, per slot, the
        greedy next id (every: after each of its tokens, a list), or with
        `logits` the f32 logits those come from.  Slots that are all empty run as
        packed prompts, others over the cache.

        With `sample` (settings by slot; slots that are not in it: greedy) ids are drawn
        with the random numbers u of [0, 1), one for each of them in the order of the
        slots, and come with their log-probabilities: (id, logp)."""
        slots = sorted(tokens)
        counts = [len(tokens[s]) if s in tokens else 0 for s in range(self.slots)]
        rows = sum(counts)
        if rows == 0 or any(not 0 <= s < self.slots or not len(tokens[s]) for s in slots):
            raise ValueError("forward: every slot named needs tokens")
        if rows > self.max_rows:
            raise ValueError(f"forward: {rows} rows, at most {self.max_rows}")
        p, H = self.pages, self.m.cfg.hidden
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        old = list(p.length)
        packed = all(old[s] == 0 for s in slots)
        out_rows = list(range(rows)) if every else [int(cu[s + 1]) - 1 for s in slots]
        if len(out_rows) > max(self.slots, min(self.max_rows, 64)):
            raise ValueError(f"forward: logits of {len(out_rows)} rows")
        if (sample is None) != (u is None) or (sample is not None and logits):
            raise ValueError("forward: sample needs u, and gives ids, not logits")
        if u is not None and (len(u) != len(out_rows) or not set(sample) <= set(slots)):
            raise ValueError(f"forward: {len(u)} random numbers for {len(out_rows)} ids, or settings of a slot "
                             "without tokens")
        if sample is not None:
            of = [s for s in slots for _ in (tokens[s] if every else (0,))]
            settings = self._settings([sample.get(s, Sampling(0.0)) for s in of], u)
        lora = self._adapters_of(slots)
        p.reserve([n + c for n, c in zip(old, counts)])
        p.ix.upload(cu, 4 * p.at["cu"])
        self.ids.upload(np.concatenate([np.asarray(tokens[s], np.int32) for s in slots]))
        shared = self.share and not packed and bool(p.forked)
        if shared:
            q8hip.kv8_share(self.ctx, p.ix, p.at["cu"], p.at["len"], p.at["table"], self.slots, rows, p.maxpages,
                            p.npages, p.page, p.at["share"])
        mark = self.a.mark()
        m, cfg, V = self.m, self.m.cfg, self.m.cfg.vocab
        try:
            self.a.align(4)
            ox = self.a.alloc(rows * H)
            q8hip.embed_gather(self.ctx, m.w.buf, m.w.o("model.embed_tokens.weight"), self.ids, 0,
                               self.a.buf, ox, rows, H, V, m.G, m.scale)
            for L in range(cfg.layers):
                at = self.a.mark()
                self._layer(L, ox, rows, packed, lora, shared)
                self.a.reset(at)
            p.set_len([n + c for n, c in zip(old, counts)])
            olg = self._head(ox, out_rows)
            if logits:
                flat = self.a.read(olg, len(out_rows) * V).reshape(-1, V)
            elif sample is not None:
                flat = self._draw(olg, *settings)
            else:
                for i in range(len(out_rows)):
                    q8hip.argmax(self.ctx, self.a.buf, olg + i * V, V, self.ids, i)
                flat = self.ids.download((len(out_rows),), np.int32).tolist()
        finally:
            self.a.reset(mark)
        if every:
            return {s: flat[cu[s]:cu[s + 1]] for s in slots}
        return dict(zip(slots, flat))

    def _adapters_of(self, slots: Sequence[int]) -> frozenset:
        """The calls of a layer that adapters of these slots change; their numbers, ranks
        and scales go to the device if they are not there."""
        ad = self.adapters
        used = [self.adapter[s] for s in slots if self.adapter[s] >= 0]
        if not used:
            return frozenset()
        now = (ad.version, tuple(self.adapter))
        if now != self.loaded:
            self.pages.ix.upload(np.array(self.adapter, np.int32), 4 * self.pages.at["adapter"])
            # (a call that an adapter does not change holds nothing of it: rank 0)
            rank = [[r if c in has else 0 for r, has in zip(ad.rank, ad.has)] for c in CALLS]
            self.pages.ix.upload(np.array(rank, np.int32).reshape(-1), 4 * self.pages.at["rank"])
            self.a.write(self.oscale, np.array(ad.scale, np.float32))
            self.loaded = now
        return frozenset().union(*(ad.has[i] for i in used))

    @staticmethod
    def _settings(how: Sequence[Sampling], u: Sequence[float]):
        """The arrays of q8_sample for rows of these settings: f32 [4 * rows], k."""
        return (np.array([[h.temperature for h in how], [h.top_p for h in how], [h.min_p for h in how], list(u)],
                         np.float32).reshape(-1), np.array([h.top_k for h in how], np.int32))

    def _draw(self, olg: int, par: np.ndarray, k: np.ndarray) -> list:
        """(id, log-probability) of each row of logits at olg."""
        n, V, p = len(k), self.m.cfg.vocab, self.pages
        opar = self.a.alloc(5 * n)
        self.a.write(opar, par)
        p.ix.upload(k, 4 * p.at["k"])
        q8hip.sample(self.ctx, self.a.buf, olg, n, V, opar, p.ix, p.at["k"], p.at["drawn"], self.a.buf, opar + 4 * n)
        ids = p.ix.download((n,), np.int32, 4 * p.at["drawn"])
        return list(zip(ids.tolist(), self.a.read(opar + 4 * n, n).tolist()))

    def use(self, adapters: Mapping[int, int]) -> None:
        """Slot s has the adapter adapters[s] from now on (-1: none).  What it has cached
        stays as it is."""
        n = self.adapters.count if self.adapters is not None else 0
        if any(not 0 <= s < self.slots or not -1 <= i < n for s, i in adapters.items()):
            raise ValueError("use: no such slot or adapter")
        for s, i in adapters.items():
            self.adapter[s] = i

    def truncate(self, lengths: Mapping[int, int]) -> None:
        """Shortens slots (rejected drafts); 0 ends a sequence.  The page that a slot's
        end falls into keeps the scale that the dropped tokens gave it: fork the slot
        before a draft, and back if it is rejected, to be without it."""
        if any(not 0 <= s < self.slots or not 0 <= n <= self.pages.length[s]
               for s, n in lengths.items()):
            raise ValueError("truncate: no such slot, or a length past its tokens")
        self.pages.set_len([lengths.get(s, -1) for s in range(self.slots)])

    def fork(self, source: Mapping[int, int]) -> None:
        """Slot s continues slot source[s], sharing its pages, with its adapter."""
        if any(not 0 <= x < self.slots for pair in source.items() for x in pair):
            raise ValueError("fork: no such slot")
        self.pages.fork([source.get(s, -1) for s in range(self.slots)])
        was = list(self.adapter)
        for s, f in source.items():
            self.adapter[s] = was[f]

    def compact(self) -> int:
        return self.pages.compact()

    def close(self) -> None:
        self.pages.close()
        for b in (self.a.buf, self.rows16, self.ids):
            b.free()
