"""Operators for several sequences at once, as timed cases: attention over packed
prompts, the 8-bit paged cache (append, attention) and the pages it is made of.

`own` false: the plain form of each operator in torch.  `own` true: the calls that
a program makes of this package's entry points.  `exact` restates the operators
in float64, sequence by sequence.

A page of the cache holds P tokens of one layer: K codes [nkv, P, hd] int8, V codes
[nkv, hd, P] int8, then a K scale and a V scale per KV head (f32), padded to 16
bytes.  Codes are whole numbers by definition (the quotient rounded once, half to
even), so they are returned as they are, beside their scales.
"""

import math

import torch

own = False

HEADS = [(32, 8, 64), (32, 8, 128), (16, 8, 128)]    # (query heads, KV heads, head_dim)


def listed():
    return [
        # four short prompts that arrive together, 64-dim heads: launch and latency count
        dict(name="packed short prompts", kind="packed", lens="1,37,200,90", nheads=32, nkv=8, head_dim=64,
             act="f32"),
        # a prompt batch of very different lengths, f32 activations as the Q8 linears give them
        dict(name="packed ragged prompts", kind="packed", lens="1,17,333,1024,2049,700,64,3900", nheads=32,
             nkv=8, head_dim=128, act="f32"),
        # a long document beside two questions, bf16 activations
        dict(name="packed long prompt bf16", kind="packed", lens="250,16001,31", nheads=32, nkv=8,
             head_dim=128, act="bf16"),
        # one decode step of 64 sequences: a row each, behind partly filled pages
        dict(name="append decode step", kind="append", nseq=64, most=1, old=4000, page=64, rows16=False,
             nheads=32, nkv=8, head_dim=128),
        # a prompt batch written to fresh pages, with the binary16 rows its attention reads
        dict(name="append prompts", kind="append", nseq=8, most=2047, old=0, page=64, rows16=True,
             nheads=32, nkv=8, head_dim=128),
        # one short conversation, one token: the smallest call
        dict(name="cache attention 1 sequence", kind="cache", nseq=1, most=1, ctx=500, page=64, nheads=32,
             nkv=8, head_dim=64),
        # a serving batch, one token each, contexts from a few tokens to 8000
        dict(name="cache attention 64 sequences", kind="cache", nseq=64, most=1, ctx=8000, page=64,
             nheads=32, nkv=8, head_dim=128),
        # drafted tokens checked in one pass: up to 5 rows a sequence, small pages
        dict(name="cache attention drafts", kind="cache", nseq=24, most=5, ctx=3000, page=16, nheads=16,
             nkv=8, head_dim=128),
        # four very long contexts
        dict(name="cache attention long", kind="cache", nseq=4, most=1, ctx=131000, page=128, nheads=32,
             nkv=8, head_dim=128),
        # the bookkeeping of a decode step of 256 slots: a page every P tokens, lengths advanced
        dict(name="pages decode step", kind="pages", nslots=256, ctx=4000, page=64, layers=2, nkv=8,
             head_dim=64, beams=1, grow=1),
        # beams of 4 forked for drafts of 5 tokens, their shared last pages copied in every layer
        dict(name="pages fork beams", kind="pages", nslots=64, ctx=2000, page=64, layers=16, nkv=8,
             head_dim=64, beams=4, grow=5),
        # a pool with holes after most sequences ended, moved together
        dict(name="pages compact", kind="compact", nslots=64, ctx=2000, page=64, layers=16, nkv=8,
             head_dim=64),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed kinds and ranges, at another size."""
    kind = rng.choice(["packed", "packed", "packed", "append", "append", "cache", "cache", "cache",
                       "pages", "compact"])
    nh, nkv, hd = rng.choice(HEADS)
    c = dict(kind=kind, nkv=nkv, head_dim=hd)
    if kind in ("packed", "append", "cache"):
        c["nheads"] = nh
    if kind == "packed":
        lens, left = [], log_int(rng, 8, 12000)
        for _ in range(rng.randint(1, 16)):
            lens.append(log_int(rng, 1, max(1, left)))
            left = max(1, left - lens[-1])
        rng.shuffle(lens)
        c.update(lens=",".join(map(str, lens)), act=rng.choice(["f32", "f32", "bf16"]))
    elif kind == "append":
        nseq = log_int(rng, 1, 128)
        c.update(nseq=nseq, most=log_int(rng, 1, max(1, 8000 // nseq)),
                 old=rng.choice([0, log_int(rng, 1, 5000)]), page=rng.choice([16, 32, 64, 128]),
                 rows16=rng.random() < 0.5)
    elif kind == "cache":
        nseq = log_int(rng, 1, 96)
        c.update(nseq=nseq, most=rng.choice([1, 1, log_int(rng, 2, 9)]),
                 ctx=log_int(rng, 1, max(2, min(60000, 400000 // nseq))),
                 page=rng.choice([16, 32, 64, 128]))
    else:
        c.update(nslots=log_int(rng, 4, 128), ctx=log_int(rng, 8, 2000), page=rng.choice([16, 32, 64]),
                 layers=rng.randint(1, 12), head_dim=64)
        if kind == "pages":
            c.update(beams=rng.choice([1, 2, 4]), grow=log_int(rng, 1, 300))
    return c


# ---- inputs -------------------------------------------------------------------

def host_ints(salt, n, lo, hi):
    """n whole numbers of [lo, hi], spread over their logarithm, hi among them, on the host: the
    lengths of a case, the same for every seed."""
    g = torch.Generator().manual_seed(1000 * n + salt)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    v = torch.exp(math.log(lo) + u * (math.log(hi + 1) - math.log(lo))).floor().long()
    v[n // 2] = hi
    return v.clamp(lo, hi).tolist()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def normal(shape, gen, std=1.0):
    return torch.randn(shape, device="cuda", generator=gen) * std


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def inv_freq(hd, theta=500000.0):
    return torch.tensor([theta ** (-2.0 * d / hd) for d in range(hd // 2)], dtype=torch.float32)


def page_bytes(c):
    return 2 * c["nkv"] * c["page"] * c["head_dim"] + (8 * c["nkv"] + 15) // 16 * 16


def parts(pool, c):
    """K codes [.., npages, nkv, P, hd], V codes [.., npages, nkv, hd, P] and scales
    [.., npages, 2, nkv] of a pool of pages (views of its bytes)."""
    nkv, P, hd = c["nkv"], c["page"], c["head_dim"]
    n, lead = nkv * P * hd, pool.shape[:-1]
    return (pool[..., :n].view(torch.int8).unflatten(-1, (nkv, P, hd)),
            pool[..., n:2 * n].view(torch.int8).unflatten(-1, (nkv, hd, P)),
            pool[..., 2 * n:2 * n + 8 * nkv].view(torch.float32).view(*lead, 2, nkv))


def random_pool(c, lead, gen):
    """Pages of random codes with scales of a few hundredths, as unit-size keys have."""
    pool = torch.randint(0, 255, (*lead, page_bytes(c)), device="cuda", generator=gen, dtype=torch.uint8)
    pool ^= 128                                             # codes -128 .. 126
    k, v, sc = parts(pool, c)
    k.clamp_(min=-127)
    v.clamp_(min=-127)
    sc.copy_(torch.exp(torch.randn(sc.shape, device="cuda", generator=gen) * 0.3) * 0.02)
    return pool


def page_table(pages, maxpages, npages, gen):
    """A table of distinct pages in random order, -1 behind each row's pages."""
    ids = torch.randperm(npages, generator=gen, device="cuda").tolist()
    tab, at = [], 0
    for n in pages:
        tab.append(ids[at:at + n] + [-1] * (maxpages - n))
        at += n
    return torch.tensor(tab, dtype=torch.int32, device="cuda")


class Ints:
    """The int32 arrays of a call in one arena, by name."""

    def __init__(self, **arrays):
        self.off, flat = {}, []
        for name, t in arrays.items():
            t = torch.as_tensor(t, dtype=torch.int32, device="cuda")
            self.off[name] = (sum(x.numel() for x in flat), t.shape)
            flat.append(t.reshape(-1))
        self.start = torch.cat(flat)
        self.now = self.start.clone()

    def __getitem__(self, name):
        at, shape = self.off[name]
        return self.now[at:at + math.prod(shape)].view(shape)

    def at(self, name):
        return self.off[name][0]


def prepare(case, seed):
    st = globals()["prepare_" + case["kind"]](case, generator(seed))
    st["case"] = case
    if own:
        for name in [n for n in ("arena", "q", "out", "kv", "pool", "kv_rows") if n in st]:
            st[name + "_buf"] = wrapped(st[name])
        st["ix_buf"] = wrapped(st["ix"].now)
    torch.cuda.synchronize()
    return st


def run(state):
    return globals()[("own_" if own else "plain_") + state["case"]["kind"]](state["case"], state)


_CTX = None


def context():
    """One library context for the process, as a program keeps it."""
    global _CTX
    if _CTX is None:
        from lama32_mojo_amd import q8hip
        _CTX = q8hip.Context(torch.cuda.current_device())
    return _CTX


def wrapped(t):
    return context().wrap(t.data_ptr(), t.numel() * t.element_size())


# ---- attention over packed prompts -----------------------------------------------

def packed_lens(c):
    return [int(x) for x in c["lens"].split(",")]


def prepare_packed(c, gen):
    nh, nkv, hd, lens = c["nheads"], c["nkv"], c["head_dim"], packed_lens(c)
    T = sum(lens)
    dt = torch.float32 if c["act"] == "f32" else torch.bfloat16
    ldq = (nh + 2 * nkv) * hd               # q inside stacked q|k|v rows, as the linears leave it
    q = normal((T, ldq), gen).to(dt)
    kv = normal((2, T, nkv * hd), gen).to(torch.float16)
    return dict(q=q, kv=kv, out=torch.empty((T, nh * hd), device="cuda", dtype=dt), ldq=ldq, lens=lens,
                ix=Ints(cu=offsets(lens)))


def own_packed(c, st):
    from lama32_mojo_amd import q8hip
    T, kvd = st["kv"].shape[1:]
    q8hip.attention_packed(context(), st["q_buf"], 0, st["kv_buf"], 0, T * kvd, st["out_buf"], 0, st["ix_buf"],
                           st["ix"].at("cu"), len(st["lens"]), T, c["nheads"], c["nkv"], c["head_dim"],
                           act=c["act"], ldq=st["ldq"])
    return st["out"]


def softmax_(s):
    """Softmax over the last axis, in place."""
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    return s


def plain_packed(c, st):
    nh, nkv, hd = c["nheads"], c["nkv"], c["head_dim"]
    T = st["q"].shape[0]
    q = st["q"][:, :nh * hd].float().view(T, nkv, nh // nkv, hd).permute(1, 2, 0, 3)
    k, v = st["kv"].float().view(2, T, nkv, hd).permute(0, 2, 1, 3)
    out = torch.empty((nkv, nh // nkv, T, hd), device="cuda")
    at = 0
    for n in st["lens"]:
        rows = slice(at, at + n)
        s = torch.matmul(q[:, :, rows].reshape(nkv, -1, hd), k[:, rows].transpose(1, 2)).view(nkv, -1, n, n)
        s *= 1.0 / math.sqrt(hd)
        s.masked_fill_(torch.ones((n, n), device="cuda", dtype=torch.bool).triu_(1), -math.inf)
        out[:, :, rows] = torch.matmul(softmax_(s).view(nkv, -1, n), v[:, rows]).view(nkv, -1, n, hd)
        at += n
    return out.permute(2, 0, 1, 3).reshape(T, nh * hd).to(st["q"].dtype)


# ---- the 8-bit cache: append --------------------------------------------------------

def prepare_append(c, gen):
    nh, nkv, hd, P, nseq = c["nheads"], c["nkv"], c["head_dim"], c["page"], c["nseq"]
    lens = host_ints(1, nseq, max(1, c["most"] // 8), c["most"])
    old = host_ints(2, nseq, max(1, c["old"] // 8), c["old"]) if c["old"] else [0] * nseq
    T = sum(lens)
    pages = [-(-(o + n) // P) for o, n in zip(old, lens)]
    npages, maxpages = sum(pages) + 7, max(pages) + 2
    ld = (nh + 2 * nkv) * hd
    x = normal((T, ld), gen) * torch.exp(normal((T, 1), gen, 0.3))
    arena = torch.empty(T * (ld + nh * hd) + hd // 2, device="cuda")
    arena[:T * ld] = x.view(-1)
    arena[T * (ld + nh * hd):] = inv_freq(hd).cuda()
    # keys above the old scales now and then: their pages are rescaled
    pool = random_pool(c, (npages,), gen)
    st = dict(arena=arena, ld=ld, T=T, lens=lens, old=old, pool=pool, maxpages=maxpages,
              ix=Ints(cu=offsets(lens), len=old, table=page_table(pages, maxpages, npages, gen)))
    if c["rows16"]:
        st["kv_rows"] = torch.empty((2, T, nkv * hd), device="cuda", dtype=torch.float16)
    return st


def append_outputs(c, st):
    nh, hd, T = c["nheads"], c["head_dim"], st["T"]
    k, v, sc = parts(st["pool"], c)
    out = dict(q=st["arena"][T * st["ld"]:T * (st["ld"] + nh * hd)].view(T, nh * hd), k=k, v=v, scales=sc)
    if c["rows16"]:
        out["rows"] = st["kv_rows"]
    return out


def own_append(c, st):
    from lama32_mojo_amd import q8hip
    nh, nkv, hd, T, ld = c["nheads"], c["nkv"], c["head_dim"], st["T"], st["ld"]
    q8hip.kv8_append(context(), st["arena_buf"], 0, nh * hd, (nh + nkv) * hd, T * (ld + nh * hd), T * ld,
                     st["pool_buf"], 0, st["pool"].shape[0], c["page"], st["ix_buf"], st["ix"].at("cu"),
                     st["ix"].at("len"), st["ix"].at("table"), c["nseq"], T, st["maxpages"], nh, nkv, hd,
                     ld=ld, kv=st.get("kv_rows_buf"), okc_f16=0, ovc_f16=T * nkv * hd)
    return append_outputs(c, st)


def plain_append(c, st):
    nh, nkv, hd, P, T, ld = c["nheads"], c["nkv"], c["head_dim"], c["page"], st["T"], st["ld"]
    ix = st["ix"]
    cu, old, tab = ix["cu"].long(), ix["len"].long(), ix["table"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(c["nseq"], device="cuda"), n, output_size=T)
    pos = old[seq] + torch.arange(T, device="cuda") - cu[seq]
    x = st["arena"][:T * ld].view(T, ld)
    inv = st["arena"][T * (ld + nh * hd):]
    # angles of far positions, and keys next to a border of two codes, in 64 bits
    ang = pos[:, None].double() * inv.double()[None]
    cs, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    h = x[:, :(nh + nkv) * hd].double().view(T, nh + nkv, 2, hd // 2)
    a, b = h[:, :, 0], h[:, :, 1]
    h = torch.cat([a * cs - b * sn, b * cs + a * sn], -1).float()
    st["arena"][T * ld:T * (ld + nh * hd)] = h[:, :nh].reshape(-1)
    k, v = h[:, nh:], x[:, (nh + nkv) * hd:].view(T, nkv, hd)
    if c["rows16"]:
        st["kv_rows"][0] = k.reshape(T, -1).half()
        st["kv_rows"][1] = v.reshape(T, -1).half()
    # every page that a sequence touches, [nseq, touched] (past the last one: the last one again)
    first, last = old // P, (old + n - 1) // P
    most = (max(st["lens"]) + P - 2) // P + 1
    slot = torch.minimum(first[:, None] + torch.arange(most, device="cuda"), last[:, None])
    page = tab.gather(1, slot)
    t = slot[:, :, None] * P + torch.arange(P, device="cuda")                # positions [nseq, touched, P]
    is_old = (t < old[:, None, None])[:, :, None, :, None]
    row = cu[:-1, None, None] + t - old[:, None, None]
    fresh = (~is_old[:, :, 0, :, 0] & (t < (old + n)[:, None, None]))[:, :, None, :, None]
    row = row.clamp(0, T - 1)
    kc, vc, sc = parts(st["pool"], c)
    for x, codes, which in ((k, kc, 0), (v, vc.transpose(-1, -2), 1)):
        new = x[row].transpose(2, 3)                                           # [nseq, touched, nkv, P, hd]
        s0 = sc[page][:, :, which] * (slot * P < old[:, None])[:, :, None]
        amax = (new.abs() * fresh).amax((-1, -2))
        s1 = torch.maximum(s0, amax / 127.0)
        was = codes[page]
        d = torch.where(s1 > 0, s1, 1.0)[..., None, None].double()
        again = torch.round(was.double() * s0[..., None, None].double() / d)
        again = torch.where((s1 > s0)[..., None, None], again, was.double())
        now = torch.where(fresh, torch.round(new.double() / d).clamp(-127, 127),
                          torch.where(is_old, again, was.double()))
        codes[page] = now.to(torch.int8)
        sc[page, which] = s1
    return append_outputs(c, st)


# ---- the 8-bit cache: attention -------------------------------------------------------

def prepare_cache(c, gen):
    nh, nkv, hd, P, nseq = c["nheads"], c["nkv"], c["head_dim"], c["page"], c["nseq"]
    lens = host_ints(1, nseq, 1, c["most"])
    ctx = host_ints(2, nseq, max(1, c["ctx"] // 16), c["ctx"])
    T = sum(lens)
    pages = [-(-(o + n) // P) for o, n in zip(ctx, lens)]
    npages, maxpages = sum(pages) + 3, max(pages) + 1
    ldq = (nh + 2 * nkv) * hd
    arena = torch.empty(T * (ldq + nh * hd), device="cuda")
    arena[:T * ldq] = normal((T * ldq,), gen)
    return dict(arena=arena, ldq=ldq, T=T, lens=lens, ctx=ctx, maxpages=maxpages,
                pool=random_pool(c, (npages,), gen),
                ix=Ints(cu=offsets(lens), len=ctx, table=page_table(pages, maxpages, npages, gen)))


def own_cache(c, st):
    from lama32_mojo_amd import q8hip
    nh, nkv, hd, T = c["nheads"], c["nkv"], c["head_dim"], st["T"]
    q8hip.kv8_attention(context(), st["arena_buf"], 0, T * st["ldq"], st["pool_buf"], 0, st["pool"].shape[0],
                        c["page"], st["ix_buf"], st["ix"].at("cu"), st["ix"].at("len"), st["ix"].at("table"),
                        c["nseq"], T, st["maxpages"], nh, nkv, hd, ldq=st["ldq"])
    return st["arena"][T * st["ldq"]:].view(T, nh * hd)


def plain_cache(c, st):
    nh, nkv, hd, P, T, nseq = c["nheads"], c["nkv"], c["head_dim"], c["page"], st["T"], c["nseq"]
    grp = nh // nkv
    ix = st["ix"]
    cu, old, tab = ix["cu"].long(), ix["len"].long(), ix["table"].long()
    n = cu[1:] - cu[:-1]
    most, held = max(st["lens"]), st["maxpages"] - 1
    tab = tab[:, :held].clamp(min=0)
    kc, vc, sc = parts(st["pool"], c)
    scales = sc[tab]                                                            # [nseq, held, 2, nkv]
    k = (kc[tab].float() * scales[:, :, 0, :, None, None]).transpose(1, 2).reshape(nseq, nkv, held * P, hd)
    v = (vc[tab].transpose(-1, -2).float() * scales[:, :, 1, :, None, None]).transpose(1, 2) \
        .reshape(nseq, nkv, held * P, hd)
    # rows padded to [nseq, most] (past a sequence's rows: its last one again)
    j = torch.minimum(torch.arange(most, device="cuda")[None], n[:, None] - 1)
    q = st["arena"][:T * st["ldq"]].view(T, st["ldq"])[:, :nh * hd]
    q = q[cu[:-1, None] + j].view(nseq, most, nkv, grp, hd).transpose(1, 2).reshape(nseq, nkv, most * grp, hd)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    s = s.view(nseq, nkv, most, grp, held * P)
    hidden = torch.arange(held * P, device="cuda") > (old[:, None] + j)[:, :, None]
    s.masked_fill_(hidden[:, None, :, None], -math.inf)
    o = torch.matmul(softmax_(s).view(nseq, nkv, most * grp, held * P), v)
    o = o.view(nseq, nkv, most, grp, hd).transpose(1, 2).reshape(nseq, most, nh * hd)
    seq = torch.repeat_interleave(torch.arange(nseq, device="cuda"), n, output_size=T)
    return o[seq, torch.arange(T, device="cuda") - cu[seq]]


# ---- pages ------------------------------------------------------------------------------

def prepare_pages(c, gen):
    """Sequences of 1 to `ctx` tokens; with beams, the first slot of each group of them
    holds one and the others are empty."""
    P, nslots, beams = c["page"], c["nslots"], c["beams"]
    length = torch.tensor(host_ints(1, nslots, max(1, c["ctx"] // 8), c["ctx"]))
    slot = torch.arange(nslots)
    source = slot - slot % beams
    length[source != slot] = 0
    pages = [-(-n // P) for n in length.tolist()]
    longest = length[source] + c["grow"]                     # of each slot, once it continues its source
    maxpages = -(-int(longest.max()) // P) + 2
    npages = sum(pages) + nslots * (-(-c["grow"] // P) + 2)
    table = page_table(pages, maxpages, npages, gen)
    ref = torch.zeros(npages, dtype=torch.int32, device="cuda")
    ref[table[table >= 0].long()] = 1
    return dict(pool=random_pool(c, (c["layers"], npages), gen), npages=npages, maxpages=maxpages,
                ix=Ints(table=table, len=length, held=pages, ref=ref, source=source, want=longest,
                        new=longest - c["grow"] // 2))       # part of what was wanted is kept


def restart(st):
    """The int32 state as it was before the pass, on the stream of the calls."""
    if own:
        with torch.cuda.stream(torch.cuda.ExternalStream(context().stream)):
            st["ix"].now.copy_(st["ix"].start)
    else:
        st["ix"].now.copy_(st["ix"].start)


def pages_outputs(st):
    return {n: st["ix"][n] for n in ("table", "len", "held", "ref")} | {"pool": st["pool"]}


def own_pages(c, st):
    from lama32_mojo_amd import q8hip
    ix, ib, ctx, pb = st["ix"], st["ix_buf"], context(), page_bytes(c)
    restart(st)
    state = (ix.at("table"), ix.at("len"), ix.at("held"), ix.at("ref"))
    shape = (c["nslots"], st["maxpages"], st["npages"])
    if c["beams"] > 1:
        q8hip.pages_fork(ctx, ib, *state, ix.at("source"), *shape)
    q8hip.pages_reserve(ctx, ib, *state, ix.at("want"), *shape, c["page"], st["pool_buf"], 0, pb, c["layers"],
                        st["npages"] * pb)
    q8hip.pages_set_len(ctx, ib, *state, ix.at("new"), *shape, c["page"])
    return pages_outputs(st)


def references(pages, on, npages):
    """How often each page is named in `pages` where `on`."""
    at = torch.where(on, pages, npages).long().reshape(-1)
    return torch.zeros(npages + 1, device="cuda", dtype=torch.int32) \
        .index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:npages]


def plain_pages(c, st):
    ix, P, npages = st["ix"], c["page"], st["npages"]
    restart(st)
    tab, length, held, ref = ix["table"], ix["len"], ix["held"], ix["ref"]
    cols = torch.arange(st["maxpages"], device="cuda", dtype=torch.int32)
    if c["beams"] > 1:                                      # fork: tables, lengths, references
        src = ix["source"].long()
        for x in (tab, length, held):
            x.copy_(x[src])
        ref.copy_(references(tab, cols < held[:, None], npages))
    # reserve: a page of its own for each slot that will write to a shared one, then the pages
    # up to the length wanted, from the lowest free page up
    want, at = ix["want"], (length // P).long()[:, None]
    mine = tab.gather(1, at)
    copy = (length % P != 0) & (want > length) & (ref[mine[:, 0].clamp(min=0).long()] > 1)
    more = ((want + P - 1) // P - held).clamp(min=0)
    need = copy.int() + more
    off = torch.cumsum(need, 0) - need
    rank = torch.cumsum((ref == 0).int(), 0) - 1
    free = torch.empty(npages + 1, device="cuda", dtype=torch.int32)
    free[torch.where(ref == 0, rank, npages).long()] = torch.arange(npages, device="cuda", dtype=torch.int32)
    own_page = torch.where(copy[:, None], free[off[:, None].clamp(max=npages)], mine)
    k = cols - held[:, None]                                # the k-th page more of a slot
    grow = (k >= 0) & (k < more[:, None])
    new = free[(off + copy)[:, None].add(k).clamp(0, npages).long()]
    ref += references(new, grow, npages) + references(own_page, copy[:, None], npages) \
        - references(mine, copy[:, None], npages)
    tab.scatter_(1, at, own_page)
    tab.copy_(torch.where(grow, new, tab))
    held += more
    st["pool"][:, own_page[:, 0].clamp(min=0).long()] = st["pool"][:, mine[:, 0].clamp(min=0).long()]
    # lengths; the pages behind them are given back
    length.copy_(ix["new"])
    keep = (length + P - 1) // P
    drop = (cols >= keep[:, None]) & (cols < held[:, None])
    ref -= references(tab, drop, npages)
    tab.masked_fill_(drop, -1)
    held.copy_(torch.minimum(held, keep))
    return pages_outputs(st)


def prepare_compact(c, gen):
    """A pool where two of three sequences have ended."""
    P, nslots = c["page"], c["nslots"]
    length = host_ints(1, nslots, max(1, c["ctx"] // 8), c["ctx"])
    alive = [i % 3 == 0 for i in range(nslots)]
    pages = [-(-n // P) for n in length]
    npages, maxpages = sum(pages) + 9, max(pages) + 1
    table = page_table(pages, maxpages, npages, gen)
    table[~torch.tensor(alive, device="cuda")] = -1
    ref = torch.zeros(npages, dtype=torch.int32, device="cuda")
    ref[table[table >= 0].long()] = 1
    return dict(pool=random_pool(c, (c["layers"], npages), gen), npages=npages, maxpages=maxpages,
                ix=Ints(table=table, len=[n * a for n, a in zip(length, alive)],
                        held=[n * a for n, a in zip(pages, alive)], ref=ref, live=[0]))


def own_compact(c, st):
    from lama32_mojo_amd import q8hip
    ix, pb = st["ix"], page_bytes(c)
    restart(st)
    q8hip.pages_compact(context(), st["ix_buf"], ix.at("table"), ix.at("held"), ix.at("ref"), ix.at("live"),
                        c["nslots"], st["maxpages"], st["npages"], st["pool_buf"], 0, pb, c["layers"],
                        st["npages"] * pb)
    return pages_outputs(st) | {"live": ix["live"]}


def plain_compact(c, st):
    ix, npages = st["ix"], st["npages"]
    restart(st)
    tab, ref = ix["table"], ix["ref"]
    ids = torch.arange(npages, device="cuda")
    live = ref > 0
    ix["live"][0] = live.sum()
    src = torch.nonzero(live & (ids >= live.sum()))[:, 0]
    dst = torch.nonzero(~live & (ids < live.sum()))[:, 0]
    st["pool"][:, dst] = st["pool"][:, src]
    to = ids.int()
    to[src] = dst.int()
    ref[dst] = ref[src]
    ref[src] = 0
    tab.copy_(torch.where(tab >= 0, to[tab.clamp(min=0).long()], tab))
    return pages_outputs(st) | {"live": ix["live"]}


# ---- work ---------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once."""
    c, k = case, case["kind"]
    hd, nkv = c["head_dim"], c["nkv"]
    if k == "packed":
        lens, nh = packed_lens(c), c["nheads"]
        T = sum(lens)
        return {"bytes": T * hd * (2 * nh * (4 if c["act"] == "f32" else 2) + 2 * 2 * nkv),
                "flops": 4 * hd * nh * sum(n * (n + 1) // 2 for n in lens)}
    if k == "append":
        T, nh = sum(host_ints(1, c["nseq"], max(1, c["most"] // 8), c["most"])), c["nheads"]
        return {"bytes": T * hd * (8 * nh + nkv * (8 + 2 + (4 if c["rows16"] else 0))),
                "flops": T * hd * (3 * nh + 3 * nkv + 4 * nkv)}
    if k == "cache":
        lens, nh = host_ints(1, c["nseq"], 1, c["most"]), c["nheads"]
        ctx = host_ints(2, c["nseq"], max(1, c["ctx"] // 16), c["ctx"])
        pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(ctx, lens))
        return {"bytes": sum(o + n for o, n in zip(ctx, lens)) * 2 * nkv * hd + 8 * sum(lens) * nh * hd,
                "flops": 4 * hd * nh * pairs}
    P, nslots = c["page"], c["nslots"]
    lens = host_ints(1, nslots, max(1, c["ctx"] // 8), c["ctx"])
    if k == "compact":
        pages = [-(-n // P) for n in lens]
        total, live = sum(pages) + 9, sum(pages[::3])
        moved = live * (total - live) // total              # of pages in random order
        return {"bytes": 2 * moved * c["layers"] * page_bytes(c) + 4 * (total + 2 * live), "flops": total}
    lens = [lens[i - i % c["beams"]] for i in range(nslots)]
    held = sum(-(-n // P) for n in lens)
    copied = sum(1 for n in lens if n % P) if c["beams"] > 1 else 0
    return {"bytes": 2 * copied * c["layers"] * page_bytes(c) + 4 * (2 * held + 8 * nslots), "flops": held}


# ---- float64 --------------------------------------------------------------------------------

def exact(case, seed):
    k = case["kind"]
    return globals()["exact_" + k](case, prepare(case, seed)) if k in ("packed", "append", "cache") else None


def attend64(q, k, v, first):
    """Row j of q [n, heads, hd] over keys 0 .. first + j of k, v [ctx, nkv, hd], head by head."""
    out = torch.empty_like(q)
    grp = q.shape[1] // k.shape[1]
    seen = torch.arange(k.shape[0], device="cuda")[None] <= first + torch.arange(len(q), device="cuda")[:, None]
    for h in range(q.shape[1]):
        e = torch.where(seen, q[:, h] @ k[:, h // grp].T.contiguous() / math.sqrt(q.shape[2]), -math.inf)
        e = torch.exp(e - e.max(1, keepdim=True).values)
        out[:, h] = e @ v[:, h // grp] / e.sum(1, keepdim=True)
    return out


def exact_packed(c, st):
    nh, nkv, hd = c["nheads"], c["nkv"], c["head_dim"]
    cu = offsets(packed_lens(c))
    q = st["q"][:, :nh * hd].double().view(-1, nh, hd)
    k, v = (x.double().view(-1, nkv, hd) for x in st["kv"])
    return torch.cat([attend64(q[a:b], k[a:b], v[a:b], 0) for a, b in zip(cu, cu[1:])]).view(-1, nh * hd)


def exact_cache(c, st):
    nh, nkv, hd = c["nheads"], c["nkv"], c["head_dim"]
    kc, vc, sc = parts(st["pool"], c)
    q = st["arena"][:st["T"] * st["ldq"]].view(st["T"], -1)[:, :nh * hd].double().view(-1, nh, hd)
    out, at = [], 0
    for i, (n, old) in enumerate(zip(st["lens"], st["ctx"])):
        pages = st["ix"]["table"][i, :-(-(old + n) // c["page"])].long()
        k = (kc[pages].double() * sc[pages, 0].double()[..., None, None]).transpose(1, 2).reshape(-1, nkv, hd)
        v = (vc[pages].double() * sc[pages, 1].double()[..., None, None]).permute(0, 3, 1, 2).reshape(-1, nkv, hd)
        out.append(attend64(q[at:at + n], k[:old + n], v[:old + n], old))
        at += n
    return torch.cat(out).view(-1, nh * hd)


def exact_append(c, st):
    """Sequence by sequence; the whole-numbered codes are compared as they are, so they have no
    value here."""
    nh, nkv, hd, P, T = c["nheads"], c["nkv"], c["head_dim"], c["page"], st["T"]
    x = st["arena"][:T * st["ld"]].view(T, -1).double()
    inv = st["arena"][T * (st["ld"] + nh * hd):].double()
    scales = parts(st["pool"], c)[2].double()
    qs, rows, at = [], [], 0
    for i, (n, old) in enumerate(zip(st["lens"], st["old"])):
        w = torch.polar(torch.ones(n, 1, hd // 2, device="cuda", dtype=torch.float64),
                        torch.arange(old, old + n, device="cuda").double()[:, None, None] * inv)
        h = x[at:at + n, :(nh + nkv) * hd].reshape(n, nh + nkv, 2, hd // 2)
        h = torch.complex(h[:, :, 0].contiguous(), h[:, :, 1].contiguous()) * w
        h = torch.cat([h.real, h.imag], -1)
        kv = torch.stack([h[:, nh:].reshape(n, -1), x[at:at + n, (nh + nkv) * hd:]])
        qs.append(h[:, :nh].reshape(n, -1))
        rows.append(kv)
        for b in range(old // P, (old + n - 1) // P + 1):
            a, z = max(b * P - old, 0), min((b + 1) * P - old, n)
            page = int(st["ix"]["table"][i, b])
            top = kv[:, a:z].reshape(2, z - a, nkv, hd).abs().amax((1, 3)) / 127.0
            scales[page] = torch.maximum(scales[page], top) if old > b * P else top
        at += n
    out = dict(q=torch.cat(qs), k=None, v=None, scales=scales)
    if c["rows16"]:
        out["rows"] = torch.cat(rows, 1)
    return out
