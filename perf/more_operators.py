"""Operators of a serving batch whose requests differ, as timed cases: drawing tokens
from rows of logits, low-rank adapters beside a shared projection, and attention of
sequences that share a long prefix in the 8-bit paged cache.

`own` false: the plain form of each operator in torch.  `own` true: the calls that
a program makes of this package's entry points.  `exact` restates the operators in
float64, row by row and sequence by sequence.

Formulas

  sample   x the row's logits, M their maximum, T the temperature, w_i = exp((x_i - M) / T).
           In the order of x descending, then index ascending, the first k tokens are kept
           (k <= 0: all), of these the ones before which less than top_p of the kept sum
           lies, of these the ones with w_i >= min_p.  The drawn token is the first one whose
           running sum exceeds u times the sum of all kept.  T <= 0: the first in the order.
           logp is the log of the token's share of the kept sum.
  adapters y[r] = base[r] + scale B (A x[r]) of the row's adapter (none: base[r]); stacked
           projections (q|k|v, gate|up) have an A each and share x.
  shared   causal attention of each sequence's rows over its cached tokens; sequences of a
           group name the same pages for their first tokens.
"""

import math

import numpy as np
import torch

own = False

HEADS = [(32, 8, 64), (32, 8, 128), (16, 8, 128)]    # (query heads, KV heads, head_dim)


def listed():
    return [
        # one conversation, a vocabulary of 128256, the usual filters: latency counts
        dict(name="sample 1 row", kind="sample", rows=1, n=128256, filters="k+p"),
        # a vocabulary of odd size (rows start at any float), min-p
        dict(name="sample odd vocabulary", kind="sample", rows=37, n=32003, filters="min-p"),
        # a serving batch in which every request has its own settings, greedy ones among them
        dict(name="sample 64 rows mixed", kind="sample", rows=64, n=128256, filters="mixed"),
        # the largest batch and vocabulary, nucleus sampling alone: most of the mass is sorted
        dict(name="sample 256 rows top-p", kind="sample", rows=256, n=151936, filters="p"),
        # one request with one small adapter at an attention output projection
        dict(name="adapters 1 row", kind="lora", lens="1", na=3, ranks="8", m=2048, widths="2048", dtype="bf16"),
        # a decode step of 64 requests over 24 adapters of several ranks at q|k|v, some without
        dict(name="adapters decode step", kind="lora", lens="1*64", na=24, ranks="8,16,16,32,64", m=4096,
             widths="4096,1024,1024", dtype="bf16"),
        # prompts of several requests in one pass at gate|up
        dict(name="adapters prompts", kind="lora", lens="700,33,1024,512,90,1,1300,256,64,150", na=5,
             ranks="16,64,32", m=4096, widths="14336,14336", dtype="bf16"),
        # float32 adapters of odd ranks, odd widths, drafted tokens beside a short prompt
        dict(name="adapters f32 odd", kind="lora", lens="5,1,3,70,2,0,1,9", na=6, ranks="5,12,31", m=1600,
             widths="1000,203,203", dtype="f32"),
        # eight answers after one system prompt, 64-dim heads, four layers
        dict(name="shared prefix small", kind="shared", groups=1, per=8, solo=0, most=1, prefix=1000, tail=100,
             page=64, layers=4, nheads=32, nkv=8, head_dim=64),
        # drafted tokens of three groups, small pages
        dict(name="shared prefix drafts", kind="shared", groups=3, per=8, solo=2, most=5, prefix=3000, tail=200,
             page=16, layers=2, nheads=16, nkv=8, head_dim=128),
        # a serving batch after one long system prompt, four requests of other origin among it
        dict(name="shared prefix 64 sequences", kind="shared", groups=1, per=60, solo=4, most=1, prefix=8000,
             tail=500, page=64, layers=2, nheads=32, nkv=8, head_dim=128),
        # many questions about one very long document
        dict(name="shared prefix long", kind="shared", groups=1, per=128, solo=0, most=1, prefix=32000,
             tail=900, page=128, layers=1, nheads=32, nkv=8, head_dim=128),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed kinds and ranges, at another size."""
    kind = rng.choice(["sample", "lora", "shared"])
    if kind == "sample":
        n = log_int(rng, 500, 151936)
        return dict(kind=kind, rows=log_int(rng, 1, min(256, 20000000 // n)), n=n,
                    filters=rng.choice(["none", "k", "p", "k+p", "min-p", "mixed", "mixed"]))
    if kind == "lora":
        if rng.random() < 0.5:
            lens = "%d*%d" % (rng.choice([1, 1, 1, 4]), log_int(rng, 1, 128))
        else:
            lens = ",".join(str(log_int(rng, 1, 1000)) for _ in range(rng.randint(1, 8)))
        m = 32 * log_int(rng, 16, 448)
        widths = [log_int(rng, 100, 8000) for _ in range(rng.randint(1, 3))]
        return dict(kind=kind, lens=lens, na=log_int(rng, 1, 40), m=m, widths=",".join(map(str, widths)),
                    ranks=",".join(str(log_int(rng, 1, 64)) for _ in range(rng.randint(1, 4))),
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    nh, nkv, hd = rng.choice(HEADS)
    groups = rng.choice([1, 1, 2, 4])
    per = log_int(rng, 2, 96 // groups)
    return dict(kind=kind, groups=groups, per=per, solo=rng.randint(0, 5), most=rng.choice([1, 1, rng.randint(2, 8)]),
                prefix=log_int(rng, 100, min(16000, 400000 // (groups * per))), tail=log_int(rng, 1, 600),
                page=rng.choice([16, 32, 64, 128]), layers=rng.randint(1, 3), nheads=nh, nkv=nkv, head_dim=hd)


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


class Ints:
    """The int32 arrays of a call in one arena, by name."""

    def __init__(self, **arrays):
        self.off, flat = {}, []
        for name, t in arrays.items():
            t = torch.as_tensor(t, dtype=torch.int32, device="cuda")
            self.off[name] = (sum(x.numel() for x in flat), t.shape)
            flat.append(t.reshape(-1))
        self.now = torch.cat(flat)

    def __getitem__(self, name):
        at, shape = self.off[name]
        return self.now[at:at + math.prod(shape)].view(shape)

    def at(self, name):
        return self.off[name][0]


def prepare(case, seed):
    st = globals()["prepare_" + case["kind"]](case, generator(seed))
    st["case"] = case
    if own:
        for name in [n for n in ("arena", "pool", "weights") if n in st]:
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


# ---- drawing tokens ----------------------------------------------------------------

SETTINGS = {                                   # (temperature, k, top_p, min_p) of rows in turn
    "none": [(1.0, 0, 1.0, 0.0)],
    "k": [(0.8, 40, 1.0, 0.0), (1.0, 200, 1.0, 0.0)],
    "p": [(1.0, 0, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.2, 0, 0.99, 0.0)],
    "k+p": [(0.7, 50, 0.95, 0.0)],
    "min-p": [(1.0, 0, 1.0, 0.05), (1.5, 0, 1.0, 0.1)],
    "mixed": [(0.7, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (0.6, 20, 0.95, 0.01),
              (1.3, 1000, 1.0, 0.0), (1.0, 0, 1.0, 0.0)],
}


def prepare_sample(c, gen):
    """Logits of a peaked head over a wide bulk; in every third row half of the tokens are
    ruled out (-inf), as a grammar does."""
    R, n = c["rows"], c["n"]
    arena = torch.empty(R * n + 5 * R, device="cuda")
    x = arena[:R * n].view(R, n)
    torch.randn((R, n), device="cuda", generator=gen, out=x)
    x *= torch.rand((R, 1), device="cuda", generator=gen) * 2 + 1
    peaks = torch.randint(0, n, (R, 20), device="cuda", generator=gen)
    x.scatter_add_(1, peaks, torch.rand((R, 20), device="cuda", generator=gen) * 10)
    out = torch.rand((len(x[2::3]), n), device="cuda", generator=gen) < 0.5
    x[2::3] = x[2::3].masked_fill(out, -math.inf)
    sets = [SETTINGS[c["filters"]][r % len(SETTINGS[c["filters"]])] for r in range(R)]
    par = arena[R * n:].view(5, R)                 # temperature, top_p, min_p, u; logp
    for i, v in ((0, 0), (1, 2), (2, 3)):
        par[i] = torch.tensor([s[v] for s in sets], device="cuda")
    par[3] = torch.rand(R, device="cuda", generator=gen)
    return dict(arena=arena, x=x, par=par, ix=Ints(k=[s[1] for s in sets], ids=[0] * R))


def own_sample(c, st):
    from lama32_mojo_amd import q8hip
    R, n = c["rows"], c["n"]
    q8hip.sample(context(), st["arena_buf"], 0, R, n, R * n, st["ix_buf"], st["ix"].at("k"), st["ix"].at("ids"),
                 lp=st["arena_buf"], olp=R * n + 4 * R)
    return dict(ids=st["ix"]["ids"], logp=st["par"][4])


def plain_sample(c, st):
    x, par = st["x"], st["par"]
    x, order = torch.sort(x.masked_fill(x.isnan(), -math.inf), dim=-1, descending=True, stable=True)
    temp, top_p, min_p, u = par[:4, :, None].double()
    greedy = temp <= 0
    # weights and their running sums in 64 bits: a token next to a border is in or out by them
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, temp))
    k = st["ix"]["k"][:, None]
    k = torch.where(greedy, 1, torch.where(k <= 0, x.shape[1], k))
    w *= torch.arange(x.shape[1], device="cuda") < k
    run_sum = torch.cumsum(w, -1)
    keep = ((run_sum - w < top_p * run_sum[:, -1:]) | (top_p >= 1)) & (w >= min_p)
    keep[:, 0] = True
    w *= keep
    run_sum = torch.cumsum(w, -1)
    last = (w > 0).sum(-1, keepdim=True) - 1       # (what is kept is a head of the order)
    at = torch.minimum((run_sum <= u * run_sum[:, -1:]).sum(-1, keepdim=True), last)
    logp = torch.log(w.gather(1, at) / run_sum[:, -1:])
    return dict(ids=order.gather(1, at)[:, 0].int(), logp=logp[:, 0].float())


# ---- adapters ------------------------------------------------------------------------

def lora_shape(c):
    """Rows, the sequences' adapters, the adapters' ranks and their sum widths."""
    a, _, b = c["lens"].partition("*")
    lens = [int(a)] * int(b) if b else [int(v) for v in c["lens"].split(",")]
    g = torch.Generator().manual_seed(7 * len(lens) + c["na"])
    # a few adapters serve most requests; one request in eight has none
    ids = (torch.rand(len(lens), generator=g) ** 2 * c["na"]).long()
    if len(lens) > 4:
        ids[torch.rand(len(lens), generator=g) < 0.125] = -1
    ranks = [int(v) for v in c["ranks"].split(",")]
    return lens, ids.tolist(), [ranks[i % len(ranks)] for i in range(c["na"])], [int(v) for v in c["widths"].split(",")]


def up8(r):
    return (r + 7) // 8 * 8


def prepare_lora(c, gen):
    lens, ids, ranks, widths = lora_shape(c)
    T, m, n, R, parts = sum(lens), c["m"], sum(widths), up8(max(ranks)), len(widths)
    # per adapter: an A per part [up8(rank), m], one B [n, up8(rank)], zeros behind the rank
    flat = normal((c["na"] * R * (parts * m + n),), gen)
    sa, sb = parts * R * m, n * R
    A, B = flat[:c["na"] * sa].view(c["na"], sa), flat[c["na"] * sa:].view(c["na"], sb)
    A *= 1.0 / math.sqrt(m)
    B *= 0.02
    for i, r in enumerate(ranks):
        A[i, :parts * up8(r) * m].view(parts, up8(r), m)[:, r:] = 0
        B[i, :n * up8(r)].view(n, up8(r))[:, r:] = 0
    weights = flat.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
    arena = torch.empty(T * (m + 2 * n) + c["na"], device="cuda")
    x, base = arena[:T * m].view(T, m), arena[T * m:T * (m + n)].view(T, n)
    x.copy_(normal((T, m), gen) * torch.exp(normal((T, 1), gen, 0.5)))
    base.copy_(normal((T, n), gen))
    arena[T * (m + 2 * n):] = torch.tensor([16.0 / r for r in ranks], device="cuda")
    return dict(arena=arena, weights=weights, x=x, base=base, y=arena[T * (m + n):T * (m + 2 * n)].view(T, n),
                scale=arena[T * (m + 2 * n):], lens=lens, sa=sa, sb=sb, R=R,
                ix=Ints(cu=offsets(lens), id=ids, rank=ranks))


def own_lora(c, st):
    from lama32_mojo_amd import q8hip
    (T, n), m, na, ix = st["base"].shape, c["m"], c["na"], st["ix"]
    widths = [int(v) for v in c["widths"].split(",")]
    q8hip.lora(context(), st["weights_buf"], 0, st["sa"], na * st["sa"], st["sb"], na, st["R"], st["arena_buf"], 0,
               T * m, T * (m + n), T * (m + 2 * n), st["ix_buf"], ix.at("cu"), ix.at("id"), ix.at("rank"),
               len(st["lens"]), T, m, widths, dtype=c["dtype"])
    return st["y"]


def plain_lora(c, st):
    """Rows by adapter, padded to [na + 1, most, m]; the last ones have none."""
    na, m, R, ix, x, base = c["na"], c["m"], st["R"], st["ix"], st["x"], st["base"]
    widths = [int(v) for v in c["widths"].split(",")]
    parts, (T, n) = len(widths), base.shape
    cu = ix["cu"].long()
    who = torch.where(ix["id"] < 0, na, ix["id"]).long()
    who = torch.repeat_interleave(who, cu[1:] - cu[:-1], output_size=T)
    who, rows = torch.sort(who, stable=True)
    count = (who == torch.arange(na + 1, device="cuda")[:, None]).sum(1)
    place = torch.arange(T, device="cuda") - (torch.cumsum(count, 0) - count)[who]
    most = int(place.max()) + 1
    xp = torch.zeros((na, most, m), device="cuda")
    real = who < na
    xp[who[real], place[real]] = x[rows[real]]
    # the adapters' matrices at their largest rank
    rank = ix["rank"].long()
    pitch, j = (rank + 7) // 8 * 8, torch.arange(R, device="cuda")
    on = (j < rank[:, None]).float()                                            # [na, R]
    A = st["weights"][:na * st["sa"]].view(na, parts * R, m)
    at = torch.arange(parts, device="cuda")[None, :, None] * pitch[:, None, None] + j
    A = torch.gather(A, 1, at.clamp(max=parts * R - 1).view(na, -1, 1).expand(-1, -1, m)).float()
    A = A * on.repeat(1, parts)[:, :, None]
    B = st["weights"][na * st["sa"]:].view(na, n * R)
    at = torch.arange(n, device="cuda")[None, :, None] * pitch[:, None, None] + j
    B = torch.gather(B, 1, at.clamp(max=n * R - 1).view(na, -1)).view(na, n, R).float() * on[:, None]
    xa = torch.matmul(xp, A.transpose(1, 2)) * st["scale"][:, None, None]
    first = torch.tensor(offsets(widths))
    d = [torch.matmul(xa[:, :, p * R:(p + 1) * R], B[:, first[p]:first[p + 1]].transpose(1, 2)) for p in range(parts)]
    st["y"].copy_(base)
    st["y"][rows[real]] += torch.cat(d, -1)[who[real], place[real]]
    return st["y"]


# ---- attention after a shared prefix ------------------------------------------------------

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


def shared_shape(c):
    """Per sequence: its rows, its cached tokens, its group (solo ones: a group each), and the
    pages that each group shares.  Groups' members are spread over the slots."""
    P, G = c["page"], c["groups"]
    ns = G * c["per"] + c["solo"]
    group = [i % G for i in range(G * c["per"])] + [G + i for i in range(c["solo"])]
    g = torch.Generator().manual_seed(ns)
    group = [group[i] for i in torch.randperm(ns, generator=g).tolist()]
    shared = [max(1, n // P) for n in host_ints(3, G, max(1, c["prefix"] // 2), c["prefix"])] + [0] * c["solo"]
    tail = host_ints(2, ns, 1, c["tail"])
    lone = host_ints(4, ns, max(1, c["prefix"] // 8), c["prefix"])
    old = [shared[k] * P + tail[i] if k < G else lone[i] for i, k in enumerate(group)]
    return host_ints(1, ns, 1, c["most"]), old, group, shared


def prepare_shared(c, gen):
    nh, nkv, hd, P, L = c["nheads"], c["nkv"], c["head_dim"], c["page"], c["layers"]
    lens, old, group, shared = shared_shape(c)
    T, ns = sum(lens), len(lens)
    mine = [-(-(o + n) // P) - shared[k] for o, n, k in zip(old, lens, group)]
    npages = sum(shared) + sum(mine) + 3
    maxpages = max(a + shared[k] for a, k in zip(mine, group)) + 1
    ids = torch.randperm(npages, generator=gen, device="cuda").tolist()
    take = lambda n: [ids.pop() for _ in range(n)]                        # noqa: E731
    heads = [take(n) for n in shared]
    table = [heads[k] + take(a) for a, k in zip(mine, group)]
    table = [row + [-1] * (maxpages - len(row)) for row in table]
    pool = torch.randint(0, 255, (L, npages, page_bytes(c)), device="cuda", generator=gen, dtype=torch.uint8)
    pool ^= 128                                             # codes -128 .. 126
    k, v, sc = parts(pool, c)
    k.clamp_(min=-127)
    v.clamp_(min=-127)
    sc.copy_(torch.exp(torch.randn(sc.shape, device="cuda", generator=gen) * 0.3) * 0.02)
    ldq = (nh + 2 * nkv) * hd                              # q inside stacked q|k|v rows
    arena = torch.empty(L * T * (ldq + nh * hd), device="cuda")
    arena[:L * T * ldq] = normal((L * T * ldq,), gen)
    return dict(arena=arena, pool=pool, ldq=ldq, T=T, lens=lens, old=old, group=group, shared=shared,
                q=arena[:L * T * ldq].view(L, T, ldq)[:, :, :nh * hd], out=arena[L * T * ldq:].view(L, T, nh * hd),
                maxpages=maxpages, ix=Ints(cu=offsets(lens), len=old, table=table, share=[0] * (8 * ns + T + 16)))


def own_shared(c, st):
    """A step's attention: what the slots share is found once, then every layer uses it."""
    from lama32_mojo_amd import q8hip
    L, npages = st["pool"].shape[:2]
    T, ns, ix, ctx = st["T"], len(st["lens"]), st["ix"], context()
    arrays = (st["ix_buf"], ix.at("cu"), ix.at("len"), ix.at("table"), ns, T, st["maxpages"])
    q8hip.kv8_share(ctx, *arrays, npages, c["page"], ix.at("share"))
    qd = c["nheads"] * c["head_dim"]
    for i in range(L):
        q8hip.kv8_attention_shared(ctx, st["arena_buf"], i * T * st["ldq"], L * T * st["ldq"] + i * T * qd,
                                   st["pool_buf"], i * npages * page_bytes(c), npages, c["page"], *arrays,
                                   c["nheads"], c["nkv"], c["head_dim"], ix.at("share"), ldq=st["ldq"])
    return st["out"]


def partial(q, k, v, seen):
    """Unnormalised sums over the keys, their largest scores and weights' sums, of q [.., r, hd]
    over k and v [.., t, hd] where seen."""
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s -= m.masked_fill(m == -math.inf, 0.0)
    s.exp_()
    return torch.matmul(s, v), m, s.sum(-1, keepdim=True)


def plain_shared(c, st):
    """The shared tokens once for all rows of a group, each sequence's own tokens for its rows,
    and the two joined."""
    nh, nkv, hd, P, T = c["nheads"], c["nkv"], c["head_dim"], c["page"], st["T"]
    grp, ns, ix = nh // nkv, len(st["lens"]), st["ix"]
    cu, old, tab = ix["cu"].long(), ix["len"].long(), ix["table"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(ns, device="cuda"), n, output_size=T)
    group = torch.tensor(st["group"], device="cuda")
    shared = torch.tensor(st["shared"], device="cuda")[group]                      # pages of each sequence
    most = max(st["lens"])
    held = max(-(-(o + w) // P) - st["shared"][k] for o, w, k in zip(st["old"], st["lens"], st["group"]))
    mine = shared[:, None] + torch.arange(held, device="cuda")
    pages = tab.gather(1, mine.clamp(max=tab.shape[1] - 1)).clamp(min=0)
    j = torch.minimum(torch.arange(most, device="cuda")[None], n[:, None] - 1)
    keys = (shared * P)[:, None] + torch.arange(held * P, device="cuda")
    seen = keys[:, None] <= (old[:, None] + j)[:, :, None]
    seen = seen[:, None, :, None].expand(-1, -1, -1, grp, -1).reshape(ns, 1, most * grp, held * P)
    where = torch.arange(T, device="cuda") - cu[seq]
    for i in range(c["layers"]):
        kc, vc, sc = parts(st["pool"][i], c)

        def values(p):                                     # pages [.., h] -> K and V [.., nkv, h * P, hd]
            s = sc[p]
            k = kc[p].float() * s[..., 0, :, None, None]
            v = vc[p].transpose(-1, -2).float() * s[..., 1, :, None, None]
            return (x.transpose(-3, -4).reshape(*p.shape[:-1], nkv, -1, hd) for x in (k, v))

        q = st["q"][i].reshape(T, nkv, grp, hd)
        k, v = values(pages)
        qs = q[cu[:-1, None] + j].permute(0, 2, 1, 3, 4).reshape(ns, nkv, most * grp, hd)
        o, m, l = (x.view(ns, nkv, most, grp, -1).permute(0, 2, 1, 3, 4)[seq, where] for x in partial(qs, k, v, seen))
        for g, h in enumerate(st["shared"]):
            if h == 0:
                continue
            rows = torch.nonzero(group[seq] == g)[:, 0]
            k, v = values(tab[st["group"].index(g), :h])
            qg = q[rows].permute(1, 0, 2, 3).reshape(nkv, -1, hd)
            og, mg, lg = (x.view(nkv, len(rows), grp, -1).transpose(0, 1)
                          for x in partial(qg, k, v, torch.ones((), device="cuda", dtype=torch.bool)))
            top = torch.maximum(m[rows], mg)
            a, b = torch.exp(m[rows] - top), torch.exp(mg - top)
            o[rows], l[rows], m[rows] = a * o[rows] + b * og, a * l[rows] + b * lg, top
        st["out"][i] = (o / l).reshape(T, nh * hd)
    return st["out"]


# ---- work ---------------------------------------------------------------------------------

def work(case):
    """Each input read once, each output written once."""
    c, k = case, case["kind"]
    if k == "sample":
        return {"bytes": 4 * c["rows"] * (c["n"] + 7), "flops": 3 * c["rows"] * c["n"]}
    if k == "lora":
        lens, ids, ranks, widths = lora_shape(c)
        n, m, T = sum(widths), c["m"], sum(lens)
        per = [r * (len(widths) * m + n) for r in ranks]
        used = {i for i, w in zip(ids, lens) if i >= 0 and w}
        return {"bytes": sum(per[i] for i in used) * (2 if c["dtype"] == "bf16" else 4) + 8 * T * n
                + 4 * m * sum(w for i, w in zip(ids, lens) if i >= 0),
                "flops": 2 * sum(w * per[i] for i, w in zip(ids, lens) if i >= 0)}
    lens, old, group, shared = shared_shape(c)
    P, hd, nh, nkv = c["page"], c["head_dim"], c["nheads"], c["nkv"]
    tokens = P * sum(shared) + sum(o + n - P * shared[g] for o, n, g in zip(old, lens, group))
    pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, lens))
    return {"bytes": c["layers"] * (tokens * 2 * nkv * hd + 8 * sum(lens) * nh * hd),
            "flops": c["layers"] * 4 * hd * nh * pairs}


# ---- float64 --------------------------------------------------------------------------------

def exact(case, seed):
    return globals()["exact_" + case["kind"]](case, prepare(case, seed))


def exact_sample(c, st):
    """Row by row, in the order of a sort by (-x, index)."""
    x, par, ks = st["x"].cpu().numpy(), st["par"].cpu().numpy().astype(np.float64), st["ix"]["k"].tolist()
    ids, logp = [], []
    for r in range(c["rows"]):
        temp, top_p, min_p, u = par[:4, r]
        order = np.argsort(-x[r], kind="stable")
        if temp <= 0:
            order, temp = order[:1], 1.0
        elif ks[r] > 0:
            order = order[:ks[r]]
        v = x[r][order].astype(np.float64)
        w = np.exp((v - v[0]) / temp)
        if top_p < 1:
            w = w[:max(1, int(np.searchsorted(np.concatenate([[0.0], np.cumsum(w)[:-1]]), top_p * w.sum())))]
        w = w[:max(1, int((w >= min_p).sum()))]
        run_sum = np.cumsum(w)
        at = min(int(np.searchsorted(run_sum, u * run_sum[-1], side="right")), int((w > 0).sum()) - 1)
        ids.append(int(order[at]))
        logp.append(math.log(w[at] / run_sum[-1]))
    return dict(ids=torch.tensor(ids, dtype=torch.int32), logp=torch.tensor(logp, dtype=torch.float64))


def exact_lora(c, st):
    lens, ids, ranks, widths = lora_shape(c)
    y, cu, first, n = st["base"].double(), offsets(lens), offsets(widths), sum(widths)
    for s, i in enumerate(ids):
        if i < 0:
            continue
        r, rows = ranks[i], slice(cu[s], cu[s + 1])
        A = st["weights"][i * st["sa"]:][:len(widths) * up8(r) * c["m"]].view(len(widths), up8(r), c["m"])
        B = st["weights"][c["na"] * st["sa"] + i * st["sb"]:][:n * up8(r)].view(n, up8(r))
        for p in range(len(widths)):
            t = st["x"][rows].double() @ A[p, :r].double().T.contiguous()
            t = t @ B[first[p]:first[p + 1], :r].double().T.contiguous()
            y[rows, first[p]:first[p + 1]] += t * st["scale"][i].double()
    return y


def exact_shared(c, st):
    """Sequence by sequence over all its tokens, head by head."""
    nh, nkv, hd, P = c["nheads"], c["nkv"], c["head_dim"], c["page"]
    out = torch.empty(st["out"].shape, device="cuda", dtype=torch.float64)
    for i in range(c["layers"]):
        kc, vc, sc = parts(st["pool"][i], c)
        at = 0
        for s, (n, old) in enumerate(zip(st["lens"], st["old"])):
            p = st["ix"]["table"][s, :-(-(old + n) // P)].long()
            seen = torch.arange(old + n, device="cuda")[None] <= old + torch.arange(n, device="cuda")[:, None]
            for g in range(nkv):
                k = (kc[p, g].double() * sc[p, 0, g].double()[:, None, None]).reshape(-1, hd)[:old + n]
                v = (vc[p, g].double() * sc[p, 1, g].double()[:, None, None]).transpose(1, 2).reshape(-1, hd)[:old + n]
                for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                    e = st["q"][i, at:at + n, h * hd:(h + 1) * hd].double() @ k.T.contiguous() / math.sqrt(hd)
                    e = torch.softmax(torch.where(seen, e, -math.inf), 1)
                    out[i, at:at + n, h * hd:(h + 1) * hd] = e @ v
            at += n
    return out
