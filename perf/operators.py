"""The operators of the paged K/V cache, as a serving program calls them, with their plain forms.

A cache is a pool of pages [page][kv head][row][dim] for K and for V and a table [sequence][n] that names each
sequence's pages in order: cache row j of sequence b is row j % page_size of page table[b][j / page_size].

  append   per token: RMS norm of every query and key head, rotation by the token's position, the query row written
           out, the key and value rows stored in the sequence's page
  decode   attention of one new token per sequence (the last row of its cache), over all of it or over a window of
           the last rows and a few first rows (sinks); optionally each row's attention weight, summed over the
           query heads of its K/V head, is added to the weight kept beside the cache
  prefill  attention of the last rows of each sequence (a ragged batch of prompt chunks), causal, same masks
  evict    each K/V head of a sequence keeps its first rows, its last rows and those with the largest weight, up to a
           budget, moved in order to fresh pages

Where `own` is false the operators run in their plain form: elementary torch operations in 32 bits, one rounding at
the end.
"""
import math
import os
import sys

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HEADS = [(32, 8, 64), (32, 8, 128), (16, 4, 128), (8, 2, 128), (8, 8, 64), (12, 2, 64), (16, 1, 128)]


def _lib():
    """this repository's package"""
    path = os.path.join(os.getcwd(), "pulsar-asm_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pulsar_b200
    return pulsar_b200


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 64 sequences, from the fp32 rows a Q8_0 GEMM gives, with weights kept for eviction
        dict(name="append batch of 64", op="append", nh=16, nkv=4, hd=128, page=32, dt="f16", x="f32", n_seq=64,
             n_tok=64, ctx=2048, partial=0.5, weights=True),
        # a prompt's chunk, all of it in one call
        dict(name="append prompt", op="append", nh=32, nkv=8, hd=128, page=64, dt="bf16", x="bf16", n_seq=3,
             n_tok=8191, ctx=777, partial=1.0, weights=False),
        # single-stream decode at a short context: latency
        dict(name="decode one sequence", op="decode", nh=32, nkv=8, hd=64, page=16, dt="f16", out="bf16", n_seq=1,
             lo=1029, hi=1029, window=0, sinks=0, weights=False),
        # batched decode, 64 ragged sequences of 16 to 2048 rows
        dict(name="decode 64 ragged", op="decode", nh=32, nkv=8, hd=64, page=16, dt="f16", out="bf16", n_seq=64,
             lo=16, hi=2048, window=0, sinks=0, weights=False),
        # two long documents: few rows of work, a long axis to split
        dict(name="decode long", op="decode", nh=32, nkv=8, hd=128, page=64, dt="bf16", out="bf16", n_seq=2,
             lo=65537, hi=131071, window=0, sinks=0, weights=False),
        # sliding-window layers with sinks, caches far longer than the window
        dict(name="decode window and sinks", op="decode", nh=16, nkv=4, hd=128, page=32, dt="f16", out="f16",
             n_seq=48, lo=100, hi=20000, window=4096, sinks=4, weights=False),
        # decode of caches kept at a budget by eviction: every step adds its weights
        dict(name="decode with weights", op="decode", nh=32, nkv=8, hd=128, page=32, dt="f16", out="bf16", n_seq=16,
             lo=2048, hi=4352, window=0, sinks=0, weights=True),
        # one 32-token chunk against a cache of some thousand rows
        dict(name="prefill chunk of 32", op="prefill", nh=32, nkv=8, hd=64, page=16, dt="f16", out="bf16", n_seq=1,
             tlo=32, thi=32, ctx=4099, window=0, sinks=0),
        # a ragged batch of whole prompts in a sliding-window layer with sinks
        dict(name="prefill ragged window", op="prefill", nh=16, nkv=4, hd=128, page=32, dt="bf16", out="bf16",
             n_seq=5, tlo=65, thi=4000, ctx=0, window=256, sinks=4),
        # one long prompt, full causal attention: the most arithmetic
        dict(name="prefill long prompt", op="prefill", nh=32, nkv=8, hd=128, page=64, dt="f16", out="bf16", n_seq=1,
             tlo=8192, thi=8192, ctx=0, window=0, sinks=0),
        # one sequence's cache, a block of tokens past its budget: latency
        dict(name="evict one sequence", op="evict", nh=16, nkv=4, hd=128, page=16, dt="bf16", n_seq=1, lo=1087, hi=1087,
             budget=1024, sinks=4, recent=256),
        # a batch's caches, most of them past their budget
        dict(name="evict to budget", op="evict", nh=32, nkv=8, hd=128, page=32, dt="f16", n_seq=16, lo=2500, hi=4352,
             budget=4096, sinks=4, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    nh, nkv, hd = rng.choice(HEADS)
    c = dict(op=rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict"]), nh=nh, nkv=nkv, hd=hd,
             page=rng.choice([16, 32, 64, 128]), dt=rng.choice(["f16", "bf16"]))
    if c["op"] == "append":
        n = _log(rng, 1, 8000)
        return dict(c, x=rng.choice(["bf16", "f16", "f32"]), n_tok=n, n_seq=rng.randint(1, min(n, 64)),
                    ctx=_log(rng, 1, 30000), partial=rng.choice([1.0, 0.5]), weights=rng.random() < 0.5)
    if c["op"] == "decode":
        n = _log(rng, 1, 256)
        hi = _log(rng, 1, min(130000, 200000000 // (n * nkv * hd)))    # as many bytes as the largest listed case
        win = rng.random() < 0.4
        return dict(c, out=rng.choice(["bf16", "f16"]), n_seq=n, lo=rng.randint(1, hi), hi=hi,
                    window=_log(rng, 16, 5000) if win else 0, sinks=rng.randint(0, 70) if win else 0,
                    weights=rng.random() < 0.3)
    if c["op"] == "prefill":
        n = _log(rng, 1, 8)
        thi = _log(rng, 1, 6000 // n)
        win = rng.random() < 0.4
        return dict(c, out=rng.choice(["bf16", "f16"]), n_seq=n, tlo=rng.randint(1, thi), thi=thi,
                    ctx=rng.choice([0, _log(rng, 1, 6000)]), window=_log(rng, 16, 2000) if win else 0,
                    sinks=rng.randint(0, 70) if win else 0)
    budget = _log(rng, 64, 4096)
    return dict(c, n_seq=_log(rng, 1, 16), lo=rng.randint(1, budget), hi=budget + _log(rng, 1, 512), budget=budget,
                sinks=rng.randint(0, 16), recent=rng.randint(0, budget // 4))


def _spread(n, lo, hi):
    """n lengths spread over [lo, hi], the longest first"""
    return [hi - int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lengths(c):
    if c["op"] == "append":        # rows in the cache before the call, and the tokens each sequence adds
        add = [c["n_tok"] // c["n_seq"] + (i < c["n_tok"] % c["n_seq"]) for i in range(c["n_seq"])]
        return _spread(c["n_seq"], max(1, c["ctx"] // 8), c["ctx"]), add
    if c["op"] == "prefill":       # rows in the cache with the chunk, and the chunk's tokens
        add = _spread(c["n_seq"], c["tlo"], c["thi"])
        return [x + t for x, t in zip(_spread(c["n_seq"], c["ctx"] // 3, c["ctx"]), add)], add
    return _spread(c["n_seq"], c["lo"], c["hi"]), None


# ------------------------------------------------------------------ inputs
def _norm(n, g):
    return 1.0 + 0.05 * torch.randn(n, generator=g, device="cuda")


def _pages(needs, page, g, spare=3):
    """(table int32 [n][most], pages in the pool): every (first, last] run of rows gets pages of its own, in no order"""
    first = [a // page for a, _ in needs]
    count = [-(-b // page) - f for (_, b), f in zip(needs, first)]
    width = max(1, max(f + n for f, n in zip(first, count)))
    total = sum(count) + spare
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(needs), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (f, n) in enumerate(zip(first, count)):
        table[b, f:f + n] = ids[at:at + n]
        at += n
    return table, total


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    nh, nkv, hd, page, dt = c["nh"], c["nkv"], c["hd"], c["page"], DT[c["dt"]]
    lens, add = _lengths(c)
    s = dict(case=c)
    dev = dict(device="cuda")

    def randn(*shape, to=dt, by=1.0):
        return (by * torch.randn(*shape, generator=g, **dev)).to(to)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, **dev)

    if c["op"] == "append":
        table, n_pages = _pages([(a, a + t) for a, t in zip(lens, add)], page, g)
        s["seq"] = torch.cat([torch.full((t,), b, dtype=torch.int32, **dev) for b, t in enumerate(add)])
        s["slot"] = torch.cat([torch.arange(a, a + t, dtype=torch.int32, **dev) for a, t in zip(lens, add)])
        s["pos"] = s["slot"].clone()
        half = int(hd * c["partial"]) // 2
        angle = torch.arange(max(a + t for a, t in zip(lens, add)), dtype=torch.float64, **dev)[:, None] \
            * 1e6 ** (-torch.arange(half, dtype=torch.float64, **dev) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # the projection's rows: q | k | v and nh gate values behind them
        s["qkv"] = randn(c["n_tok"], (nh + 2 * nkv) * hd + nh, to=DT[c["x"]], by=2.0)
        s["q_norm"], s["k_norm"] = _norm(hd, g), _norm(hd, g)
        s["q"] = torch.zeros(c["n_tok"], nh, hd, dtype=dt, **dev)
        weights = c["weights"]
    elif c["op"] == "evict":
        kept = [min(n, c["budget"]) for n in lens]
        both, n_pages = _pages([(0, n) for n in lens + kept], page, g)
        table = both[:len(lens)].contiguous()
        s["dst"] = both[len(lens):].contiguous()
        s["new_length"] = torch.zeros(len(lens), dtype=torch.int32, **dev)
        weights = True
    else:
        table, n_pages = _pages([(0, n) for n in lens], page, g)
        rows = sum(add) if add else len(lens)
        s["q"] = randn(rows, nh, hd, by=1.5)
        s["out"] = torch.zeros(rows, nh, hd, dtype=DT[c["out"]], **dev)
        if add:
            s["start"] = ints([sum(add[:i]) for i in range(len(add) + 1)])
        weights = c.get("weights", False)
    s["table"] = table
    if c["op"] != "append":
        s["length"] = ints(lens)
    s["k"], s["v"] = randn(n_pages, nkv, page, hd), randn(n_pages, nkv, page, hd)
    # accumulated weights: few rows hold most of it
    s["weight"] = torch.rand(n_pages, nkv, page, generator=g, **dev).pow(8) * 20 if weights else None
    return s


# ------------------------------------------------------------- plain forms
def _plain_append(s, c):
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    x = s["qkv"].float()
    n, half = x.shape[0], s["cos"].shape[1]
    q, k, v = x[:, :(nh + 2 * nkv) * hd].view(n, nh + 2 * nkv, hd).split([nh, nkv, nkv], 1)
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

    def rotated(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5) * w
        a, b = y[..., :half], y[..., hd // 2:hd // 2 + half]
        return torch.cat([a * cos - b * sin, y[..., half:hd // 2], b * cos + a * sin, y[..., hd // 2 + half:]], -1)

    s["q"].copy_(rotated(q, s["q_norm"]))
    seq, slot = s["seq"].long(), s["slot"].long()
    at = s["table"][seq, slot // page].long()
    s["k"][at, :, slot % page] = rotated(k, s["k_norm"]).to(s["k"].dtype)
    s["v"][at, :, slot % page] = v.to(s["v"].dtype)
    if s["weight"] is not None:
        s["weight"][at, :, slot % page] = 0.0
    return [s["q"], s["k"], s["v"], s["weight"]]


def _rows(pool, table):
    """[n_seq][kv head][row][...] of every page in the table"""
    x = pool[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _visible(c, last, rows):
    """last [...]: the query's own row -> [..., rows]"""
    j = torch.arange(rows, device="cuda")
    t = last[..., None]
    seen = j <= t
    return seen & ((j > t - c["window"]) | (j < c["sinks"])) if c["window"] else seen


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the seen rows; (output, weights)"""
    x = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~seen, -torch.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    x = x / x.sum(-1, keepdim=True)
    return torch.matmul(x, v), x


def _plain_decode(s, c):
    nkv, hd, n = c["nkv"], c["hd"], c["n_seq"]
    k, v = _rows(s["k"], s["table"]).float(), _rows(s["v"], s["table"]).float()
    q = s["q"].float().view(n, nkv, -1, hd)
    seen = _visible(c, s["length"].long() - 1, k.shape[2])
    v = torch.where(seen[:, None, :, None], v, 0.0)
    o, p = _attend(q, k, v, seen[:, None, None], hd ** -0.5)
    s["out"].copy_(o.reshape(n, -1, hd))
    if not c["weights"]:
        return [s["out"], None]
    page = c["page"]
    p = torch.where(seen[:, None], p.sum(2), 0.0).view(n, nkv, -1, page).transpose(1, 2)
    kept = (s["table"] >= 0)
    s["weight"].index_add_(0, s["table"][kept].long(), p[kept])
    return [s["out"], s["weight"]]


def _plain_prefill(s, c):
    nh, nkv, hd, n = c["nh"], c["nkv"], c["hd"], c["n_seq"]
    k, v = _rows(s["k"], s["table"]).float(), _rows(s["v"], s["table"]).float()
    start, rows = s["start"].long(), s["q"].shape[0]
    of = torch.searchsorted(start, torch.arange(rows, device="cuda"), right=True) - 1    # each row's sequence
    i = torch.arange(rows, device="cuda") - start[of]                                     # and its place in the chunk
    count, most = start[1:] - start[:-1], max(_lengths(c)[1])
    q = torch.zeros(n, most, nh, hd, device="cuda")
    q[of, i] = s["q"].float()
    t = (s["length"].long() - count)[:, None] + torch.arange(most, device="cuda")
    seen = _visible(c, t, k.shape[2])[:, None, None]
    q = q.view(n, most, nkv, -1, hd).permute(0, 2, 3, 1, 4)      # [seq][kv head][head of its group][token][dim]
    o, _ = _attend(q, k[:, :, None], v[:, :, None], seen, hd ** -0.5)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, most, nh, hd)[of, i])
    return s["out"]


def _plain_evict(s, c):
    page, n, nkv = c["page"], c["n_seq"], c["nkv"]
    w = _rows(s["weight"], s["table"])
    length = s["length"].long()[:, None, None]
    j = torch.arange(w.shape[2], device="cuda")
    rank = w.masked_fill((j < c["sinks"]) | (j >= length - c["recent"]), torch.inf).masked_fill(j >= length, -torch.inf)
    keep = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    keep = torch.where(keep < length, keep, w.shape[2]).sort(-1).values      # in order, none past the end
    s["new_length"].copy_(s["length"].clamp(max=c["budget"]))
    b, h, i = (keep < w.shape[2]).nonzero(as_tuple=True)
    src = keep[b, h, i]
    a = s["table"][b, src // page].long(), h, src % page
    z = s["dst"][b, i // page].long(), h, i % page
    s["k"][z], s["v"][z], s["weight"][z] = s["k"][a], s["v"][a], s["weight"][a]
    return [s["k"], s["v"], s["weight"], s["new_length"]]


# --------------------------------------------------------------- the calls
def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
                "evict": _plain_evict}[c["op"]](s, c)
    cache = s.get("cache")
    if cache is None:        # the handle of the two pools, which a program keeps as long as them
        cache = s["cache"] = _lib().KVPages(s["k"], s["v"], s["weight"])
    if c["op"] == "append":
        cache.append(s["table"], s["seq"], s["slot"], s["pos"], s["qkv"], s["q"], q_norm=s["q_norm"],
                     k_norm=s["k_norm"], eps=1e-5, cos=s["cos"], sin=s["sin"])
        return [s["q"], s["k"], s["v"], s["weight"]]
    if c["op"] == "decode":
        cache.decode(s["table"], s["length"], s["q"], s["out"], window=c["window"], sinks=c["sinks"],
                     accumulate=c["weights"])
        return [s["out"], s["weight"]]
    if c["op"] == "prefill":
        cache.prefill(s["table"], s["start"], s["length"], s["q"], s["out"], window=c["window"], sinks=c["sinks"])
        return s["out"]
    cache.evict(s["table"], s["length"], s["dst"], s["new_length"], c["budget"], sinks=c["sinks"], recent=c["recent"])
    return [s["k"], s["v"], s["weight"], s["new_length"]]


def _seen_by(c, t):
    """rows that the query at row t sees"""
    w, k = c["window"], c["sinks"]
    return t + 1 if not w else min(w, t + 1) + min(k, max(0, t + 1 - w))


def work(c):
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    lens, add = _lengths(c)
    row = nkv * hd * 2
    if c["op"] == "append":
        x = {"f32": 4, "bf16": 2, "f16": 2}[c["x"]]
        half = int(hd * c["partial"]) // 2
        wide = (nh + 2 * nkv) * hd
        return dict(bytes=c["n_tok"] * (wide * (x + 2) + 12 + 8 * half + (4 * nkv if c["weights"] else 0)),
                    flops=c["n_tok"] * (nh + nkv) * (4 * hd + 6 * half))
    if c["op"] == "evict":
        kept = [min(n, c["budget"]) for n in lens]
        return dict(bytes=sum(n * nkv * 4 for n in lens) + sum(n * (4 * row + 4 * nkv) for n in kept),
                    flops=sum(n * nkv for n in lens))
    if c["op"] == "decode":
        seen = sum(_seen_by(c, n - 1) for n in lens)
        return dict(bytes=seen * (2 * row + (8 * nkv if c["weights"] else 0)) + 4 * len(lens) * nh * hd,
                    flops=4 * seen * nh * hd)
    pairs = sum(_seen_by(c, t) for n, m in zip(lens, add) for t in range(n - m, n))
    # rows that some query of the chunk sees: the first one's window and all behind it, and the sinks
    lo = [max(0, n - m + 1 - c["window"]) if c["window"] else 0 for n, m in zip(lens, add)]
    read = sum(n - a + min(c["sinks"], a) for n, a in zip(lens, lo))
    return dict(bytes=read * 2 * row + 4 * sum(add) * nh * hd, flops=4 * pairs * nh * hd)


# ------------------------------------------------------------ in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    lens, add = _lengths(c)
    grp = nh // nkv

    def place(b, j):
        return s["table"][b].long()[j // page], j % page

    if c["op"] == "append":
        x, pos = s["qkv"].double(), s["pos"].long()
        k, v = s["k"].double(), s["v"].double()
        half = s["cos"].shape[1]
        z = torch.complex(s["cos"].double(), s["sin"].double())[pos]
        page_of = torch.stack([s["table"][b, j // page] for b, j in zip(s["seq"].tolist(), s["slot"].tolist())]).long()
        row_of = s["slot"].long() % page

        def head(h, w):
            y = x[:, h * hd:(h + 1) * hd]
            y = w.double() * y / (y.pow(2).sum(1, keepdim=True) / hd + 1e-5).sqrt()
            r = torch.complex(y[:, :half], y[:, hd // 2:hd // 2 + half]) * z
            y = y.clone()
            y[:, :half], y[:, hd // 2:hd // 2 + half] = r.real, r.imag
            return y

        q = torch.stack([head(h, s["q_norm"]) for h in range(nh)], 1)
        for h in range(nkv):
            k[page_of, h, row_of] = head(nh + h, s["k_norm"])
            v[page_of, h, row_of] = x[:, (nh + nkv + h) * hd:(nh + nkv + h + 1) * hd]
        w = s["weight"]
        if w is not None:
            w = w.double()
            w[page_of, :, row_of] = 0.0
        return [q, k, v, w]
    if c["op"] == "evict":
        k, v, w = s["k"].double(), s["v"].double(), s["weight"].double()
        for b, n in enumerate(lens):
            j = torch.arange(n, device="cuda")
            at = place(b, j)
            for h in range(nkv):
                mine = w[at[0], h, at[1]].tolist()
                free = [i for i in range(n) if c["sinks"] <= i < n - c["recent"]]
                free.sort(key=lambda i: (-mine[i], i))
                gone = set(free[len(free) - max(0, n - c["budget"]):])
                kept = torch.tensor([i for i in range(n) if i not in gone], device="cuda")
                to = torch.arange(len(kept), device="cuda")
                dst = s["dst"][b].long()[to // page], h, to % page
                src = at[0][kept], h, at[1][kept]
                k[dst], v[dst], w[dst] = s["k"][src].double(), s["v"][src].double(), s["weight"][src].double()
        return [k, v, w, None]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    w = s["weight"].double() if c.get("weights") else None
    row = 0
    for b, n in enumerate(lens):
        m = add[b] if add else 1
        j = torch.arange(n, device="cuda")
        pg, at = place(b, j)
        t = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = j > t
        if c["window"]:
            hidden = hidden | ((t - j >= c["window"]) & (j >= c["sinks"]))
        for h in range(nkv):
            k, v = s["k"][pg, h, at].double(), s["v"][pg, h, at].double()
            for e in range(h * grp, (h + 1) * grp):
                x = s["q"][row:row + m, e].double() @ k.T / math.sqrt(hd)
                x[hidden] = -math.inf
                p = torch.softmax(x, 1)
                out[row:row + m, e] = p @ v
                if w is not None:
                    w[pg, h, at] += p[0]
        row += m
    return out if c["op"] == "prefill" else [out, w]
