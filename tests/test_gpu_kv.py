"""The paged K/V cache on the device (pb_kv_append, pb_kv_decode,
pb_kv_prefill, pb_kv_evict) against the 64-bit oracle of kv_oracle.py.

Tolerances, from the arithmetic (u = eps / 2 of a type, the half step):
append: a mean of D squares, a root, and a rotation of two products in fp32:
(D / 2 + 16) 2^-24 (|a| + |b|) of the pair's values, then one rounding, u of
the result (and half the smallest fp16 step, 2^-25). V is one rounding: exact.
Attention: a probability is off by its fp32 score's error (`slack` of the
oracle, which becomes twice that relative to the sum), ex2's 2^-22, n 2^-24
for the sum of n terms, and its own rounding to the cache's type for the
matrix product, u (or 2^-25 of the largest, for an fp16 subnormal); the
output's rounding adds u of the result. Weights are fp32: no u."""
import numpy as np
import pytest

import kv_oracle as KO

pytestmark = pytest.mark.gpu


def U(torch, dt):
    return torch.finfo(dt).eps / 2


def f64(t):
    return t.detach().cpu().double().numpy()


class Cache:
    """pools of n_pages pages full of NaN, in one of three memory orders, and a table of random pages"""

    def __init__(self, pb, torch, lens, nkv, D, ps, dt, layout="head", weights=False, seed=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // ps) for n in lens]
        n_pages = sum(need) + spare
        nan = float("nan")
        if layout == "head":
            k, v = (torch.full((n_pages, nkv, ps, D), nan, dtype=dt, device="cuda") for _ in "kv")
        elif layout == "row":      # [page][row][head][dim]
            k, v = (torch.full((n_pages, ps, nkv, D), nan, dtype=dt, device="cuda").transpose(1, 2) for _ in "kv")
        else:                      # K and V interleaved, rows padded
            kv = torch.full((n_pages, 2, nkv, ps, D + 8), nan, dtype=dt, device="cuda")
            k, v = kv[:, 0, :, :, :D], kv[:, 1, :, :, :D]
        w = torch.rand((n_pages, nkv, ps), generator=g).cuda() if weights else None
        self.h = pb.KVPages(k, v, w)
        self.k, self.v, self.w, self.ps, self.nkv, self.D, self.dt = k, v, w, ps, nkv, D, dt
        ids = torch.randperm(n_pages, generator=g).int()
        self.table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.lens, self.g, self.torch, self.n_pages = list(lens), g, torch, n_pages
        self.fill()

    def fill(self):
        torch = self.torch
        for b, n in enumerate(self.lens):
            if n:
                pg, r, ok = KO.rows_of(self.table.numpy(), b, n, self.ps, self.n_pages)
                pg, r = torch.from_numpy(pg).long().cuda(), torch.from_numpy(r).cuda()
                for t in (self.k, self.v):
                    t[pg, :, r] = torch.randn((n, self.nkv, self.D), generator=self.g).to(self.dt).cuda()

    def dev(self):
        return self.table.cuda()


def check(torch, got, want, spread, slack, tiny, n, dt, out, what, u=None):
    p_err = 2 * slack[..., None] + 2.0 ** -21 + n * 2.0 ** -24 + (U(torch, dt) if u is None else u)
    tol = spread * p_err + 2.0 ** -25 * tiny + U(torch, out) * (np.abs(want) + spread * p_err) + 2.0 ** -25
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], tol[bad][:5])


def oracle_rows(c, q, lens, counts, scale, window, sinks):
    """(out, spread, slack, tiny) of every row, and the weights' sums per sequence"""
    k, v, qq, tb = f64(c.k), f64(c.v), f64(q), c.table.numpy()
    res, sums, r = [], [], 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        n = max(0, min(n, c.table.shape[1] * c.ps))
        for i in range(m):
            x = KO.attend(qq[r], k, v, None, tb, b, n - m + i, n, scale, window, sinks)
            res.append(x[:4])
            sums.append(x[4])
            r += 1
    if not res:
        return None, sums
    return [np.stack(x) for x in zip(*res)], sums


# ------------------------------------------------------------------ append
APPEND = [  # nh, nkv, D, ps, cache, x, half, layout, weights, pos, norms, n
    (32, 8, 64, 16, "float16", "bfloat16", 32, "head", True, False, True, 1),
    (16, 4, 128, 32, "float16", "float32", 32, "row", True, True, True, 9),
    (4, 4, 128, 64, "bfloat16", "float16", 64, "mixed", False, True, True, 33),
    (5, 1, 64, 256, "bfloat16", "bfloat16", 5, "head", True, True, True, 70),
    (12, 2, 64, 128, "float16", "float32", 0, "row", False, False, True, 6),
    (7, 1, 128, 16, "float16", "float16", 64, "head", False, False, False, 17),
    (32, 8, 128, 16, "bfloat16", "bfloat16", 64, "head", False, False, True, 2500),
]


@pytest.mark.parametrize("nh,nkv,D,ps,dt,xt,half,layout,weights,pos,norms,n", APPEND)
def test_append(pb, cuda, nh, nkv, D, ps, dt, xt, half, layout, weights, pos, norms, n):
    torch = cuda
    dt, xt = getattr(torch, dt), getattr(torch, xt)
    rng = np.random.default_rng(n)
    S = min(n, 4)
    ctx = [3 + 29 * b for b in range(S)]
    per = [n // S + (b < n % S) for b in range(S)]
    c = Cache(pb, torch, [a + m for a, m in zip(ctx, per)], nkv, D, ps, dt, layout, weights, seed=n)
    seq = np.concatenate([np.full(m, b) for b, m in enumerate(per)]).astype(np.int32)
    slot = np.concatenate([np.arange(a, a + m) for a, m in zip(ctx, per)]).astype(np.int32)
    order = rng.permutation(n)
    seq, slot = seq[order], slot[order]
    n_rope = int(slot.max()) + 40
    p = (slot + rng.integers(0, 40, n)).astype(np.int32) if pos else None
    if n > 8:      # padding of every kind
        seq[1], slot[2], seq[3], slot[4] = -1, -5, S, c.table.shape[1] * ps
        if p is not None and half:
            p[5] = n_rope
        j = 6      # a row whose page is not one
        c.table[seq[j], slot[j] // ps] = -1 if n % 2 else c.n_pages
    wide = (nh + 2 * nkv) * D
    big = torch.full((n, wide + 24), float("nan"), dtype=xt)
    big[:, :wide] = torch.from_numpy(rng.standard_normal((n, wide)) * 2).to(xt)
    q = torch.full((n, nh, D), 7.0, dtype=dt, device="cuda")
    ang = np.arange(n_rope)[:, None] * 1e4 ** (-np.arange(max(half, 1)) / max(half, 1))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (rng.standard_normal((2, D)) * 0.1 + 1).astype(np.float32) if norms else (None, None)
    K, V, Q = f64(c.k), f64(c.v), f64(q)
    W = f64(c.w) if weights else None
    KO.append(K, V, W, c.table.numpy(), seq, slot, p, f64(big), nh, qn, kn, 1e-5, cos if half else None, sin, Q)
    # the size of a value's rotation pair, for the tolerance
    mq, mk = f64(q) * 0, np.zeros_like(K)
    for nw in (0,):
        one, zero = np.ones_like(cos), np.zeros_like(cos)
        KO.append(mk, np.zeros_like(V), None, c.table.numpy(), seq, slot, p, np.nan_to_num(f64(big)), nh, qn, kn, 1e-5,
                  one if half else None, zero, mq)
    d = lambda a: None if a is None else torch.from_numpy(a).cuda()
    c.h.append(c.dev(), d(seq), d(slot), d(p), big.cuda(), q, q_norm=d(qn), k_norm=d(kn), eps=1e-5,
               cos=d(cos) if half else None, sin=d(sin) if half else None)
    torch.cuda.synchronize()

    def close(got, want, mag, what):
        pair = np.abs(mag) + np.roll(np.abs(mag), D // 2, -1)
        tol = (D / 2 + 16) * 2.0 ** -24 * pair
        tol = tol + U(torch, dt) * (np.abs(want) + tol) + 2.0 ** -25
        same = np.isnan(got) & np.isnan(want)
        bad = ~(same | (np.abs(got - want) <= tol))
        assert not bad.any(), (what, np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5])

    close(f64(q), Q, mq, "q")
    close(f64(c.k), K, mk, "k")
    vr = f64(torch.from_numpy(V).to(dt))
    assert np.array_equal(f64(c.v), vr, equal_nan=True), "v"
    if weights:
        assert np.array_equal(f64(c.w), W), "weights"


@pytest.mark.parametrize("xt", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("nh,D,extra,skip", [(12, 64, 12, 0), (6, 64, 6, 0), (7, 128, 7, 0), (4, 128, 8, 1), (4, 64, 16, 4)])
def test_append_rows_at_any_element(pb, cuda, nh, D, extra, skip, xt):
    """rows with a value per head behind v, or from within a wider tensor, are not on 16 bytes: the same bits as from a
    copy that is"""
    torch = cuda
    xt, nkv, n = getattr(torch, xt), nh if nh == 7 else 2, 37
    wide = (nh + 2 * nkv) * D
    g = torch.Generator().manual_seed(nh + extra)
    big = (torch.randn((n, wide + extra + skip), generator=g) * 2).to(xt).cuda()
    x = big[:, skip:]
    ang = torch.arange(64).double()[:, None] * 1e4 ** (-torch.arange(D // 2).double() / (D // 2))
    cos, sin = ang.cos().float().cuda(), ang.sin().float().cuda()
    norm = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got = []
    for rows in (x[:, :wide].clone().contiguous(), x):
        c = Cache(pb, torch, [64], nkv, D, 16, torch.float16, seed=1)
        q = torch.zeros((n, nh, D), dtype=torch.float16, device="cuda")
        c.h.append(c.dev(), i([0] * n), i(list(range(5, 5 + n))), None, rows, q, q_norm=norm, k_norm=norm, cos=cos, sin=sin)
        torch.cuda.synchronize()
        got.append((q, c.k, c.v))
    assert got[0][0].abs().max() > 1
    for a, b in zip(*got):
        assert np.array_equal(f64(a), f64(b), equal_nan=True)


def test_append_refuses_what_the_pointers_do_not_show(pb, cuda):
    torch = cuda
    c = Cache(pb, torch, [40], 2, 64, 16, torch.float16)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    x, q = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    t = c.dev()
    for bad in (dict(q=q.bfloat16()), dict(qkv=x[:, :-64]), dict(qkv=x.double()), dict(qkv=x.cpu()), dict(seq=i(0).long()),
                dict(seq=i(0, 0)), dict(slot=i(0).cpu()), dict(table=t.long()), dict(table=t[:, ::2]), dict(cos=torch.zeros(9, 8).cuda()),
                dict(q_norm=torch.ones(32).cuda()), dict(q=torch.zeros(1, 4, 128, dtype=torch.float16).cuda()[:, :, ::2])):
        a = dict(table=t, seq=i(0), slot=i(39), pos=None, qkv=x, q=q)
        a.update(bad)
        with pytest.raises(pb.PBError):
            c.h.append(**a)
    with pytest.raises(pb.PBError):
        pb.KVPages(c.k, c.v[:2])
    with pytest.raises(pb.PBError):
        pb.KVPages(c.k.float(), c.v.float())
    with pytest.raises(pb.PBError):
        pb.KVPages(c.k, c.v, torch.zeros(3, device="cuda"))


# ------------------------------------------------------------------ decode
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 130, 255, 257, 500, 777, 1031]
DECODE = [  # nh, nkv, D, ps, cache, out, layout, window, sinks, lens
    (32, 8, 64, 16, "float16", "bfloat16", "head", 0, 0, LENS),
    (8, 2, 128, 32, "bfloat16", "bfloat16", "row", 0, 0, LENS),
    (4, 4, 128, 64, "float16", "float16", "mixed", 0, 0, LENS),
    (16, 1, 64, 128, "bfloat16", "float16", "head", 0, 0, LENS),
    (15, 3, 128, 256, "float16", "bfloat16", "row", 0, 0, LENS),
    (7, 1, 64, 16, "float16", "float16", "mixed", 0, 0, [1031]),
    (12, 2, 128, 16, "float16", "float16", "head", 0, 0, [40] * 130),
    (16, 4, 128, 32, "float16", "bfloat16", "head", 100, 4, LENS),
    (9, 1, 64, 16, "bfloat16", "bfloat16", "head", 33, 70, LENS),
    (2, 2, 64, 64, "float16", "float16", "row", 1, 0, LENS),
    (2, 2, 128, 64, "float16", "float16", "row", 2000, 3, LENS),
    (8, 8, 128, 128, "float16", "float16", "head", 256, 130, LENS),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("nh,nkv,D,ps,dt,ot,layout,window,sinks,lens", DECODE)
def test_decode(pb, cuda, nh, nkv, D, ps, dt, ot, layout, window, sinks, lens, weights):
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    c = Cache(pb, torch, lens, nkv, D, ps, dt, layout, weights, seed=nh + D)
    if window:      # rows behind the window are gone: their pages freed, the rest of them NaN
        for b, n in enumerate(lens):
            pg, r, _ = KO.rows_of(c.table.numpy(), b, n, ps, c.n_pages)
            hid = np.nonzero(~KO.seen(n - 1, n, window, sinks))[0]
            for t in (c.k, c.v):
                t[torch.from_numpy(pg[hid]).long().cuda(), :, torch.from_numpy(r[hid]).cuda()] = float("nan")
            for p in range(-(-n // ps)):
                if not KO.seen(n - 1, n, window, sinks)[p * ps:(p + 1) * ps].any():
                    c.table[b, p] = -1
    S = len(lens)
    big = torch.randn((S, nh + 1, D), generator=c.g).to(dt).cuda()
    q = big[:, :nh]
    out = torch.full((S + 2, nh, D), 9.0, dtype=ot, device="cuda")
    w0 = f64(c.w) if weights else None
    scale = 0.7 * D ** -0.5
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.decode(c.dev(), length, q, out[:S], scale=scale, window=window, sinks=sinks, accumulate=weights)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), sums = oracle_rows(c, q, lens, [1] * S, scale, window, sinks)
    check(torch, f64(out)[:S], o, spread, slack, tiny, max(lens), dt, ot, "out")
    assert (out[S:] == 9.0).all()
    if weights:
        w = w0.copy()
        err = np.zeros_like(w)
        for b, n in enumerate(lens):
            pg, r, ok = KO.rows_of(c.table.numpy(), b, n, ps, c.n_pages)
            for h in range(nkv):
                grp = slice(h * (nh // nkv), (h + 1) * (nh // nkv))
                w[pg[ok], h, r[ok]] += sums[b][h][ok]
                err[pg[ok], h, r[ok]] = sums[b][h][ok] * (2 * slack[b][grp].max() + 2.0 ** -21 + (n + 32) * 2.0 ** -24)
        got = f64(c.w)
        bad = ~(np.abs(got - w) <= err + 2.0 ** -22 * np.abs(w))
        assert not bad.any(), (np.argwhere(bad)[:4].tolist(), got[bad][:4], w[bad][:4])
        untouched = w == w0
        assert np.array_equal(got[untouched], w0[untouched])


def test_decode_long_cache_split(pb, cuda):
    """one sequence over every SM, a few around it, the longest row near the type's largest values"""
    torch = cuda
    lens = [20011, 1, 3000, 0, 9000]
    c = Cache(pb, torch, lens, 2, 128, 64, torch.float16, seed=5)
    q = (torch.randn((5, 8, 128), generator=c.g) * 3).half().cuda()
    out = torch.empty((5, 8, 128), dtype=torch.float16, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.decode(c.dev(), length, q, out)
    torch.cuda.synchronize()
    first = out.clone()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, [1] * 5, 128 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, max(lens), c.dt, torch.float16, "long")
    for _ in range(3):
        out.fill_(3.0)
        c.h.decode(c.dev(), length, q, out)
        assert torch.equal(out, first)      # the same bits every time


def test_decode_bad_lengths_pages_and_bounds(pb, cuda):
    """lengths past max_len or the table count as the bound, negative ones as 0; bad pages hide their rows; a sequence
    that sees nothing gets zeros"""
    torch = cuda
    lens = [100, 100, 100, 100, 100]
    c = Cache(pb, torch, lens, 2, 64, 16, torch.bfloat16, weights=True, seed=9)
    c.table[1, 2], c.table[1, 5], c.table[2, :] = -7, c.n_pages, -1
    q = torch.randn((5, 8, 64), generator=c.g).bfloat16().cuda()
    out = torch.empty((5, 8, 64), dtype=torch.bfloat16, device="cuda")
    said = torch.tensor([100, 100, 100, -4, 2**31 - 1], dtype=torch.int32, device="cuda")
    c.table[4, 4:] = -1          # its rows end at 64
    w0 = f64(c.w)
    c.h.decode(c.dev(), said, q, out, max_len=80, accumulate=True)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, [80, 80, 80, 0, 80], [1] * 5, 64 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, 80, c.dt, torch.bfloat16, "bounds")
    assert (out[2] == 0).all() and (out[3] == 0).all()
    used = [int(p) for b in (0, 1, 4) for p in c.table[b, :5] if 0 <= p < c.n_pages]
    rest = [p for p in range(c.n_pages) if p not in used]
    assert np.array_equal(f64(c.w)[rest], w0[rest])


def test_decode_extreme_values(pb, cuda):
    """scores of +-thousands (one row takes all the weight), an infinite key, a NaN where it is seen"""
    torch = cuda
    lens = [300, 300, 300, 300]
    c = Cache(pb, torch, lens, 1, 128, 32, torch.float16, seed=4)
    q = torch.randn((4, 4, 128), generator=c.g).half().cuda()
    q[0] *= 500
    pg, r, _ = KO.rows_of(c.table.numpy(), 1, 300, 32, c.n_pages)
    c.k[int(pg[77]), 0, int(r[77]), 3] = -float("inf")
    q[1, :, 3] = 1.0                       # every head: score -inf there
    pg2, r2, _ = KO.rows_of(c.table.numpy(), 2, 300, 32, c.n_pages)
    c.v[int(pg2[10]), 0, int(r2[10]), 5] = float("nan")
    out = torch.empty((4, 4, 128), dtype=torch.float16, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.decode(c.dev(), length, q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, [1] * 4, 128 ** -0.5, 0, 0)
    got = f64(out)
    slack = np.minimum(slack, 1.0)
    assert np.isfinite(got[0]).all() and np.isfinite(got[1]).all()
    check(torch, got[[0, 3]], o[[0, 3]], spread[[0, 3]], slack[[0, 3]], tiny[[0, 3]], 300, c.dt, torch.float16, "large scores")
    clean = slack[3:4].repeat(1, 0)        # row 1's own slack is infinite with its key
    check(torch, got[1:2], o[1:2], spread[1:2], clean, tiny[1:2], 300, c.dt, torch.float16, "minus infinity")
    assert np.isnan(got[2, :, 5]).all() and np.isfinite(np.delete(got[2], 5, -1)).all()


# ----------------------------------------------------------------- prefill
PREFILL = [  # nh, nkv, D, ps, cache, out, layout, window, sinks, (rows in the cache, rows of the chunk)
    (8, 2, 64, 16, "float16", "bfloat16", "head", 0, 0, [(32, 32), (1, 1), (77, 77), (200, 65), (131, 1)]),
    (8, 2, 128, 32, "bfloat16", "bfloat16", "row", 0, 0, [(130, 130), (129, 2), (300, 33), (64, 64)]),
    (4, 4, 128, 64, "float16", "float16", "mixed", 0, 0, [(257, 257), (500, 128)]),
    (3, 1, 64, 128, "float16", "float16", "head", 0, 0, [(150, 150), (99, 98), (5, 5)]),
    (5, 1, 128, 16, "float16", "bfloat16", "head", 0, 0, [(90, 60), (31, 31)]),
    (16, 1, 128, 256, "bfloat16", "float16", "head", 0, 0, [(300, 41), (20, 20)]),
    (7, 1, 64, 64, "bfloat16", "bfloat16", "row", 0, 0, [(400, 100)]),
    (8, 2, 64, 16, "float16", "float16", "head", 16, 4, [(200, 200), (33, 33), (400, 17)]),
    (8, 2, 128, 32, "bfloat16", "bfloat16", "head", 100, 0, [(350, 350), (101, 1)]),
    (4, 1, 128, 64, "float16", "bfloat16", "mixed", 140, 70, [(500, 300), (64, 64)]),
    (2, 2, 64, 128, "float16", "float16", "head", 1, 0, [(260, 260)]),
    (2, 1, 128, 16, "float16", "float16", "head", 5000, 5, [(260, 130)]),
    (8, 1, 64, 16, "float16", "bfloat16", "head", 24, 200, [(700, 300)]),
]


@pytest.mark.parametrize("nh,nkv,D,ps,dt,ot,layout,window,sinks,seqs", PREFILL)
def test_prefill(pb, cuda, nh, nkv, D, ps, dt, ot, layout, window, sinks, seqs):
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    seqs = seqs[:1] + [(9, 0)] + seqs[1:]      # one sequence has no rows in the batch
    lens, counts = [a for a, _ in seqs], [m for _, m in seqs]
    c = Cache(pb, torch, lens, nkv, D, ps, dt, layout, seed=nh + D + window)
    if window:      # what no query of a chunk sees is NaN, whole pages of it freed
        for b, (n, m) in enumerate(seqs):
            any_ = np.zeros(n, bool)
            for t in range(n - m, n):
                any_ |= KO.seen(t, n, window, sinks)
            pg, r, _ = KO.rows_of(c.table.numpy(), b, n, ps, c.n_pages)
            hid = np.nonzero(~any_)[0]
            for t in (c.k, c.v):
                t[torch.from_numpy(pg[hid]).long().cuda(), :, torch.from_numpy(r[hid]).cuda()] = float("nan")
            for p in range(-(-n // ps)):
                if not any_[p * ps:(p + 1) * ps].any():
                    c.table[b, p] = -1
    pad = 3                                    # rows before the first and behind the last sequence
    rows = sum(counts)
    q = torch.randn((rows + 2 * pad, nh, D), generator=c.g).to(dt).cuda()
    out = torch.full((rows + 2 * pad, nh + 2, D), 9.0, dtype=ot, device="cuda")
    start = torch.tensor(np.concatenate([[0], np.cumsum(counts)]) + pad, dtype=torch.int32, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = 1.3 * D ** -0.5
    c.h.prefill(c.dev(), start, length, q, out[:, :nh], scale=scale, window=window, sinks=sinks)
    torch.cuda.synchronize()
    c.h.status()
    (o, spread, slack, tiny), _ = oracle_rows(c, q[pad:pad + rows], lens, counts, scale, window, sinks)
    check(torch, f64(out)[pad:pad + rows, :nh], o, spread, slack, tiny, max(lens), dt, ot, "out")
    assert (out[:pad] == 9.0).all() and (out[pad + rows:] == 9.0).all() and (out[:, nh:] == 9.0).all()


def test_prefill_small_chunk_long_cache(pb, cuda):
    """few rows against a long cache: the cache is split over the SMs, the same bits every time"""
    torch = cuda
    lens, counts = [9001, 16, 4100], [33, 16, 7]
    c = Cache(pb, torch, lens, 2, 64, 16, torch.float16, seed=3)
    q = torch.randn((56, 8, 64), generator=c.g).half().cuda()
    out = torch.empty((56, 8, 64), dtype=torch.float16, device="cuda")
    start = torch.tensor([0, 33, 49, 56], dtype=torch.int32, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), start, length, q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, counts, 64 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, max(lens), c.dt, torch.float16, "chunk")
    first = out.clone()
    for _ in range(3):
        out.fill_(1.0)
        c.h.prefill(c.dev(), start, length, q, out)
        assert torch.equal(out, first)


def test_prefill_bad_pages_and_lengths(pb, cuda):
    """bad pages hide their rows; a chunk longer than its cache: the rows before the cache's first see nothing"""
    torch = cuda
    c = Cache(pb, torch, [100, 100, 100], 1, 128, 16, torch.float16, seed=6)
    c.table[0, 1], c.table[0, 3], c.table[1, :] = -1, 10 ** 9, c.n_pages
    q = torch.randn((60, 4, 128), generator=c.g).half().cuda()
    out = torch.full((60, 4, 128), 5.0, dtype=torch.float16, device="cuda")
    start = torch.tensor([0, 30, 40, 60], dtype=torch.int32, device="cuda")
    said = torch.tensor([100, 100, 12], dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), start, said, q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, [100, 100, 12], [30, 10, 20], 128 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, 100, c.dt, torch.float16, "bad pages")
    assert (out[30:40] == 0).all() and (out[40:48] == 0).all()


def test_prefill_extreme_scores(pb, cuda):
    torch = cuda
    c = Cache(pb, torch, [400], 2, 128, 32, torch.bfloat16, seed=8)
    q = (torch.randn((400, 8, 128), generator=c.g) * 200).bfloat16().cuda()
    out = torch.empty((400, 8, 128), dtype=torch.bfloat16, device="cuda")
    start = torch.tensor([0, 400], dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), start, torch.tensor([400], dtype=torch.int32, device="cuda"), q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, [400], [400], 128 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, np.minimum(slack, 1.0), tiny, 400, c.dt, torch.bfloat16, "large scores")


@pytest.mark.parametrize("nh,nkv,D", [(8, 2, 64), (16, 1, 128), (4, 4, 128)])
def test_fp16_output_of_a_bf16_cache(pb, cuda, nh, nkv, D):
    """an output with more bits than the cache's type: the probabilities keep two numbers of that type, each a half
    step of 2^-8 (2^-16 together), so that the output's own rounding is the largest error"""
    torch = cuda
    lens, counts = [2, 3, 17, 200, 70, 2600], [2, 3, 5, 130, 1, 40]
    c = Cache(pb, torch, lens, nkv, D, 32, torch.bfloat16, seed=D + nh)
    S = len(lens)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for m in ([1] * S, counts):
        q = (torch.randn((sum(m), nh, D), generator=c.g) * 0.5).bfloat16().cuda()
        out = torch.empty((sum(m), nh, D), dtype=torch.float16, device="cuda")
        if m is counts:
            start = torch.tensor(np.concatenate([[0], np.cumsum(m)]), dtype=torch.int32, device="cuda")
            c.h.prefill(c.dev(), start, length, q, out)
            c.h.status()
        else:
            c.h.decode(c.dev(), length, q, out)
        torch.cuda.synchronize()
        (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, m, D ** -0.5, 0, 0)
        check(torch, f64(out), o, spread, slack, tiny * 0, max(lens), c.dt, torch.float16, "%d rows" % sum(m), u=2.0 ** -16)


# ------------------------------------------------------------------- evict
EVICT = [  # nkv, D, ps, dtype, layout, lens, budget, sinks, recent, weights
    (4, 128, 16, "bfloat16", "head", [300, 200, 201, 0, 1, 77], 200, 4, 50, "random"),
    (2, 64, 32, "float16", "row", [500, 499, 130], 128, 0, 0, "random"),
    (1, 64, 64, "float16", "mixed", [1000], 700, 1, 699, "random"),
    (3, 128, 16, "float16", "head", [400, 333], 160, 2, 30, "ties"),
    (2, 64, 16, "bfloat16", "head", [400, 333], 160, 0, 16, "zeros"),
    (2, 64, 16, "float16", "head", [400, 333], 160, 3, 16, "odd"),
    (1, 64, 256, "float16", "head", [700], 256, 256, 0, "random"),
    (1, 64, 128, "float16", "head", [12000], 1025, 5, 100, "random"),
    (8, 64, 16, "float16", "head", [40, 30], 50, 5, 10, "random"),
]


@pytest.mark.parametrize("nkv,D,ps,dt,layout,lens,budget,sinks,recent,kind", EVICT)
def test_evict(pb, cuda, nkv, D, ps, dt, layout, lens, budget, sinks, recent, kind):
    torch = cuda
    S = len(lens)
    kept = [min(n, budget) for n in lens]
    c = Cache(pb, torch, lens + kept, nkv, D, ps, getattr(torch, dt), layout, True, seed=budget)
    table, dst = c.table[:S].contiguous(), c.table[S:].contiguous()
    rng = np.random.default_rng(budget)
    w = torch.from_numpy(rng.random(tuple(c.w.shape)).astype(np.float32) ** 6 * 30)
    if kind == "ties":
        w = (w * 0.2).round()
    elif kind == "zeros":
        w = w * 0
    elif kind == "odd":
        w.view(-1)[::7] = float("nan")
        w.view(-1)[1::11] = -1.0
        w.view(-1)[2::13] = float("inf")
        w.view(-1)[3::5] = 1e-42
    c.w.copy_(w.cuda())
    K, V, W = f64(c.k), f64(c.v), f64(c.w)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    c.h.evict(table.cuda(), length, dst.cuda(), new, budget, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    assert new.tolist() == kept
    K2, V2, W2 = K.copy(), V.copy(), W.copy()
    for b, n in enumerate(lens):
        pg, r, _ = KO.rows_of(table.numpy(), b, n, ps, c.n_pages)
        to, tr, _ = KO.rows_of(dst.numpy(), b, kept[b], ps, c.n_pages)
        for h in range(nkv):
            at = KO.evict_rows(W[pg, h, r], n, budget, sinks, recent)
            assert len(at) == kept[b]
            K2[to, h, tr], V2[to, h, tr], W2[to, h, tr] = K[pg[at], h, r[at]], V[pg[at], h, r[at]], W[pg[at], h, r[at]]
    for got, want, what in ((c.k, K2, "k"), (c.v, V2, "v"), (c.w, W2, "weights")):
        assert np.array_equal(f64(got), want, equal_nan=True), what


def test_evict_lengths_in_place_and_bad_pages(pb, cuda):
    torch = cuda
    c = Cache(pb, torch, [300, 300, 150, 150], 2, 64, 16, torch.float16, "head", True, seed=2)
    table, dst = c.table[:2].contiguous(), c.table[2:].contiguous()
    table[0, 3], dst[1, 1] = -1, c.n_pages
    W, K = f64(c.w), f64(c.k)
    length = torch.tensor([300, 2**31 - 1], dtype=torch.int32, device="cuda")
    c.h.evict(table.cuda(), length, dst.cuda(), length, 150, sinks=0, recent=10, max_len=299)
    torch.cuda.synchronize()
    assert length.tolist() == [150, 150]
    for b in range(2):
        pg, r, ok = KO.rows_of(table.numpy(), b, 299, 16, c.n_pages)
        to, tr, dok = KO.rows_of(dst.numpy(), b, 150, 16, c.n_pages)
        for h in range(2):
            at = np.asarray(KO.evict_rows(np.where(ok, W[np.where(ok, pg, 0), h, r], 0), 299, 150, 0, 10))
            m = ok[at] & dok
            assert np.array_equal(f64(c.k)[to[m], h, tr[m]], K[pg[at[m]], h, r[at[m]]])
            assert np.array_equal(f64(c.w)[to[m], h, tr[m]], W[pg[at[m]], h, r[at[m]]])


def test_evict_lengths_in_place_of_more_rows_than_run_at_once(pb, cuda):
    """the lengths are replaced while CTAs that read them have not started: 64
    K/V heads of 4096 kept rows; and a sequence within the budget beside it"""
    torch = cuda
    lens, budget, nkv, D, ps = [4200, 100], 4096, 64, 128, 64
    kept = [4096, 100]
    c = Cache(pb, torch, lens + kept, nkv, D, ps, torch.float16, "head", True, seed=9)
    table, dst = c.table[:2].contiguous(), c.table[2:].contiguous()
    W = c.w.cpu().numpy()
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = []
    for b, n in enumerate(lens):
        pg, r, _ = KO.rows_of(table.numpy(), b, n, ps, c.n_pages)
        for h in range(nkv):
            at = np.asarray(KO.evict_rows(W[pg, h, r].astype(np.float64), n, budget, 0, 8))
            pa, ra = (torch.from_numpy(np.ascontiguousarray(x)).cuda().long() for x in (pg[at], r[at]))
            want.append((c.k[pa, h, ra], c.v[pa, h, ra], c.w[pa, h, ra]))
    c.h.evict(table.cuda(), length, dst.cuda(), length, budget, sinks=0, recent=8)
    torch.cuda.synchronize()
    assert length.tolist() == kept
    for b, n in enumerate(kept):
        to, tr, _ = KO.rows_of(dst.numpy(), b, n, ps, c.n_pages)
        to, tr = torch.from_numpy(np.ascontiguousarray(to)).cuda().long(), torch.from_numpy(np.ascontiguousarray(tr)).cuda().long()
        for h in range(nkv):
            k, v, w = want[b * nkv + h]
            assert torch.equal(c.k[to, h, tr], k) and torch.equal(c.v[to, h, tr], v) and torch.equal(c.w[to, h, tr], w), (b, h)


# ---------------------------------------------------------------- together
def test_prompt_decode_evict_decode(pb, cuda):
    """as a server uses them: prompts appended and attended in chunks, decode steps that add weights, eviction to fresh
    pages, more steps (slots behind the kept rows, positions going on), each result against the oracle on the cache as
    it then is; replayed from a captured graph on another stream for the last steps"""
    torch = cuda
    nh, nkv, D, ps, dt = 8, 2, 64, 16, torch.float16
    S, budget = 3, 64
    prompt = [70, 33, 90]
    c = Cache(pb, torch, [160] * S + [96] * S, nkv, D, ps, dt, "head", True, seed=12)
    for t in (c.k, c.v):
        t.fill_(float("nan"))
    table, fresh = c.table[:S].contiguous(), c.table[S:].contiguous()
    rng = np.random.default_rng(3)
    wide = (nh + 2 * nkv) * D
    ang = np.arange(200)[:, None] * 1e4 ** (-np.arange(D // 2) / (D // 2))
    cos, sin = torch.from_numpy(np.cos(ang)).float().cuda(), torch.from_numpy(np.sin(ang)).float().cuda()
    qn, kn = torch.ones(D).cuda() * 1.1, torch.ones(D).cuda() * 0.9
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    done = [0] * S
    while any(d < p for d, p in zip(done, prompt)):
        m = [min(32, p - d) for d, p in zip(done, prompt)]
        seq = i32(sum([[b] * m[b] for b in range(S)], []))
        slot = i32(sum([list(range(done[b], done[b] + m[b])) for b in range(S)], []))
        n = sum(m)
        x = torch.from_numpy(rng.standard_normal((n, wide))).bfloat16().cuda()
        q, out = torch.empty((n, nh, D), dtype=dt, device="cuda"), torch.empty((n, nh, D), dtype=torch.bfloat16, device="cuda")
        c.h.append(table.cuda(), seq, slot, None, x, q, q_norm=qn, k_norm=kn, cos=cos, sin=sin)
        done = [d + a for d, a in zip(done, m)]
        c.h.prefill(table.cuda(), i32(np.concatenate([[0], np.cumsum(m)]).tolist()), i32(done), q, out, window=48, sinks=2)
        torch.cuda.synchronize()
        c.table = table
        (o, spread, slack, tiny), _ = oracle_rows(c, q, done, m, D ** -0.5, 48, 2)
        check(torch, f64(out), o, spread, slack, tiny, 200, dt, torch.bfloat16, "prompt")

    x = torch.empty((S, wide), dtype=torch.float32, device="cuda")
    q, out = torch.empty((S, nh, D), dtype=dt, device="cuda"), torch.empty((S, nh, D), dtype=torch.bfloat16, device="cuda")
    seq, slot, pos, length = i32(list(range(S))), i32(done), i32(done), i32(done)
    scratch = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    tb = table.cuda()

    def step(tb, stream=None):
        c.h.append(tb, seq, slot, pos, x, q, q_norm=qn, k_norm=kn, cos=cos, sin=sin, stream=stream)
        c.h.decode(tb, length, q, out, accumulate=True, scratch=scratch, stream=stream)

    def verify(lens, what):
        (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, [1] * S, D ** -0.5, 0, 0)
        check(torch, f64(out), o, spread, slack, tiny, 200, dt, torch.bfloat16, what)

    lens = list(done)
    for k in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal((S, wide))).float())
        slot.copy_(i32(lens)); pos.copy_(i32(lens))
        lens = [n + 1 for n in lens]
        length.copy_(i32(lens))
        step(tb)
        torch.cuda.synchronize()
        verify(lens, "step %d" % k)
    position = list(lens)
    c.h.evict(tb, length, fresh.cuda(), length, budget, sinks=2, recent=16)
    torch.cuda.synchronize()
    lens = [min(n, budget) for n in lens]
    assert length.tolist() == lens
    c.table, tb = fresh, fresh.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    with torch.cuda.stream(side):
        slot.copy_(i32(lens)); pos.copy_(i32(position)); length.copy_(i32([n + 1 for n in lens]))
        step(tb, side)          # once before the capture
    side.synchronize()
    for t, o in zip((c.k, c.v, c.w), before):
        t.copy_(o)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(tb, side)
    for k in range(6):
        x.copy_(torch.from_numpy(rng.standard_normal((S, wide))).float())
        slot.copy_(i32(lens)); pos.copy_(i32(position))
        lens, position = [n + 1 for n in lens], [p + 1 for p in position]
        length.copy_(i32(lens))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        verify(lens, "replayed step %d" % k)


def test_two_streams_at_once(pb, cuda):
    """the same cache read by calls on two streams, each with scratch of its own"""
    torch = cuda
    lens = [3000, 2000, 1500]
    c = Cache(pb, torch, lens, 2, 128, 32, torch.float16, seed=1)
    q = torch.randn((3, 8, 128), generator=c.g).half().cuda()
    length, tb = torch.tensor(lens, dtype=torch.int32, device="cuda"), c.dev()
    want = torch.empty_like(q)
    c.h.decode(tb, length, q, want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(q) for _ in range(20)]
    for n, o in enumerate(outs):
        c.h.decode(tb, length, q, o, stream=streams[n % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_empty_calls(pb, cuda):
    torch = cuda
    c = Cache(pb, torch, [40, 20], 2, 64, 16, torch.float16, weights=True)
    e = lambda *s, dt=torch.int32: torch.empty(s, dtype=dt, device="cuda")
    q, none = e(0, 4, 64, dt=torch.float16), e(0)
    c.h.append(c.dev(), none, none, None, e(0, 8 * 64, dt=torch.bfloat16), q)
    c.h.decode(e(0, 3), none, q, q.clone(), accumulate=True)
    c.h.prefill(e(0, 3), torch.zeros(1, dtype=torch.int32, device="cuda"), none, q, q.clone())
    c.h.prefill(c.dev(), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([40, 20], dtype=torch.int32, device="cuda"),
                q, q.clone())
    c.h.evict(e(0, 3), none, e(0, 3), none.clone(), 5)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(pb, cuda):
    """pages 2^30 elements apart: the third begins 2^32 bytes in"""
    torch = cuda
    ps, nkv, D, far = 32, 2, 64, 1 << 30
    big = torch.zeros(2 * far + (1 << 20), dtype=torch.float16, device="cuda")
    k = big.as_strided((3, nkv, ps, D), (far, ps * D, D, 1))
    v = big.as_strided((3, nkv, ps, D), (far, ps * D, D, 1), storage_offset=1 << 16)
    w = torch.rand((3, nkv, ps), device="cuda")
    h = pb.KVPages(k, v, w)
    rng = np.random.default_rng(0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = i32([2, 1], [0, -1]).view(2, 2)
    n = 50
    x = torch.from_numpy(rng.standard_normal((n, 8 * D))).half().cuda()
    q = torch.empty((n, 4, D), dtype=torch.float16, device="cuda")
    h.append(table, torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda"), None, x, q)
    torch.cuda.synchronize()
    xs = x.view(n, 8, D)
    assert torch.equal(q, xs[:, :4])
    assert torch.equal(k[2].transpose(0, 1), xs[:32, 4:6]) and torch.equal(v[1, :, :18].transpose(0, 1), xs[32:, 6:])

    class C_:
        pass
    c = C_()
    c.k, c.v, c.table, c.ps = k, v, table[:1].cpu(), ps
    out = torch.empty_like(q)
    h.prefill(table[:1].contiguous(), i32(0, n), i32(n), q, out)
    last = torch.empty((1, 4, D), dtype=torch.float16, device="cuda")
    h.decode(table[:1].contiguous(), i32(n), q[-1:], last)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, [n], [n], D ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, n, torch.float16, torch.float16, "prefill")
    check(torch, f64(last), o[-1:], spread[-1:], slack[-1:], tiny[-1:], n, torch.float16, torch.float16, "decode")
    keep = KO.evict_rows(torch.cat([w[2, 1], w[1, 1]]).cpu().numpy(), n, 20, 1, 3)
    new = i32(0)
    rows = torch.cat([k[2, 1], k[1, 1]])[torch.tensor(keep).cuda()].clone()
    h.evict(table[:1].contiguous(), i32(n), i32(0).view(1, 1), new, 20, sinks=1, recent=3)
    torch.cuda.synchronize()
    assert new.item() == 20 and torch.equal(k[0, 1, :20], rows)


def test_shared_prefix_pages(pb, cuda):
    """sequences whose tables begin with the same pages"""
    torch = cuda
    c = Cache(pb, torch, [64, 30, 45, 9], 2, 128, 16, torch.bfloat16, seed=11)
    own = c.table.clone()
    c.table = torch.full((3, 8), -1, dtype=torch.int32)
    lens = [64 + 30, 64 + 45, 64 + 9]
    for b in range(3):
        c.table[b, :4] = own[0, :4]
        m = -(-(lens[b] - 64) // 16)
        c.table[b, 4:4 + m] = own[b + 1, :m]
    counts = [30, 45, 9]
    q = torch.randn((84, 8, 128), generator=c.g).bfloat16().cuda()
    out, one = torch.empty_like(q), torch.empty((3, 8, 128), dtype=torch.bfloat16, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), torch.tensor([0, 30, 75, 84], dtype=torch.int32, device="cuda"), length, q, out)
    last = q[[29, 74, 83]].contiguous()
    c.h.decode(c.dev(), length, last, one)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, counts, 128 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, 110, c.dt, torch.bfloat16, "prefill")
    at = [29, 74, 83]
    check(torch, f64(one), o[at], spread[at], slack[at], tiny[at], 110, c.dt, torch.bfloat16, "decode")


def test_captured_prefill_and_evict(pb, cuda):
    """replays follow the starts, lengths and tables that lie on the device then; scratch in the graph's own pool"""
    torch = cuda
    lens, counts = [700, 90], [20, 12]
    c = Cache(pb, torch, lens + [64, 64], 2, 64, 16, torch.float16, "head", True, seed=21)
    table, dst = c.table[:2].contiguous(), c.table[2:].contiguous()
    c.table = table
    q = torch.randn((40, 8, 64), generator=c.g).half().cuda()
    out = torch.zeros_like(q)
    start = torch.tensor([0, 20, 32], dtype=torch.int32, device="cuda")
    length, new = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    tb, db = table.cuda(), dst.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.h.prefill(tb, start, length, q, out, window=300, sinks=3)
        c.h.evict(tb, length, db, new, 64, sinks=2, recent=8)
    for lens, counts in (([700, 90], [20, 12]), ([333, 40], [5, 33]), ([64, 17], [1, 1])):
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        start.copy_(torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32))
        out.fill_(2.0)
        W, K = f64(c.w), f64(c.k)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        rows = sum(counts)
        (o, spread, slack, tiny), _ = oracle_rows(c, q[:rows], lens, counts, 64 ** -0.5, 300, 3)
        check(torch, f64(out)[:rows], o, spread, slack, tiny, 700, c.dt, torch.float16, lens)
        assert (out[rows:] == 2.0).all() and new.tolist() == [min(n, 64) for n in lens]
        for b, n in enumerate(lens):
            pg, r, _ = KO.rows_of(table.numpy(), b, n, 16, c.n_pages)
            to, tr, _ = KO.rows_of(dst.numpy(), b, min(n, 64), 16, c.n_pages)
            for h in range(2):
                at = KO.evict_rows(W[pg, h, r], n, 64, 2, 8)
                assert np.array_equal(f64(c.k)[to, h, tr], K[pg[at], h, r[at]])


def test_prefill_of_many_sequences(pb, cuda):
    """more sequences than a CTA has threads; some without rows, one token each; the rows between them stay"""
    torch = cuda
    S = 500
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 20, S).tolist()
    counts = [int(rng.integers(0, min(4, n + 1))) for n in lens]
    c = Cache(pb, torch, lens, 1, 64, 16, torch.float16, seed=31)
    rows = sum(counts)
    q = torch.randn((rows, 2, 64), generator=c.g).half().cuda()
    out, one = torch.empty_like(q), torch.empty((S, 2, 64), dtype=torch.float16, device="cuda")
    start = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), start, length, q, out)
    q1 = torch.randn((S, 2, 64), generator=c.g).half().cuda()
    c.h.decode(c.dev(), length, q1, one)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, counts, 64 ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, 20, c.dt, torch.float16, "prefill")
    (o, spread, slack, tiny), _ = oracle_rows(c, q1, lens, [1] * S, 64 ** -0.5, 0, 0)
    check(torch, f64(one), o, spread, slack, tiny, 20, c.dt, torch.float16, "decode")


# --------------------------------------------------- rows that lie on no page
EVICT_GONE = [  # nkv, D, ps, dtype, layout, lens, pages without a name, budget, sinks, recent, weights
    (2, 128, 16, "bfloat16", "head", [300, 300, 170, 120, 90, 77, 310, 0],
     [[0, 1, 2], [5, 9, 18], [2, 4, 10], [0, 3], range(6), [], [], []], 160, 5, 20, "random"),
    (2, 64, 16, "float16", "row", [300, 300, 170, 120, 90, 77, 310, 0],
     [[0, 1, 2], [5, 9, 18], [2, 4, 10], [0, 3], range(6), [], [], []], 160, 5, 20, "zeros"),
    (1, 64, 32, "float16", "mixed", [300, 300, 170, 120, 90, 77], [[0], [4, 9], [2, 5], [0, 2], [0, 1, 2], []], 400, 3, 20, "random"),
    (3, 128, 64, "float16", "head", [9000, 8700, 700], [[0, 1, 2, 50, 139], [], [10]], 8600, 64, 100, "random"),
    (1, 64, 16, "bfloat16", "head", [5000, 4990], [[0, 260], range(0, 300, 2)], 4990, 0, 0, "random"),
    (64, 128, 64, "float16", "head", [4300, 100], [[0, 40], [0]], 4096, 0, 8, "random"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("nkv,D,ps,dt,layout,lens,gone,budget,sinks,recent,kind", EVICT_GONE)
def test_evict_leaves_rows_without_a_page_out(pb, cuda, nkv, D, ps, dt, layout, lens, gone, budget, sinks, recent, kind, in_place):
    """the fresh pages hold NaN and may be more than the kept rows need: every row of the new length is a row that was
    seen before, and nothing behind it is written"""
    torch = cuda
    S = len(lens)
    c = Cache(pb, torch, lens + [min(n, budget) for n in lens], nkv, D, ps, getattr(torch, dt), layout, True, seed=budget + D)
    table, dst = c.table[:S].contiguous(), c.table[S:].contiguous()
    for t in (c.k, c.v):
        t[torch.unique(dst[dst >= 0]).long().cuda()] = float("nan")
    for b in range(S):
        for i, p in enumerate(gone[b]):
            table[b, p] = (-1, c.n_pages, 10 ** 9)[i % 3]
    if kind == "zeros":
        c.w.zero_()
    K, V, W = c.k.clone(), c.v.clone(), c.w.clone()
    w = f64(c.w)
    kept = []
    for b, n in enumerate(lens):
        pg, r, ok = KO.rows_of(table.numpy(), b, n, ps, c.n_pages)
        for h in range(nkv):
            at = KO.evict_rows_named(w[np.where(ok, pg, 0), h, r], ok, n, budget, sinks, recent)
            to, tr, _ = KO.rows_of(dst.numpy(), b, len(at), ps, c.n_pages)
            i = [torch.from_numpy(np.ascontiguousarray(x)).long().cuda() for x in (to, tr, pg[at], r[at])]
            for t, o in ((K, c.k), (V, c.v), (W, c.w)):
                t[i[0], h, i[1]] = o[i[2], h, i[3]]
        kept.append(len(at))
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = length if in_place else torch.full((S,), -1, dtype=torch.int32, device="cuda")
    c.h.evict(table.cuda(), length, dst.cuda(), new, budget, sinks=sinks, recent=recent,
              scratch=torch.zeros(4 * S * nkv * budget, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    assert new.tolist() == kept
    bits = lambda t: t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)
    for got, want, what in ((c.k, K, "k"), (c.v, V, "v"), (c.w, W, "weights")):
        assert torch.equal(bits(got), bits(want)), what
    # the next step sees the kept rows alone
    c.table = dst
    q = torch.randn((S, 2 * nkv, D), generator=c.g).to(c.dt).cuda()
    out = torch.empty_like(q)
    c.h.decode(dst.cuda(), new, q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, kept, [1] * S, D ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny, max(kept), c.dt, c.dt, "decode behind it")


# ------------------------------------- one row far above a long, even rest
def far_below(pb, torch, n, nkv, D, dt, gap, first, noise, seed):
    """row `first` of a cache of n rows scores `gap` above the others (q = 4 in dimension 0, scale 1) and has V = 0, so
    that what the others leave is the whole output"""
    c = Cache(pb, torch, [n], nkv, D, 64, dt, seed=seed)
    pg, r, _ = KO.rows_of(c.table.numpy(), 0, n, 64, c.n_pages)
    pg, r = torch.from_numpy(pg).long().cuda(), torch.from_numpy(r).cuda()
    k = torch.zeros((n, nkv, D))
    k[:, :, 0] = torch.randn((n, nkv), generator=c.g) * noise / 4
    k[first, :, 0] = gap / 4
    v = torch.ones((n, nkv, D))
    v[:, :, 1::2] += 0.5 * torch.randn((n, nkv, D // 2), generator=c.g)
    v[first] = 0
    c.k[pg, :, r], c.v[pg, :, r] = k.to(dt).cuda(), v.to(dt).cuda()
    return c


FAR = [("float16", "float16"), ("float16", "bfloat16"), ("bfloat16", "bfloat16")]


@pytest.mark.parametrize("dt,ot", FAR)
@pytest.mark.parametrize("D,gap,first,noise", [(64, 16.0, 0, 0.0), (128, 17.5, 0, 0.0), (128, 18.0, 0, 0.3), (64, 18.0, 9000, 0.0),
                                               (128, 20.0, 3, 0.3)])
def test_decode_small_probabilities_are_kept(pb, cuda, D, gap, first, noise, dt, ot):
    """The probabilities are relative to the largest, times 2^15 in fp16: half a step of what is not normal there is
    2^-25 2^-15 of the largest, whatever the cache's length. One sequence, whose pieces have maxima of their own, and
    many that share its pages, so that a CTA goes through a whole one."""
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    n = 20011
    c = far_below(pb, torch, n, 2, D, dt, gap, first, noise, seed=D)
    for S, nh in ((1, 24), (300, 2)):
        q = torch.zeros((S, nh, D), dtype=dt, device="cuda")
        q[:, :, 0] = 4.0
        out = torch.empty((S, nh, D), dtype=ot, device="cuda")
        length = torch.full((S,), n, dtype=torch.int32, device="cuda")
        c.h.decode(c.dev().expand(S, -1).contiguous(), length, q, out, scale=1.0)
        torch.cuda.synchronize()
        (o, spread, slack, tiny), _ = oracle_rows(c, q[:1], [n], [1], 1.0, 0, 0)
        for b in {0, S // 2, S - 1}:
            check(torch, f64(out)[b:b + 1], o, spread, slack, tiny * 2.0 ** -15, n, dt, ot, (S, b))


@pytest.mark.parametrize("dt,ot", FAR)
@pytest.mark.parametrize("D,gap,first,noise,chunk", [(64, 16.0, 0, 0.0, 16), (128, 17.5, 0, 0.0, 40), (128, 18.0, 0, 0.3, 5000),
                                                     (64, 18.0, 9000, 0.0, 5000), (128, 20.0, 3, 0.3, 16)])
def test_prefill_small_probabilities_are_kept(pb, cuda, D, gap, first, noise, chunk, dt, ot):
    """as in decode, but times 2^7 at the least: the maximum that the probabilities are relative to may be 2^8 behind.
    Few rows split over the SMs, and many rows with the whole line in each CTA."""
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    n, nh = 20011, 8
    c = far_below(pb, torch, n, 2, D, dt, gap, first, noise, seed=D + 1)
    q = torch.zeros((chunk, nh, D), dtype=dt, device="cuda")
    q[:, :, 0] = 4.0
    out = torch.empty((chunk, nh, D), dtype=ot, device="cuda")
    c.h.prefill(c.dev(), torch.tensor([0, chunk], dtype=torch.int32, device="cuda"),
                torch.tensor([n], dtype=torch.int32, device="cuda"), q, out, scale=1.0)
    torch.cuda.synchronize()
    c.h.status()
    k, v, qq, got = f64(c.k), f64(c.v), f64(q), f64(out)
    for i in sorted({0, chunk // 2, chunk - 2, chunk - 1}):
        o, spread, slack, tiny, _ = KO.attend(qq[i], k, v, None, c.table.numpy(), 0, n - chunk + i, n, 1.0, 0, 0)
        check(torch, got[i:i + 1], o[None], spread[None], slack[None], tiny[None] * 2.0 ** -7, n, dt, ot, i)


# ------------------------------------------------ rows that belong to no head
@pytest.mark.parametrize("nh,nkv,D,dt", [(12, 2, 64, "float16"), (18, 2, 64, "bfloat16"), (24, 2, 64, "float16")])
def test_prefill_time_does_not_depend_on_left_shared_memory(pb, cuda, nh, nkv, D, dt):
    """groups of 6, 9 and 12 heads leave 32, 56 and 32 of a CTA's 128 rows without a head. A decode over rows of NaN, or
    of zeros, fills every SM's shared memory first; the prompt behind it then took a fifth longer with NaN (medians
    differ by some 2 % between runs)."""
    torch = cuda
    dt, n = getattr(torch, dt), 3000
    fills = []
    for bits in (0, -1):
        x = torch.full((600, 8, 64, 64), bits, dtype=torch.int16, device="cuda").view(torch.float16)
        h = pb.KVPages(x, x.clone())
        a = (torch.arange(600, dtype=torch.int32, device="cuda").view(1, 600), torch.tensor([600 * 64], dtype=torch.int32, device="cuda"),
             torch.zeros((1, 32, 64), dtype=torch.float16, device="cuda"))
        fills.append((h, a + (torch.empty_like(a[2]),)))
    c = Cache(pb, torch, [n], nkv, D, 64, dt, seed=nh)
    q = torch.randn((n, nh, D), generator=c.g).to(dt).cuda()
    out, table = torch.empty_like(q), c.dev()
    start, length = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    times, first = [[], []], None
    for _ in range(25):
        for k, (h, a) in enumerate(fills):
            h.decode(*a)
            torch.cuda._sleep(200000)      # (the call's host time passes meanwhile)
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            c.h.prefill(table, start, length, q, out)
            e[1].record()
            torch.cuda.synchronize()
            times[k].append(e[0].elapsed_time(e[1]))
            first = out.clone() if first is None else first
            assert torch.equal(out, first)
    assert np.median(times[1]) < 1.1 * np.median(times[0]), [np.median(t) for t in times]


# -------------------------------------------------- lines of many key tiles
@pytest.mark.parametrize("nh,nkv,D,ps,dt,window", [(8, 2, 64, 16, "float16", 0), (8, 2, 128, 64, "bfloat16", 0),
                                                   (6, 1, 64, 32, "bfloat16", 0), (5, 1, 128, 16, "float16", 1100),
                                                   (16, 8, 64, 128, "float16", 1000)])
def test_prefill_of_some_thousand_rows(pb, cuda, nh, nkv, D, ps, dt, window):
    """prompts whose CTAs go through 25 to 50 key tiles each: every ring stage is used several times, pages are looked up
    several times; not split over the keys"""
    torch = cuda
    dt = getattr(torch, dt)
    lens, counts = [1500, 3100], [1500, 2500]
    c = Cache(pb, torch, lens, nkv, D, ps, dt, seed=nh + ps)
    rows = sum(counts)
    q = torch.randn((rows, nh, D), generator=c.g).to(dt).cuda()
    out = torch.full((rows, nh, D), 9.0, dtype=dt, device="cuda")
    start = torch.tensor([0, 1500, 4000], dtype=torch.int32, device="cuda")
    c.h.prefill(c.dev(), start, torch.tensor(lens, dtype=torch.int32, device="cuda"), q, out, window=window, sinks=5)
    torch.cuda.synchronize()
    c.h.status()
    # in 64 bits, a whole head at a time
    k, v, qq, got, r = f64(c.k), f64(c.v), f64(q), f64(out), 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        pg, rr, _ = KO.rows_of(c.table.numpy(), b, n, ps, c.n_pages)
        sees = np.stack([KO.seen(t, n, window, 5) for t in range(n - m, n)])
        for h in range(nh):
            kk, vv, x = k[pg, h // (nh // nkv), rr], v[pg, h // (nh // nkv), rr], qq[r:r + m, h]
            s = np.where(sees, x @ kk.T * D ** -0.5, -np.inf)
            e = np.exp(s - s.max(1, keepdims=True))
            p = e / e.sum(1, keepdims=True)
            slack = 2.0 ** -24 * ((D + 8) * np.where(sees, np.abs(x) @ np.abs(kk).T, 0).max(1) * D ** -0.5 + 16)
            check(torch, got[r:r + m, h], p @ vv, p @ np.abs(vv), slack, sees @ np.abs(vv) / e.sum(1, keepdims=True), n, dt, dt,
                  (b, h))
        r += m


@pytest.mark.parametrize("dt,ot,u", [("bfloat16", "bfloat16", 2.0 ** -16), ("float16", "float16", 2.0 ** -22),
                                     ("bfloat16", "float16", 2.0 ** -16), ("float16", "bfloat16", 2.0 ** -11)])
@pytest.mark.parametrize("nh,nkv,D", [(8, 2, 64), (16, 1, 128), (4, 4, 128)])
def test_decode_rounds_at_the_store(pb, cuda, nh, nkv, D, dt, ot, u):
    """the probabilities keep more bits than the output has, u (two numbers of the cache's type, each off by half a step
    of what is left, or fp16 for bf16), so that the output's own rounding is the largest error"""
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    lens = [1, 2, 3, 17, 200, 70, 2600, 900]
    c = Cache(pb, torch, lens, nkv, D, 32, dt, seed=D + nh)
    S = len(lens)
    q = (torch.randn((S, nh, D), generator=c.g) * 0.5).to(dt).cuda()
    out = torch.empty((S, nh, D), dtype=ot, device="cuda")
    c.h.decode(c.dev(), torch.tensor(lens, dtype=torch.int32, device="cuda"), q, out)
    torch.cuda.synchronize()
    (o, spread, slack, tiny), _ = oracle_rows(c, q, lens, [1] * S, D ** -0.5, 0, 0)
    check(torch, f64(out), o, spread, slack, tiny * 2.0 ** -15, max(lens), dt, ot, "out", u=u)


def test_a_wait_that_gives_up_is_reported_once(pb, cuda):
    """the prompt kernel's wait on a barrier that nothing arrives at, with a limit of 20 ms: recorded by whichever
    stream, reported by the next status of any, once; the calls behind it run as before"""
    torch = cuda
    c = Cache(pb, torch, [200], 2, 64, 16, torch.float16, seed=2)
    q = torch.randn((200, 4, 64), generator=c.g).half().cuda()
    start, length = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 200], [200]))
    want, out = torch.empty_like(q), torch.empty_like(q)
    c.h.prefill(c.dev(), start, length, q, want)
    c.h.status()
    side = torch.cuda.Stream()
    for k in range(3):
        pb.device_kv_wait(20_000_000, side if k else None)
        if k == 1:
            pb.device_kv_wait(20_000_000)         # two records, one report
        torch.cuda.synchronize()                      # (a status waits for its own stream alone)
        with pytest.raises(pb.PBError, match=r"gave up \(role 14\)"):      # (15: the wait behind it, which returns at once)
            c.h.status(None if k else side)
        c.h.status()
        c.h.status(side)
    c.h.prefill(c.dev(), start, length, q, out)
    c.h.status()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dt,ot", FAR + [("bfloat16", "float16")])
def test_scores_near_the_end_of_fp32_integers(pb, cuda, dt, ot):
    """scores of 2^25, whose neighbours are 4 apart, in powers of two: a factor in the probabilities that is subtracted
    from such a maximum would come out as another one and pass fp16's largest value. The scores themselves are exact
    (products of powers of two, and 8): row 100 is 2^8 above row 0, everything else 2^24 below."""
    torch = cuda
    dt, ot = getattr(torch, dt), getattr(torch, ot)
    D, n, nh, scale = 64, 300, 4, 0.6931471824645996      # 2^(scale log2(e) s) = 2^s in fp32
    c = Cache(pb, torch, [n], 2, D, 32, dt, seed=3)
    pg, r, _ = KO.rows_of(c.table.numpy(), 0, n, 32, c.n_pages)
    pg, r = torch.from_numpy(pg).long().cuda(), torch.from_numpy(r).cuda()
    k = torch.zeros((n, 2, D))
    k[0, :, 0], k[100, :, 0], k[100, :, 1] = 8192.0, 8192.0, 8.0
    k[1:100, :, 0], k[101:, :, 0] = 4096.0, 4096.0
    c.k[pg, :, r] = k.to(dt).cuda()
    q = torch.zeros((n, nh, D), dtype=dt, device="cuda")
    q[:, :, 0], q[:, :, 1] = 4096.0, 1.0
    v = f64(c.v[pg, :, r])                                 # [row][kv head][dim]
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    one, out = torch.empty((1, nh, D), dtype=ot, device="cuda"), torch.empty((n, nh, D), dtype=ot, device="cuda")
    c.h.decode(c.dev(), length, q[-1:], one, scale=scale)
    c.h.prefill(c.dev(), torch.tensor([0, n], dtype=torch.int32, device="cuda"), length, q, out, scale=scale)
    chunk = torch.empty((2, nh, D), dtype=ot, device="cuda")
    c.h.prefill(c.dev(), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), length, q[-2:], chunk, scale=scale)
    torch.cuda.synchronize()
    for h in range(nh):
        both = (256 * v[100, h // 2] + v[0, h // 2]) / 257
        # a probability's rounding in the cache's type, the store's, and a few of fp32
        tol = (U(torch, dt) + U(torch, ot) + 2.0 ** -20) * (256 * np.abs(v[100, h // 2]) + np.abs(v[0, h // 2])) / 257 + 2.0 ** -25
        for got, want in ((one[0], both), (out[99], v[0, h // 2]), (out[100], both), (out[n - 1], both), (chunk[0], both), (chunk[1], both)):
            assert (np.abs(f64(got)[h] - want) <= tol + (U(torch, ot) + 2.0 ** -20) * np.abs(want)).all(), h
