"""The paged K/V cache's operators in 64 bits, from their formulas (numpy), for
test_kv.py and test_gpu_kv.py: pools [page][kv head][row][dim], tables
[sequence][n]. A table entry outside the pool hides its rows."""
import numpy as np


def rows_of(table, b, n, page_size, n_pages):
    """(page, row in page, valid) of rows 0..n-1 of sequence b"""
    j = np.arange(n)
    pg = np.asarray(table)[b][j // page_size] if n else np.zeros(0, int)
    return pg, j % page_size, (pg >= 0) & (pg < n_pages)


def seen(t, n, window, sinks):
    """rows 0..n-1 that the token at row t sees"""
    j = np.arange(n)
    s = j <= t
    if window > 0:
        s &= (j > t - window) | (j < sinks)
    return s


def append(k, v, w, table, seq, slot, pos, x, nh, qn, kn, eps, cos, sin, q):
    """in place on float64 k, v, w, q"""
    n_pages, nkv, ps, D = k.shape
    half = 0 if cos is None else cos.shape[1]

    def head(y, nw, p):
        y = y.astype(np.float64)
        if nw is not None:
            y = y * nw / np.sqrt((y * y).mean() + eps)
        if half:
            a, b = y[:half].copy(), y[D // 2:D // 2 + half].copy()
            c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
            y[:half], y[D // 2:D // 2 + half] = a * c - b * s, b * c + a * s
        return y

    for i in range(x.shape[0]):
        b, j = int(seq[i]), int(slot[i])
        p = j if pos is None else int(pos[i])
        if not (0 <= b < len(table) and 0 <= j < table.shape[1] * ps) or (half and not 0 <= p < cos.shape[0]):
            continue
        pg, r = int(table[b][j // ps]), j % ps
        if not 0 <= pg < n_pages:
            continue
        xs = x[i][:(nh + 2 * nkv) * D].reshape(nh + 2 * nkv, D)
        for h in range(nh):
            q[i, h] = head(xs[h], qn, p)
        for h in range(nkv):
            k[pg, h, r] = head(xs[nh + h], kn, p)
            v[pg, h, r] = xs[nh + nkv + h]
            if w is not None:
                w[pg, h, r] = 0.0


def attend(q, k, v, w, table, b, t, n, scale, window, sinks):
    """one token's heads q [nh][D] at row t of sequence b with n rows -> (out, spread [nh][D], slack [nh], p [nkv][n]).
    spread = sum p |v|; slack bounds the relative error of a probability from fp32 scores."""
    n_pages, nkv, ps, D = k.shape
    nh = q.shape[0]
    out, spread, slack = np.zeros((nh, D)), np.zeros((nh, D)), np.zeros(nh)
    tiny, psum = np.zeros((nh, D)), np.zeros((nkv, n))
    pg, r, ok = rows_of(table, b, n, ps, n_pages)
    at = np.nonzero(ok & seen(t, n, window, sinks))[0]
    if not len(at):
        return out, spread, slack, tiny, psum
    for kh in range(nkv):
        kk, vv = k[pg[at], kh, r[at]].astype(np.float64), v[pg[at], kh, r[at]].astype(np.float64)
        for h in range(kh * (nh // nkv), (kh + 1) * (nh // nkv)):
            s = kk @ q[h].astype(np.float64) * scale
            e = np.exp(s - s.max())
            p = e / e.sum()
            out[h], spread[h] = p @ vv, p @ np.abs(vv)
            # an fp32 dot of D terms is off by at most D half steps of sum |q k|; the scaling, the
            # subtraction of the maximum and the power of two add a few half steps of |s|
            mag = (np.abs(kk) @ np.abs(q[h].astype(np.float64))).max() * scale
            slack[h] = 2.0 ** -24 * ((D + 8) * mag + 16)
            tiny[h] = np.abs(vv).sum(0) / e.sum()
            psum[kh, at] += p
    return out, spread, slack, tiny, psum


def evict_rows(wgt, n, budget, sinks, recent):
    """the rows of one K/V head that stay, in order (wgt: the weights of rows 0..n-1)"""
    if n <= budget:
        return list(range(n))
    wgt = [float(x) if x > 0 else 0.0 for x in wgt]
    lo, hi = min(sinks, n), max(min(sinks, n), n - recent)
    free = sorted(range(lo, hi), key=lambda j: (-wgt[j], j))
    gone = set(free[len(free) - (n - budget):])
    return [j for j in range(n) if j not in gone]


def evict_rows_named(wgt, named, n, budget, sinks, recent):
    """the same where some rows lie on no page (named: which do): those are left out, as if they were not there, but the
    first and the last rows are counted by their place in the sequence"""
    have = [j for j in range(n) if named[j]]
    if len(have) <= budget:
        return have
    wgt = [float(x) if x > 0 else 0.0 for x in wgt]
    lo, hi = min(sinks, n), max(min(sinks, n), n - recent)
    free = sorted((j for j in have if lo <= j < hi), key=lambda j: (-wgt[j], j))
    gone = set(free[len(free) - (len(have) - budget):])
    return [j for j in have if j not in gone]
