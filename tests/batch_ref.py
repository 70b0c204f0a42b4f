"""A batch's decode step in plain numpy: rows of the paged cache as they are stored,
attention and sampling in 64 bits."""
import numpy as np

U11 = 2.0 ** -11  # half a step of fp16
U24 = 2.0 ** -24  # of fp32


def quant(orc, x):
    """e4m3 bytes and fp16 scale bits of fp16 rows x [..., dim]: fp32 amax / 448 + 1e-12,
    IEEE quotients (a NaN has no part in amax)."""
    x = np.asarray(x, np.float16).astype(np.float32)
    with np.errstate(all="ignore"):
        amax = np.fmax.reduce(np.abs(x), axis=-1, initial=np.float32(0))
        s = (amax / np.float32(448) + np.float32(1e-12)).astype(np.float32)
        y = (x / s[..., None]).astype(np.float32)
        return orc.e4m3_encode(y.reshape(-1)).reshape(x.shape), s.astype(np.float16)


def table_of(rng, n_pages, counts, width, bad=-1):
    """Pages in a shuffled order: table [len(counts), width], `bad` behind each sequence's last."""
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(counts), width), bad, np.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    assert at <= n_pages
    return table


def places(table, n_pages, page, seq, pos):
    """(page, row, whether there is one) of each token."""
    seq, pos = np.asarray(seq, np.int64), np.asarray(pos, np.int64)
    ok = (seq >= 0) & (seq < table.shape[0]) & (pos >= 0) & (pos < table.shape[1] * page)
    pid = np.where(ok, table[np.where(ok, seq, 0), np.where(ok, pos // page, 0)], -1)
    ok &= (pid >= 0) & (pid < n_pages)
    return np.where(ok, pid, 0), np.where(ok, pos % page, 0), ok


def attend(q, k, v, table, page, seq, pos, scale, window):
    """q [T, n_q, dim]; k, v [pages, kv, page, dim] as numbers: outputs in 64 bits and
    how far a kernel in fp32 may be off them in fp16.

    A score of D products in fp32, scaled: at most (D + 6) half steps of sum |q k| scale
    and 2 of itself, its weight off by as much times itself; the exponential and its
    argument 4 and as many half steps as the score has units; sums over n tokens, in
    chains and their joins, (n / 16 + 64) half steps of sum w |v|; numerators are two fp16
    whose largest is 2^12 or more, each off by 2^-22 of itself or half the least step,
    2^-25, which is 2^-37 of the largest: n times that of max w times max |v|.  A score's error moves numerator and denominator: twice.  Then
    half an fp16 step."""
    T, n_q, D = q.shape
    n_kv = k.shape[1]
    out = np.zeros((T, n_q, D))
    bound = np.zeros((T, n_q, D))
    for t in range(T):
        s = seq[t]
        if not 0 <= s < table.shape[0] or pos[t] < 0:
            continue
        j = np.arange(max(0, pos[t] + 1 - window) if window else 0, min(pos[t] + 1, table.shape[1] * page))
        pid, row, ok = places(table, k.shape[0], page, np.full(j.size, s), j)
        pid, row = pid[ok], row[ok]
        if not pid.size:
            continue
        for g in range(n_kv):
            kk, vv = k[pid, g, row].astype(np.float64), v[pid, g, row].astype(np.float64)
            qq = q[t, g * (n_q // n_kv):(g + 1) * (n_q // n_kv)].astype(np.float64)
            x = (qq @ kk.T) * scale
            off = np.abs(qq) @ np.abs(kk).T * abs(scale) * (D + 6) * U24 + np.abs(x) * 2 * U24
            top = x.max(1, keepdims=True)
            w = np.exp(x - top)
            off = off + off.max(1, keepdims=True) + (4 + np.abs(x) + np.abs(top)) * 2 * U24
            w /= w.sum(1, keepdims=True)
            o = w @ vv
            h = slice(g * (n_q // n_kv), (g + 1) * (n_q // n_kv))
            out[t, h] = o
            mass = w @ np.abs(vv)
            bound[t, h] = (np.expm1(2 * off) * w) @ np.abs(vv) + np.abs(o) * (np.expm1(2 * off) * w).sum(1, keepdims=True) \
                + mass * ((pid.size / 16 + 64) * 2 * U24 + 2.0 ** -22) + pid.size * 2.0 ** -37 * w.max() * np.abs(vv).max()
    return out, bound * 1.01 + np.abs(out) * U11 * 1.001 + 2.0 ** -25


def choose(l, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Token, its probability, and how near the draw came to another token (in units of
    the kept mass) for each row of l."""
    B, V = l.shape
    ids, p, near = np.zeros(B, np.int64), np.zeros(B), np.ones(B)
    for b in range(B):
        x = np.where(np.isnan(l[b]), -np.inf, l[b].astype(np.float64))
        if np.isposinf(x).any():
            x = np.where(np.isposinf(x), 0.0, -np.inf)
        order = np.argsort(-x, kind="stable")
        x = x[order]
        if x[0] == -np.inf:
            ids[b] = -1
            continue
        t = 1.0 if temperature is None else float(temperature[b])
        if not t > 0:
            ids[b], p[b] = order[0], 1.0
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(x == -np.inf, 0.0, np.exp((x - x[0]) / t))
        n = V
        if top_k is not None and 0 < top_k[b] < V:
            n = int(top_k[b])
        run = np.cumsum(w)
        if top_p is not None and top_p[b] < 1:
            n = min(n, int((run < max(float(top_p[b]), 0.0) * run[n - 1]).sum()) + 1)
        if min_p is not None and min_p[b] > 0:
            n = min(n, int((w >= min(float(min_p[b]), 1.0)).sum()))
        r = 0.0 if not u[b] >= 0 else min(float(u[b]), 1 - 2.0 ** -24)
        i = min(int((run[:n] <= r * run[n - 1]).sum()), n - 1)
        ids[b], p[b] = order[i], w[i] / run[n - 1]
        near[b] = np.abs(run[:n] - r * run[n - 1])[w[:n] > 0].min() / run[n - 1]
    return ids, p, near
