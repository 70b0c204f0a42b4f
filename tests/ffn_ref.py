"""Plain 64-bit forms of the feed-forward branch's operators, with the bounds
their fp32 kernels are held to, for the tests."""
import numpy as np

U24, U11 = 2.0 ** -24, 2.0 ** -11  # half steps of fp32 and fp16, relative


def quant(rng, *shape):
    """INT4 experts [E, rows, cols]: packed u8, fp16 scales and the fp64 weights."""
    E, rows, cols = shape
    packed = rng.integers(0, 256, (E, rows, cols // 2), dtype=np.uint8)
    scales = ((0.02 + 0.2 * rng.random((E, rows, cols // 128))) / np.sqrt(cols)).astype(np.float16)
    nib = np.stack((packed & 15, packed >> 4), -1).reshape(E, rows, cols).astype(np.float64) - 8.0
    return packed, scales, nib * np.repeat(scales.astype(np.float64), 128, axis=2)


def norm(h, add, w, eps):
    """(hsum, out) in fp64 and out's bound."""
    s = h.astype(np.float64) + (0.0 if add is None else add.astype(np.float64))
    y = s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * w.astype(np.float64)
    # hsum's rounding, the sum of squares (at most H / 64 + 16 additions in a row,
    # halved by the root), root, quotient, two products; then fp16
    big = np.abs(s).max(1, keepdims=True) if s.size else np.abs(s)
    rel = (h.shape[1] / 64 + 32) * U24
    lost = 0.0 if add is None else U24 * big / np.sqrt((s * s).mean(1, keepdims=True) + eps) * np.abs(w.astype(np.float64))
    return s, y, np.abs(y) * (U11 * 1.001 + rel) + lost + 2.0 ** -25


def choose(logits, bias, k, score="sigmoid", n_group=1, topk_group=1, renorm=True, eps=1e-6, scale=1.0):
    """ids [S, k] and weights [S, k] in fp64 from fp64 logits [S, E]."""
    S, E = logits.shape
    ids, wt = np.zeros((S, k), np.int32), np.zeros((S, k))
    with np.errstate(all="ignore"):
        for t in range(S):
            l = logits[t]
            if score == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-l))
            elif np.all(l == -np.inf):
                s = np.zeros(E)
            else:
                p = np.exp(l - l.max())
                s = p / p.sum()
            c = s if bias is None else s + bias.astype(np.float64)
            c = np.where(np.isnan(c), -np.inf, c)
            allowed = list(range(E))
            if n_group > 1:
                per = E // n_group
                best = []
                for g in range(n_group):
                    v = sorted(c[g * per:(g + 1) * per], reverse=True)[:2]
                    b = v[0] + v[1] if per > 1 else v[0]
                    best.append(-np.inf if np.isnan(b) else b)
                kept = sorted(range(n_group), key=lambda g: (-best[g], g))[:topk_group]
                allowed = [e for e in allowed if e // per in kept]
            ids[t] = sorted(allowed, key=lambda e: (-c[e], e))[:k]
            w = s[ids[t]]
            if renorm:
                d = w.sum() + np.float64(np.float32(eps))
                w = np.zeros(k) if d == 0.0 else w / d
            wt[t] = w * np.float64(np.float32(scale))
    return ids, wt


def weights_bound(logits, far, ids, weights, score="sigmoid", renorm=True, scale=1.0, eps=1e-6, **kw):
    """Of the weights of experts ids, their logits at most far off."""
    most = far.max(1, keepdims=True)
    if score == "sigmoid":  # slope s (1 - s) <= 1/4, and its square
        s = 1.0 / (1.0 + np.exp(-logits))
        ds = np.take_along_axis(s * (1 - s) * far + far * far, ids, 1)
    else:                   # s (dl - sum s dl), and its square
        p = np.exp(logits - logits.max(1, keepdims=True))
        s = p / p.sum(1, keepdims=True)
        ds = np.take_along_axis(s * 2 * most * (1 + 2 * most), ids, 1)
    s = np.take_along_axis(s, ids, 1)
    if renorm:
        total = s.sum(1, keepdims=True) + eps
        ds = (ds + s / total * ds.sum(1, keepdims=True)) / (total - ds.sum(1, keepdims=True))
    return abs(scale) * ds * 1.01 + 1.001 * U24 * np.abs(weights) + 1e-12


def pairs(ids, S, k, E):
    """(row s * k + j, token s, expert) of the pairs that take part."""
    if ids is None:
        return [(s, s, 0) for s in range(S)]
    return [(s * k + j, s, int(ids[s, j])) for s in range(S) for j in range(k) if 0 <= ids[s, j] < E]


def up(x, ids, W1, W3, k):
    """act [S k, F] fp64 (NaN where a pair takes no part) and its bound."""
    S, (E, F, H) = x.shape[0], W1.shape
    act, bound = np.full((S * k, F), np.nan), np.full((S * k, F), np.nan)
    xd = x.astype(np.float64)
    # a group's 128 products, then a fused add for each of H / 128 groups and the
    # meeting of at most 16 partial sums
    n = (128 + H / 128 + 20) * U24
    for r, s, e in pairs(ids, S, k, E):
        g, u = W1[e] @ xd[s], W3[e] @ xd[s]
        dg, du = n * (np.abs(W1[e]) @ np.abs(xd[s])), n * (np.abs(W3[e]) @ np.abs(xd[s]))
        silu = g / (1.0 + np.exp(-g))
        act[r] = silu * u
        # |silu'| <= 1.1; exp of an argument rounded to fp32 is |g| 2^-23 off
        bound[r] = (np.abs(act[r]) * (U11 * 1.001 + (np.abs(g) + 8.0) * 2 * U24) + 1.1 * dg * (np.abs(u) + du)
                    + (np.abs(silu) + 1.1 * dg) * du + 2.0 ** -25)
    return act, bound


def down(act, ids, weights, W2, res, k):
    """out [S, H] fp64 and its bound; act fp16 [S k, F]."""
    S, (E, H, F) = res.shape[0], W2.shape
    out, mag, bound = res.astype(np.float64), np.abs(res.astype(np.float64)), np.zeros(res.shape)
    n = (128 + F / 128 + 20) * U24
    for r, s, e in pairs(ids, S, k, E):
        w = 1.0 if weights is None else float(weights.reshape(-1)[r])
        a = act[r].astype(np.float64)
        y = w * (W2[e] @ a)
        out[s] += y
        mag[s] += np.abs(y)
        bound[s] += n * abs(w) * (np.abs(W2[e]) @ np.abs(a))
    return out, bound + (k + 3) * U24 * mag
