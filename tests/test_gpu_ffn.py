"""The feed-forward branch's operators on the GPU against 64-bit forms."""
import numpy as np
import pytest
import torch

import ffn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cia, dev):
    from cuda_inf_amd import kernels
    return kernels


def t(a, dev):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def within(got, want, bound, what):
    err = np.abs(np.asarray(got, np.float64) - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(err / bound)} of the bound"


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize("S,H,add", [(1, 2048, False), (1, 8, True), (5, 64, True), (3, 1000, False),
                                     (2, 2056, True), (7, 4096, False), (2, 8200, True), (4, 20000, False),
                                     (513, 2048, True)])
def test_norm(K, dev, S, H, add):
    rng = np.random.default_rng(S * 7 + H)
    h = (rng.standard_normal((S, H)) * (1 + 50 * (rng.random(H) < 0.02))).astype(np.float32)
    b = rng.standard_normal((S, H)).astype(np.float32) if add else None
    w = (1 + 0.3 * rng.standard_normal(H)).astype(np.float16)
    hd, bd = t(h, dev), t(b, dev)
    out = torch.full((S, H), 7.0, dtype=torch.float16, device=dev)
    hs = torch.empty_like(hd)
    K.add_rmsnorm(hd, t(w, dev), out, S, H, 1e-5, add=bd, hsum=hs)
    _, y, bound = ref.norm(h, b, w, 1e-5)
    within(out.cpu().numpy(), y, bound, "norm")
    assert torch.equal(hs, hd if bd is None else hd + bd)
    # in place, and without the sum
    out2 = torch.empty_like(out)
    K.add_rmsnorm(hd, t(w, dev), out2, S, H, 1e-5, add=bd)
    assert torch.equal(out, out2)
    K.add_rmsnorm(hd, t(w, dev), out2, S, H, 1e-5, add=bd, hsum=hd)
    assert torch.equal(out, out2) and torch.equal(hd, hs)


@pytest.mark.parametrize("H", [(1 << 24) - 8, 1 << 24, (1 << 22) + 8])
def test_norm_of_the_longest_rows(K, dev, H):
    """Rows whose elements are all alike, whose squares lose the same at every addition
    where they are added up in one fp32 chain: the bound does not grow with H."""
    rng = np.random.default_rng(H)
    w = (1 + rng.random(H)).astype(np.float16)
    value = np.array([1.3361171, 1.0165276, 0.03], np.float32)
    h = np.repeat(value[:, None], H, 1)
    h[2] = rng.standard_normal(H)
    out = torch.empty((3, H), dtype=torch.float16, device=dev)
    K.add_rmsnorm(t(h, dev), t(w, dev), out, 3, H, 1e-5)
    got = out.cpu().numpy()
    for r in range(3):
        s = h[r].astype(np.float64)
        y = s / np.sqrt((s * s).mean() + 1e-5) * w.astype(np.float64)
        # 8 squares a step, the steps in 64 bits, at most 16 additions where the row's
        # parts meet: 24 half steps, halved by the root; mean, eps, root, quotient, two
        # products; then fp16
        within(got[r], y, np.abs(y) * (ref.U11 * 1.001 + (12 + 8) * ref.U24) + 2.0 ** -25, f"row {r}")


def test_norm_rows_of_zeros_and_beyond_numbers(K, dev):
    h = torch.zeros((4, 256), device=dev)
    h[1, 3], h[2, 5] = float("nan"), float("inf")
    h[3] = 1e18  # (squares past fp32's range would need 2e19)
    w = torch.ones(256, dtype=torch.float16, device=dev)
    out = torch.empty((4, 256), dtype=torch.float16, device=dev)
    K.add_rmsnorm(h, w, out, 4, 256)
    o = out.float().cpu()
    assert (o[0] == 0).all() and o[1].isnan().all()
    assert o[2, 5].isnan() and (o[2, :5] == 0).all()
    assert (o[3] == 1).all()


# ------------------------------------------------------------------ router
@pytest.mark.parametrize("S,H,E,kw", [
    (1, 2048, 32, dict(k=4)),
    (5, 256, 1, dict(k=1)),
    (3, 8, 7, dict(k=7, renorm=False)),
    (17, 1000, 33, dict(k=5, score="softmax")),
    (65, 512, 64, dict(k=8, score="softmax", renorm=False, scale=2.5)),
    (9, 1280, 128, dict(k=6, n_group=8, topk_group=3)),
    (4, 384, 256, dict(k=16, n_group=16, topk_group=1, score="softmax")),
    (6, 128, 24, dict(k=2, n_group=24, topk_group=2)),
    (40, 640, 200, dict(k=3)),
    (300, 2048, 32, dict(k=4, eps=0.0)),
    (2, 8200, 20, dict(k=2)),
    (1030, 72, 40, dict(k=4)),
    (1024, 256, 17, dict(k=5, score="softmax")),
    (2050, 136, 100, dict(k=3, n_group=4, topk_group=2)),
])
@pytest.mark.parametrize("bias", [False, True])
def test_route(K, dev, S, H, E, kw, bias):
    kw = dict(kw)
    k = kw.pop("k")
    rng = np.random.default_rng(S + 3 * H + E)
    x = rng.standard_normal((S, H)).astype(np.float16)
    gate = (rng.standard_normal((E, H)) / np.sqrt(H)).astype(np.float16)
    b = (0.1 * rng.standard_normal(E)).astype(np.float32) if bias else None
    l = x.astype(np.float64) @ gate.astype(np.float64).T
    ids, wt = ref.choose(l, b, k, **kw)
    gi = torch.full((S, k), -7, dtype=torch.int32, device=dev)
    gw, gl = torch.zeros((S, k), device=dev), torch.zeros((S, E), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, bias=t(b, dev), logits=gl, **kw)
    assert np.array_equal(gi.cpu().numpy(), ids)
    # logits: sums of 32 products in fp32, their sum in 64 bits, one rounding
    far = 32 * ref.U24 * (np.abs(x.astype(np.float64)) @ np.abs(gate.astype(np.float64)).T)
    within(gl.cpu().numpy(), l, ref.U24 * np.abs(l) + far, "logits")
    within(gw.cpu().numpy(), wt, ref.weights_bound(l, far, ids, wt, **kw), "weights")
    # the logits are optional
    g2, w2 = torch.empty_like(gi), torch.empty_like(gw)
    K.moe_route(t(x, dev), t(gate, dev), g2, w2, S, H, E, k, bias=t(b, dev), **kw)
    assert torch.equal(gi, g2) and torch.equal(gw, w2)
    # a token's experts do not depend on the tokens beside it
    if S > 1:
        for i in (0, S // 2, S - 1):
            K.moe_route(t(x[i:i + 1], dev), t(gate, dev), g2, w2, 1, H, E, k, bias=t(b, dev), **kw)
            assert torch.equal(gi[i], g2[0])


@pytest.mark.parametrize("S,E,kw", [(5, 32, dict(k=4)), (70, 40, dict(k=6, score="softmax")), (600, 32, dict(k=4)),
                                    (1100, 64, dict(k=4, n_group=8, topk_group=3)),
                                    (1100, 130, dict(k=8, score="softmax", n_group=13, topk_group=2))])
def test_route_of_near_choices(K, dev, S, E, kw):
    """Gate rows a few fp16 steps apart, rows of x that are zero, equal or not finite:
    the choice is the 64-bit sums', ties to the lowest index."""
    kw = dict(kw)
    k, H = kw.pop("k"), 512
    rng = np.random.default_rng(E)
    x = rng.standard_normal((S, H)).astype(np.float16)
    base = rng.standard_normal(H) / np.sqrt(H)
    gate = np.repeat(base[None], E, 0).astype(np.float16)
    step = rng.integers(-2, 3, (E, H)).astype(np.int16) * (rng.random((E, H)) < 0.01)
    gate = (gate.view(np.int16) + step.astype(np.int16)).view(np.float16)
    gate[E - 1] = gate[0]
    x[0] = 0
    x[S // 2] = 0
    x[S - 1] = x[1]
    x[3, 7] = np.inf
    x[2, 5] = np.nan
    good = ~np.isnan(x).any(1) & ~np.isinf(x).any(1)
    l = np.zeros((S, E))
    l[good] = x[good].astype(np.float64) @ gate.astype(np.float64).T
    ids, _ = ref.choose(l, None, k, **kw)
    # (sums in 64 bits are 1e-14 off in an order of their own: rows that hang on it say nothing)
    s = np.sort(l, 1)
    clear = good & ~((np.diff(s, axis=1) > 0) & (np.diff(s, axis=1) < 1e-12)).any(1)
    assert clear.sum() > 0.9 * S - 3
    gi = torch.full((S, k), -7, dtype=torch.int32, device=dev)
    gw = torch.zeros((S, k), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, **kw)
    got = gi.cpu().numpy()
    assert np.array_equal(got[clear], ids[clear])
    for r in got[~good]:  # distinct experts all the same
        assert len(set(r.tolist())) == k and (r >= 0).all() and (r < E).all()


@pytest.mark.parametrize("S", [40, 1100, 2050])
@pytest.mark.parametrize("E,kw", [(32, dict(k=4, n_group=2, topk_group=1)), (64, dict(k=6, n_group=8, topk_group=3)),
                                  (64, dict(k=3, n_group=8, topk_group=1, score="softmax")),
                                  (132, dict(k=5, n_group=12, topk_group=5, score="softmax"))])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("apart", [False, True])
def test_route_of_near_groups(K, dev, S, E, kw, bias, apart):
    """Groups in pairs of equal gate rows, or of rows whose logits are 2^-26 apart, with
    an odd number of groups kept: the last one kept and the first one left out are
    such a pair.  Numbers are whole multiples of small powers of two, so that 64 bits
    hold every sum exactly, in any order, and fp32 does not."""
    kw = dict(kw)
    k, H, per = kw.pop("k"), 512, E // kw["n_group"]
    rng = np.random.default_rng(E + S)
    x = rng.integers(-2047, 2048, (S, H)) / 1024.0
    gate = rng.integers(-2047, 2048, (E // 2, H)) / 65536.0
    gate = np.repeat(gate.reshape(-1, 1, per, H), 2, axis=1).reshape(E, H)
    if apart:
        x[:, 7] = rng.integers(-1, 2, S) / 1024.0
        gate[:, 7] = rng.integers(-2047, 2047, E) / 65536.0
        second = np.arange(E) // per % 2 == 1
        gate[second, 7] = gate[np.flatnonzero(second) - per, 7] + 1.0 / 65536.0
    x, gate = x.astype(np.float16), gate.astype(np.float16)
    b = np.repeat(0.1 * rng.standard_normal((E // 2 // per, 1, per)), 2, axis=1).reshape(E).astype(np.float32) if bias else None
    l = (x.astype(np.float64) * 2.0 ** 10) @ (gate.astype(np.float64) * 2.0 ** 16).T * 2.0 ** -26
    ids, wt = ref.choose(l, b, k, **kw)
    gi, gw = torch.full((S, k), -7, dtype=torch.int32, device=dev), torch.zeros((S, k), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, bias=t(b, dev), **kw)
    wrong = (gi.cpu().numpy() != ids).any(1)
    assert not wrong.any(), f"{wrong.sum()} of {S} tokens, first {np.flatnonzero(wrong)[0]}"
    far = 32 * ref.U24 * (np.abs(x.astype(np.float64)) @ np.abs(gate.astype(np.float64)).T)
    within(gw.cpu().numpy(), wt, ref.weights_bound(l, far, ids, wt, **kw), "weights")
    i1, w1 = torch.empty((1, k), dtype=torch.int32, device=dev), torch.empty((1, k), device=dev)
    for i in range(0, S, S // 13):
        K.moe_route(t(x[i:i + 1], dev), t(gate, dev), i1, w1, 1, H, E, k, bias=t(b, dev), **kw)
        assert torch.equal(i1[0], gi[i])


def near_tokens(rng, S, near, H, E, n_group, topk_group, k, unit):
    """Whole numbers x [S, H], gate [E, H] (a logit is unit times their product's sum)
    and bias [E]: of the first tokens, two of the choices by softmax and bias that
    follow one another lie some 1e-11 apart."""
    per = E // n_group
    x = rng.integers(-2047, 2048, (S, H)).astype(np.float64)
    gate = rng.integers(-2047, 2048, (E, H)).astype(np.float64)
    gate[:, :16] = rng.integers(-7, 8, (E, 16))  # (x moves the logits little here)
    bias = (0.2 * rng.standard_normal(E)).astype(np.float32)

    def soft(l):
        p = np.exp(l - l.max(-1, keepdims=True))
        return p / p.sum(-1, keepdims=True)

    for t in range(near):
        l = x[t] @ gate.T * unit
        c = soft(l) + bias
        kept = np.argsort(-np.sort(c.reshape(n_group, per), 1)[:, -2:].sum(1), kind="stable")[:topk_group]
        of = (kept[:, None] * per + np.arange(per)).reshape(-1)
        of = of[np.argsort(-c[of], kind="stable")][:k + 1]
        j = int(np.argmin(c[of[:-1]] - c[of[1:]]))
        a, b = of[j], of[j + 1]
        for few, most in ((False, 2047), (False, 512), (True, 2047), (True, 2047), (True, 40), (True, 3)):
            cols = np.arange(16) if few else rng.permutation(np.arange(16, H))[:16]
            move = rng.integers(-most, most + 1, (3000, 16)) * (rng.random((3000, 16)) < (1.0 if few else 0.3))
            move[0] = 0
            move = np.clip(x[t, cols] + move, -2047, 2047) - x[t, cols]
            s = soft(l + move @ gate[:, cols].T * unit)
            x[t, cols] += move[np.argmin(np.abs(s[:, a] - s[:, b] + np.float64(bias[a]) - np.float64(bias[b])))]
            l = x[t] @ gate.T * unit
    return x, gate, bias


@pytest.mark.parametrize("E,H,unit,kw", [(48, 256, 2.0 ** -24, dict(k=4, n_group=6, topk_group=3)),
                                         (48, 512, 2.0 ** -24, dict(k=4, n_group=12, topk_group=2)),
                                         (128, 256, 2.0 ** -23, dict(k=6, n_group=8, topk_group=2)),
                                         (48, 256, 2.0 ** -23, dict(k=4, n_group=1, topk_group=1))])
def test_route_of_near_choices_by_softmax_and_bias(K, dev, E, H, unit, kw):
    """Beside a bias a score's distance to another hangs on the sum over all experts,
    those of the groups that are left out among them."""
    kw = dict(kw, score="softmax")
    k, S = kw.pop("k"), 1100
    X, G, b = near_tokens(np.random.default_rng(E + H), S, 64, H, E, kw["n_group"], kw["topk_group"], k, unit)
    x, gate = (X * (unit * 65536.0)).astype(np.float16), (G / 65536.0).astype(np.float16)
    l = X @ G.T * unit  # (exact: whole numbers below 2^31)
    ids, wt = ref.choose(l, b, k, **kw)
    # (scores in 64 bits are 1e-16 off: tokens that hang on it say nothing)
    p = np.exp(l - l.max(1, keepdims=True))
    clear = (np.diff(np.sort(p / p.sum(1, keepdims=True) + b, 1), axis=1) > 1e-14).all(1)
    assert clear.sum() > S - 20
    gi, gw = torch.full((S, k), -7, dtype=torch.int32, device=dev), torch.zeros((S, k), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, bias=t(b, dev), **kw)
    wrong = (gi.cpu().numpy() != ids).any(1) & clear
    assert not wrong.any(), f"{wrong.sum()} of {S} tokens, first {np.flatnonzero(wrong)[0]}"


@pytest.mark.parametrize("E,kw", [(32, dict(k=4)), (9, dict(k=3, score="softmax")),
                                  (64, dict(k=5, n_group=8, topk_group=2, score="softmax", renorm=False)),
                                  (256, dict(k=8, n_group=4, topk_group=2)), (100, dict(k=10))])
@pytest.mark.parametrize("bias", [False, True])
def test_select_of_logits(K, dev, E, kw, bias):
    """Equal logits, infinities and what is not a number among them."""
    kw = dict(kw)
    k = kw.pop("k")
    rng = np.random.default_rng(E)
    l = rng.standard_normal((70, E)).astype(np.float32)
    l[1] = 0.25                                  # all equal
    l[2, ::2] = l[2, 1]                          # many equal
    l[3, rng.random(E) < 0.9] = -np.inf
    l[4] = -np.inf
    l[5] *= 1e30
    l[6, 0] = np.inf if kw.get("score") != "softmax" else 90.0
    l[7] = np.round(l[7])
    b = np.round(rng.standard_normal(E), 1).astype(np.float32) if bias else None
    if bias:
        b[E // 2:] = -np.inf                     # experts that are shut
    ids, wt = ref.choose(l.astype(np.float64), b, k, **kw)
    # (from logits that are given, 64 bits up to one rounding)
    gi, gw = torch.empty((70, k), dtype=torch.int32, device=dev), torch.empty((70, k), device=dev)
    K.moe_select(t(l, dev), gi, gw, 70, E, k, bias=t(b, dev), **kw)
    assert np.array_equal(gi.cpu().numpy(), ids)
    within(gw.cpu().numpy(), wt, 1.001 * ref.U24 * np.abs(wt) + 1e-12, "weights")


def test_select_of_nan(K, dev):
    """A row with a NaN: the experts stay distinct and in range, the weights of NaN
    scores are NaN; other rows are not touched."""
    l = torch.randn((3, 16), device=dev)
    l[1, 5] = float("nan")
    ids, w = torch.empty((3, 4), dtype=torch.int32, device=dev), torch.empty((3, 4), device=dev)
    K.moe_select(l, ids, w, 3, 16, 4)
    assert 5 not in ids[1].tolist() and not w.isnan().any()
    K.moe_select(l, ids, w, 3, 16, 4, score="softmax")
    assert ids[1].tolist() == [0, 1, 2, 3] and w[1].isnan().all()
    assert not w[0].isnan().any() and not w[2].isnan().any()


# ------------------------------------------------------------------ experts
def make(rng, S, k, E, H, F, how="even"):
    ids = None
    if how != "dense":
        ids = np.stack([rng.permutation(E)[:k] if k <= E else rng.integers(0, E, k) for _ in range(S)]).astype(np.int32)
    if how == "one":      # every pair on one expert
        ids[:] = E - 1
    if how == "holes":
        ids[rng.random((S, k)) < 0.3] = -1
        ids[0] = [E, -5, 2 ** 31 - 1, -2 ** 31][:k] + [-1] * max(0, k - 4)
    if how == "none":
        ids[:] = -1
    if how == "skew":
        ids[:S * 3 // 4] = 0
    return ids


SIZES = [
    # S, k, E, H, F, how
    (1, 4, 32, 2048, 256, "even"),
    (1, 1, 1, 128, 128, "dense"),
    (1, 16, 16, 256, 128, "even"),
    (2, 6, 3, 384, 256, "even"),        # ids repeat within a token
    (7, 4, 8, 1792, 384, "holes"),
    (16, 1, 1, 640, 256, "dense"),
    (17, 1, 1, 256, 512, "dense"),
    (33, 2, 4, 512, 1792, "holes"),
    (45, 4, 32, 256, 384, "holes"),
    (60, 4, 5, 896, 256, "skew"),
    (64, 1, 1, 2048, 128, "dense"),
    (129, 1, 1, 384, 384, "dense"),
    (150, 2, 256, 128, 128, "even"),
    (3, 2, 2, 128, 7168, "even"),
    (5, 1, 1, 8320, 128, "dense"),
    (90, 3, 7, 4096, 128, "skew"),
    (9, 2, 4, 256, 256, "none"),
    (257, 2, 3, 256, 640, "one"),
    (300, 3, 6, 384, 256, "holes"),
    (700, 4, 8, 256, 256, "skew"),
    (1111, 1, 1, 256, 384, "dense"),
    (4200, 1, 1, 128, 256, "dense"),
    (20, 1, 1, 256, 256, "holes"),
    (1400, 1, 1, 128, 128, "holes"),
    (8500, 2, 6, 128, 128, "holes"),
    (1500, 2, 16, 2048, 128, "even"),
    (1300, 2, 4, 128, 2304, "holes"),
]


@pytest.mark.parametrize("S,k,E,H,F,how", SIZES)
def test_up(K, dev, S, k, E, H, F, how):
    rng = np.random.default_rng(S + k + E + H + F)
    x = rng.standard_normal((S, H)).astype(np.float16)
    p1, s1, W1 = ref.quant(rng, E, F, H)
    p3, s3, W3 = ref.quant(rng, E, F, H)
    ids = make(rng, S, k, E, H, F, how)
    want, bound = ref.up(x, ids, W1, W3, k)
    act = torch.full((S, k, F), 3.0, dtype=torch.float16, device=dev)
    ws = torch.full((K.moe_workspace_bytes(S, k, E, H, F),), 0xAB, dtype=torch.uint8, device=dev)
    args = (t(x, dev), t(ids, dev), (t(p1, dev), t(s1, dev)), (t(p3, dev), t(s3, dev)))
    K.moe_up_int4(*args, act, S, k, ws)
    got = act.view(S * k, F).cpu().numpy()
    out = np.isnan(want[:, 0])
    assert (got[out] == 3.0).all(), "rows of pairs that take no part were written"
    within(got[~out], want[~out], bound[~out], "act")
    first = act.clone()
    K.moe_up_int4(*args, act, S, k, ws)
    assert torch.equal(first, act)


@pytest.mark.parametrize("S,k,E,H,F,how", SIZES)
@pytest.mark.parametrize("weighted", [True, False])
def test_down(K, dev, S, k, E, H, F, how, weighted):
    H, F = F, H  # the same contraction lengths as test_up
    rng = np.random.default_rng(S + k + E + H + F + 1)
    act = rng.standard_normal((S * k, F)).astype(np.float16)
    p2, s2, W2 = ref.quant(rng, E, H, F)
    ids = make(rng, S, k, E, F, H, how)
    wt = rng.standard_normal((S, k)).astype(np.float32) if weighted else None
    res = rng.standard_normal((S, H)).astype(np.float32)
    want, bound = ref.down(act, ids, wt, W2, res, k)
    if ids is not None:  # what the rows of pairs that take no part hold is not read
        dead = (ids.reshape(-1) < 0) | (ids.reshape(-1) >= E)
        act[dead] = np.nan
        if weighted:
            wt.reshape(-1)[dead] = np.nan
    rd = t(res, dev)
    out = torch.full((S, H), 5.0, device=dev)
    ws = torch.full((K.moe_workspace_bytes(S, k, E, H, F),), 0xFF, dtype=torch.uint8, device=dev)
    args = (t(act, dev), t(ids, dev), t(wt, dev), (t(p2, dev), t(s2, dev)))
    K.moe_down_int4(*args, rd, out, S, k, ws)
    within(out.cpu().numpy(), want, bound, "out")
    K.moe_down_int4(*args, rd, rd, S, k, ws)  # in place
    assert torch.equal(rd, out)


@pytest.mark.parametrize("S,k,E", [(2, 2, 4), (30, 2, 4), (400, 2, 4), (700, 2, 4)])
def test_small_numbers(K, dev, S, k, E):
    """fp16 numbers below the normal ones keep their value, in x, scales and act."""
    H, F = 512, 256
    rng = np.random.default_rng(S)
    small = lambda *n: (rng.integers(-1000, 1001, n) * 2.0 ** -24).astype(np.float16)
    ids = make(rng, S, k, E, H, F)
    p1, s1, _ = ref.quant(rng, E, F, H)
    p3, s3, _ = ref.quant(rng, E, F, H)
    p2, s2, _ = ref.quant(rng, E, H, F)
    wide = lambda p, s: (np.stack((p & 15, p >> 4), -1).reshape(E, p.shape[1], -1).astype(np.float64) - 8.0
                         ) * np.repeat(s.astype(np.float64), 128, axis=2)
    res = np.zeros((S, H), np.float32)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device=dev)
    act, out = torch.empty((S, k, F), dtype=torch.float16, device=dev), torch.empty((S, H), device=dev)
    for tiny_x in (True, False):
        big = lambda s: (s.astype(np.float64) * 3000).astype(np.float16)
        if tiny_x:
            x, a, c1, c3, c2 = small(S, H), small(S * k, F), big(s1), big(s3), big(s2)
        else:
            x, a = (100 * rng.standard_normal((S, H))).astype(np.float16), rng.standard_normal((S * k, F)).astype(np.float16)
            c1, c3, c2 = (np.abs(small(*s.shape)) for s in (s1, s3, s2))
        want, bound = ref.up(x, ids, wide(p1, c1), wide(p3, c3), k)
        K.moe_up_int4(t(x, dev), t(ids, dev), (t(p1, dev), t(c1, dev)), (t(p3, dev), t(c3, dev)), act, S, k, ws)
        within(act.view(S * k, F).cpu().numpy(), want, bound, "act")
        want, bound = ref.down(a, ids, None, wide(p2, c2), res, k)
        K.moe_down_int4(t(a, dev), t(ids, dev), None, (t(p2, dev), t(c2, dev)), t(res, dev), out, S, k, ws)
        within(out.cpu().numpy(), want, bound, "out")


@pytest.mark.parametrize("S", [3, 300, 1100])
def test_route_of_small_numbers(K, dev, S):
    rng = np.random.default_rng(S)
    H, E, k = 640, 20, 4
    x = (rng.integers(-1000, 1001, (S, H)) * 2.0 ** -24).astype(np.float16)
    gate = (1000 * rng.standard_normal((E, H))).astype(np.float16)
    l = x.astype(np.float64) @ gate.astype(np.float64).T
    ids, wt = ref.choose(l, None, k)
    gi, gw = torch.empty((S, k), dtype=torch.int32, device=dev), torch.empty((S, k), device=dev)
    gl = torch.empty((S, E), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, logits=gl)
    assert np.array_equal(gi.cpu().numpy(), ids)
    far = 32 * ref.U24 * (np.abs(x.astype(np.float64)) @ np.abs(gate.astype(np.float64)).T)
    within(gl.cpu().numpy(), l, ref.U24 * np.abs(l) + far, "logits")


@pytest.mark.parametrize("S,E", [(2, 20), (2, 100), (300, 20), (300, 100), (1100, 20)])
def test_route_of_a_bad_gate(K, dev, S, E):
    """Infinities and NaN in two experts' gates reach those experts' logits alone."""
    rng = np.random.default_rng(S + E)
    H, k = 4168, 4
    x = rng.standard_normal((S, H)).astype(np.float16)
    gate = (rng.standard_normal((E, H)) / 64).astype(np.float16)
    gate[3, 5], gate[7, 4100], gate[9, 0], gate[9, 1] = np.nan, np.inf, np.inf, -np.inf
    with np.errstate(invalid="ignore"):
        l = x.astype(np.float64) @ gate.astype(np.float64).T
    assert np.isnan(l[:, 3]).all() and np.isinf(l[:, 7]).all()
    ids, _ = ref.choose(l, None, k)
    gi, gw = torch.empty((S, k), dtype=torch.int32, device=dev), torch.empty((S, k), device=dev)
    gl = torch.empty((S, E), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, logits=gl)
    got = gl.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(l)) and np.array_equal(got[:, 7], l[:, 7].astype(np.float32))
    assert np.array_equal(gi.cpu().numpy(), ids)


def test_experts_apart(K, dev):
    """Experts at a stride larger than an expert, as tensors of a weight blob lie."""
    rng = np.random.default_rng(11)
    S, k, E, H, F = 21, 2, 5, 256, 384
    x = rng.standard_normal((S, H)).astype(np.float16)
    p, s, W = ref.quant(rng, 2 * E, F, H)
    ids = make(rng, S, k, E, H, F)
    pd, sd = t(p, dev).view(E, 2, F, H // 2), t(s, dev).view(E, 2, F, H // 128)
    act = torch.empty((S, k, F), dtype=torch.float16, device=dev)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device=dev)
    K.moe_up_int4(t(x, dev), t(ids, dev), (pd[:, 0], sd[:, 0]), (pd[:, 1], sd[:, 1]), act, S, k, ws)
    want, bound = ref.up(x, ids, W[0::2], W[1::2], k)
    within(act.view(S * k, F).cpu().numpy(), want, bound, "act")


@pytest.mark.parametrize("S", [3, 40, 600])
def test_a_bad_row_stays_alone(K, dev, S):
    """NaN and infinities in one token's row reach no other token's outputs."""
    rng = np.random.default_rng(S)
    k, E, H, F = 2, 4, 256, 256
    x = rng.standard_normal((S, H)).astype(np.float16)
    p1, s1, W1 = ref.quant(rng, E, F, H)
    p2, s2, W2 = ref.quant(rng, E, H, F)
    ids = make(rng, S, k, E, H, F)
    want, bound = ref.up(x, ids, W1, W1, k)
    bad = S // 2
    xb = x.copy()
    xb[bad] = np.nan
    w1 = (t(p1, dev), t(s1, dev))
    act = torch.empty((S, k, F), dtype=torch.float16, device=dev)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device=dev)
    K.moe_up_int4(t(xb, dev), t(ids, dev), w1, w1, act, S, k, ws)
    got = act.cpu().numpy()
    assert np.isnan(got[bad]).all()
    keep = np.arange(S) != bad
    within(got[keep], want.reshape(S, k, F)[keep], bound.reshape(S, k, F)[keep], "act")
    a = got.copy()
    a[bad] = np.inf
    res = np.zeros((S, H), np.float32)
    out = torch.empty((S, H), device=dev)
    K.moe_down_int4(t(a, dev), t(ids, dev), None, (t(p2, dev), t(s2, dev)), t(res, dev), out, S, k, ws)
    o = out.cpu().numpy()
    assert not np.isfinite(o[bad]).any() and np.isfinite(o[keep]).all()


@pytest.mark.parametrize("S,k,E,H,F", [(2300, 4, 16, 512, 1792), (900, 1, 1, 384, 2048), (700, 2, 8, 1024, 384),
                                       (40, 4, 32, 1024, 512)])
def test_passes_without_a_wait(K, dev, S, k, E, H, F):
    """Passes in a row, two sets of inputs in turn, nothing waiting between them: every
    one gives the first one's bits."""
    rng = np.random.default_rng(S)
    sets = []
    for _ in range(2):
        x = t(rng.standard_normal((S, H)).astype(np.float16), dev)
        w = [tuple(t(a, dev) for a in ref.quant(rng, E, r, c)[:2]) for r, c in ((F, H), (F, H), (H, F))]
        ids = t(make(rng, S, k, E, H, F, "even" if E > 1 else "dense"), dev)
        wt = t(rng.random((S, k)).astype(np.float32), dev) if E > 1 else None
        res = t(rng.standard_normal((S, H)).astype(np.float32), dev)
        ws = torch.empty(K.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device=dev)
        sets.append((x, w, ids, wt, res, ws))
    got = [[], []]
    for i in range(24):
        x, w, ids, wt, res, ws = sets[i & 1]
        act = torch.empty((S, k, F), dtype=torch.float16, device=dev)
        out = torch.empty((S, H), device=dev)
        K.moe_up_int4(x, ids, w[0], w[1], act, S, k, ws)
        K.moe_down_int4(act, ids, wt, w[2], res, out, S, k, ws)
        got[i & 1].append((act, out))
    torch.cuda.synchronize()
    for passes in got:
        for act, out in passes[1:]:
            assert torch.equal(act, passes[0][0]) and torch.equal(out, passes[0][1])


# ------------------------------------------------------------------ together
def block(dev, rng, E, k, H, F, max_batch, **kw):
    from cuda_inf_amd.layer import MoeBlock
    (p1, s1, W1), (p3, s3, W3), (p2, s2, W2) = (ref.quant(rng, E, r, c) for r, c in ((F, H), (F, H), (H, F)))
    nw = (1 + 0.2 * rng.standard_normal(H)).astype(np.float16)
    gate = bias = None
    if E > 1:
        gate = (rng.standard_normal((E, H)) / np.sqrt(H)).astype(np.float16)
        bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
        kw.update(gate=t(gate, dev), bias=t(bias, dev), top_k=k)
    B = MoeBlock(t(nw, dev), *((t(p, dev), t(s, dev)) for p, s in ((p1, s1), (p3, s3), (p2, s2))),
                 max_batch=max_batch, device=dev, **kw)
    return B, (nw, gate, bias, W1, W3, W2)


def plain_block(h, w, k, **kw):
    """The branch in 64 bits; what lies between its operators is rounded as they hand it on."""
    nw, gate, bias, W1, W3, W2 = w
    x = ref.norm(h, None, nw, 1e-5)[1].astype(np.float16)
    ids = wt = None
    if gate is not None:
        ids, wt = ref.choose(x.astype(np.float64) @ gate.astype(np.float64).T, bias, k, **kw)
        wt = wt.astype(np.float32)
    act = ref.up(x, ids, W1, W3, k)[0].astype(np.float16)
    return ref.down(act, ids, wt, W2, h, k)[0]


@pytest.mark.parametrize("S,E,k,H,F", [(1, 32, 4, 2048, 256), (6, 8, 3, 256, 384), (50, 1, 1, 256, 512),
                                       (400, 8, 2, 256, 256)])
def test_block(K, dev, S, E, k, H, F):
    rng = np.random.default_rng(S + E)
    B, w = block(dev, rng, E, k, H, F, max_batch=S + 3)
    h = rng.standard_normal((S, H)).astype(np.float32)
    hd = t(h, dev)
    B.forward(hd)
    want = plain_block(h, w, k)
    # an fp16 step of x or act may fall the other way: 2^-10 of some terms of the sums
    err = np.abs(hd.cpu().numpy() - want)
    assert np.linalg.norm(err) <= 2.0 ** -10 * np.linalg.norm(want - h)
    # operators one by one give the branch's bits
    x = torch.empty((S, H), dtype=torch.float16, device=dev)
    act = torch.empty((S, k, F), dtype=torch.float16, device=dev)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device=dev)
    h2 = t(h, dev)
    norm_w, w1, w3, w2, gate, bias = B._keep
    K.add_rmsnorm(h2, norm_w, x, S, H)
    ids = wt = None
    if E > 1:
        ids, wt = torch.empty((S, k), dtype=torch.int32, device=dev), torch.empty((S, k), device=dev)
        K.moe_route(x, gate, ids, wt, S, H, E, k, bias=bias)
    K.moe_up_int4(x, ids, w1, w3, act, S, k, ws)
    K.moe_down_int4(act, ids, wt, w2, h2, h2, S, k, ws)
    assert torch.equal(hd, h2)


def test_layer_of_attention_and_experts(K, dev):
    """Two layers -- norm, attention branch, feed-forward branch -- over a prompt
    and decode tokens, against the plain forms fed with the same attention."""
    from cuda_inf_amd.layer import HIDDEN, AttnLayer
    rng = np.random.default_rng(5)
    E, k, F, prompt = 8, 2, 256, 70
    layers = []
    for _ in range(2):
        L = AttnLayer(256, nsplit=0, max_batch=prompt, device=dev,
                      qk_norm=(torch.ones(64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)))
        proj = []
        for n in (2048, 512, 512, 2048):
            p, s, _ = ref.quant(rng, 1, n, HIDDEN)
            proj.append((t(p[0], dev), t(s[0], dev)))
        L.set_projections(*proj)
        nw = t((1 + 0.2 * rng.standard_normal(HIDDEN)).astype(np.float16), dev)
        B, w = block(dev, rng, E, k, HIDDEN, F, max_batch=prompt)
        layers.append((L, nw, B, w))
    past = 0
    for S in (prompt, 1, 1, 3):
        h = t(rng.standard_normal((S, HIDDEN)).astype(np.float32), dev)
        x = torch.empty((S, HIDDEN), dtype=torch.float16, device=dev)
        for L, nw, B, w in layers:
            K.add_rmsnorm(h, nw, x, S, HIDDEN)
            L.block_forward(x, h, past)
            before = h.cpu().numpy()
            B.forward(h)
            want = plain_block(before, w, k)
            err = np.abs(h.cpu().numpy() - want)
            assert np.linalg.norm(err) <= 2.0 ** -10 * np.linalg.norm(want - before)
        past += S


def test_block_captured(K, dev):
    """A branch in a graph: every replay gives the eager result, with eager calls of
    the same branch between the replays."""
    rng = np.random.default_rng(9)
    for S, E in ((1, 8), (5, 8), (300, 8), (40, 1)):
        k = 2 if E > 1 else 1
        B, _ = block(dev, rng, E, k, 256, 384, max_batch=S)
        hs = [torch.from_numpy(rng.standard_normal((S, 256)).astype(np.float32)).to(dev) for _ in range(3)]
        want = []
        for h in hs:
            o = h.clone()
            B.forward(o)
            want.append(o)
        buf = hs[0].clone()
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                B.forward(buf)
        torch.cuda.synchronize()
        for h, o in zip(hs * 2, want * 2):
            buf.copy_(h)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(buf, o)
            e = h.clone()
            B.forward(e)
            torch.cuda.synchronize()
            assert torch.equal(e, o)


def test_blocks_refusals(K, dev):
    rng = np.random.default_rng(3)
    B, _ = block(dev, rng, 4, 2, 256, 128, max_batch=4, score="softmax", renorm=False, renorm_eps=0.0, scale=1.5)
    B.forward(torch.zeros((0, 256), device=dev))
    for bad, what in ((torch.zeros((5, 256), device=dev), "max_batch"), (torch.zeros((1, 255), device=dev), "fp32"),
                      (torch.zeros((1, 256), dtype=torch.float16, device=dev), "fp32"),
                      (torch.zeros((1, 256)), "device"), (torch.zeros((256, 2), device=dev).t(), "contiguous")):
        with pytest.raises(ValueError, match=what):
            B.forward(bad)
    norm_w, w1, w3, w2, gate, bias = B._keep
    from cuda_inf_amd.layer import MoeBlock
    for args, kw in (((norm_w, w1, w3, w3), dict(gate=gate)), ((norm_w, w1, w3, w2), dict()),
                     ((norm_w[:-1], w1, w3, w2), dict(gate=gate)), ((norm_w, w1, w3, w2), dict(gate=gate.float())),
                     ((norm_w, w1, w3, w2), dict(gate=gate, bias=bias[:2]))):
        with pytest.raises(ValueError):
            MoeBlock(*args, device=dev, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        K.moe_up_int4(norm_w, None, (w1[0][:, :, ::2], w1[1]), w3, norm_w, 1, 1, B.ws)
    with pytest.raises(ValueError, match="do not fit"):
        K.moe_up_int4(norm_w, None, (w1[0], w1[1][:, 1:]), w3, norm_w, 1, 1, B.ws)
    with pytest.raises(ValueError, match="w3: experts"):
        K.moe_up_int4(norm_w, None, w1, w2, norm_w, 1, 1, B.ws)


def test_a_block_for_a_batch_that_no_call_takes(K, dev):
    rng = np.random.default_rng(4)
    for E, k, most in ((4, 2, 1 << 19), (1, 1, 1 << 20)):
        for n in (-1, most + 1):
            with pytest.raises(ValueError, match="max_batch"):
                block(dev, rng, E, k, 128, 128, max_batch=n)


def test_another_stream(K, dev):
    rng = np.random.default_rng(10)
    B, _ = block(dev, rng, 8, 2, 256, 384, max_batch=64)
    h = torch.from_numpy(rng.standard_normal((64, 256)).astype(np.float32)).to(dev)
    want = h.clone()
    B.forward(want)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        B.forward(h)
    s.synchronize()
    assert torch.equal(h, want)


def test_offsets_past_32_bits(K, dev):
    """Rows whose elements lie past the 2^32nd, against the same rows on their own and
    64-bit forms."""
    rng = np.random.default_rng(12)
    S, H, E, k = (1 << 21) + 3, 2056, 8, 2
    assert S * H > 1 << 32
    h = torch.empty((S, H), device=dev).normal_()
    x = torch.empty((S, H), dtype=torch.float16, device=dev)
    w = torch.ones(H, dtype=torch.float16, device=dev)
    gate = t((rng.standard_normal((E, H)) / 45).astype(np.float16), dev)
    K.add_rmsnorm(h, w, x, S, H)
    ids, wt = torch.empty((S, k), dtype=torch.int32, device=dev), torch.empty((S, k), device=dev)
    K.moe_route(x, gate, ids, wt, S, H, E, k)
    for i in (0, S // 2, S - 3):
        o, i1, w1 = torch.empty_like(x[:3]), torch.empty_like(ids[:3]), torch.empty_like(wt[:3])
        K.add_rmsnorm(h[i:i + 3].clone(), w, o, 3, H)
        assert torch.equal(o, x[i:i + 3])
        K.moe_route(o, gate, i1, w1, 3, H, E, k)
        assert torch.equal(i1, ids[i:i + 3])
    del h, x, ids, wt
    S, k, E, n, wide = 1 << 18, 4, 3, 128, 4224
    assert S * k * wide > 1 << 32
    ids = np.stack([rng.permutation(E + 1)[:k] for _ in range(1024)]).astype(np.int32)
    ids = np.tile(ids, (S // 1024, 1))  # (id E: no expert)
    rows = np.array([0, S // 2 + 1, S - 2, S - 1])
    x = t(rng.standard_normal((1024, n)).astype(np.float16), dev).repeat(S // 1024, 1)
    p1, s1, W1 = ref.quant(rng, E, wide, n)
    p3, s3, W3 = ref.quant(rng, E, wide, n)
    act = torch.full((S, k, wide), 3.0, dtype=torch.float16, device=dev)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, n, wide), dtype=torch.uint8, device=dev)
    K.moe_up_int4(x, t(ids, dev), (t(p1, dev), t(s1, dev)), (t(p3, dev), t(s3, dev)), act, S, k, ws)
    want, bound = ref.up(x[rows].cpu().numpy(), ids[rows], W1, W3, k)
    got = act[rows].view(-1, wide).cpu().numpy()
    dead = ids[rows].reshape(-1) == E
    assert (got[dead] == 3.0).all()
    within(got[~dead], want[~dead], bound[~dead], "act")
    del act, ws
    p2, s2, W2 = ref.quant(rng, E, wide, n)
    a = t(rng.standard_normal((1024 * k, n)).astype(np.float16), dev).repeat(S // 1024, 1)
    out = torch.ones((S, wide), device=dev)
    ws = torch.empty(K.moe_workspace_bytes(S, k, E, wide, n), dtype=torch.uint8, device=dev)
    K.moe_down_int4(a, t(ids, dev), None, (t(p2, dev), t(s2, dev)), out, out, S, k, ws)
    want, bound = ref.down(a.view(S, k, n)[rows].view(-1, n).cpu().numpy(), ids[rows], None, W2,
                           np.ones((len(rows), wide), np.float32), k)
    within(out[rows].cpu().numpy(), want, bound, "out")
