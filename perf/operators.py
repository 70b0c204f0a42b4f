"""The feed-forward half of a layer as measurable calls: the norm that feeds it,
the router, and the experts' INT4 products.

Each case is a dict of plain values; ``prepare`` makes what the calling program
holds before the call (inputs, weights, buffers), ``run`` makes one pass --
through the framework's entry points where ``own`` is true, in elementary torch
operations where it is not -- ``work`` states the bytes and operations such a
pass cannot do without, and ``exact`` computes the same outputs in 64 bits.

Kinds
  norm   residual addition and RMSNorm: h + add in fp32, and its norm in fp16
  route  router product, scores, choice of k experts and their weights
  up     the chosen experts' gate and up products with SwiGLU between them
  down   the chosen experts' down products, weighted and added to the residual

INT4 weights have one fp16 scale per 128 inputs: w = (nibble - 8) * scale.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5       # of the norm
RENORM = 1e-6    # added to the sum of the chosen scores
GROUP = 128      # inputs per INT4 scale


# ------------------------------------------------------------------ the cases
def listed():
    # hidden size 2048; 32 experts of 1792, 4 to a token; the dense form is one
    # expert that takes every row
    moe = dict(E=32, k=4, H=2048, F=1792)
    return [
        # a decode token: the residual alone, no addition
        dict(name="norm_1", kind="norm", S=1, H=2048, add=False),
        # a long prompt, another branch's output added first
        dict(name="norm_4096_add", kind="norm", S=4096, H=2048, add=True),
        # a decode token's router: sigmoid scores, a bias for balance
        dict(name="route_1", kind="route", S=1, H=2048, E=32, k=4, score="sigmoid", bias=True,
             n_group=1, topk_group=1, renorm=True),
        # a ragged prompt through a finer-grained router with expert groups
        dict(name="route_301_groups", kind="route", S=301, H=1280, E=128, k=6, score="softmax",
             bias=False, n_group=8, topk_group=3, renorm=False),
        # a long prompt's router
        dict(name="route_4096", kind="route", S=4096, H=2048, E=32, k=4, score="sigmoid", bias=True,
             n_group=1, topk_group=1, renorm=True),
        # a decode token through its 4 experts
        dict(name="up_1", kind="up", S=1, pad=0, **moe),
        # a batch of decode tokens, three places of the batch empty
        dict(name="up_45", kind="up", S=45, pad=3, **moe),
        # a long prompt, the experts' shares as uneven as routers make them
        dict(name="up_4096", kind="up", S=4096, pad=0, **moe),
        dict(name="down_1", kind="down", S=1, pad=0, **moe),
        dict(name="down_45", kind="down", S=45, pad=3, **moe),
        dict(name="down_4096", kind="down", S=4096, pad=0, **moe),
        # the dense form over an ordinary prompt
        dict(name="down_700_dense", kind="down", S=700, pad=0, E=1, k=1, H=2048, F=7168),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "route", "route", "up", "up", "up", "down", "down", "down"])
    if kind == "norm":
        H = 8 * _log_int(rng, 8, 1024)
        return dict(kind=kind, S=_log_int(rng, 1, min(16384, 2 ** 23 // H)), H=H,
                    add=rng.random() < 0.5)
    if kind == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        E = n_group * _log_int(rng, 4, 256 // n_group)
        topk_group = rng.randint(1, n_group)
        H = 128 * _log_int(rng, 2, 32)
        most = min(16384, 4096 * 32 * 2048 // (E * H))
        return dict(kind=kind, S=_log_int(rng, 1, most), H=H, E=E,
                    k=rng.randint(1, min(8, E // n_group * topk_group)),
                    score=rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.5,
                    n_group=n_group, topk_group=topk_group, renorm=rng.random() < 0.5)
    dense = rng.random() < 0.2
    E = 1 if dense else _log_int(rng, 4, 64)
    k = 1 if dense else rng.randint(1, min(8, E))
    H, F = 128 * _log_int(rng, 2, 32), 128 * _log_int(rng, 2, 56 if dense else 32)
    # at most the weights and the operations of the largest listed case
    E = max(1 if dense else k, min(E, 32 * 1792 * 2048 // (H * F)))
    most = max(1, min(4096, 4096 * 4 * 1792 * 2048 // (k * H * F), 4096 * 4 * 1792 // (k * F),
                      4096 * 2048 // H))
    S = _log_int(rng, 1, most)
    return dict(kind=kind, S=S, pad=0 if dense or rng.random() < 0.5 else rng.randint(0, S // 8),
                E=E, k=k, H=H, F=F)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int4(g, E, rows, cols):
    """INT4 weights of E experts: bytes [E, rows, cols / 2], scales [E, rows, cols / 128]."""
    packed = torch.randint(0, 256, (E, rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand((E, rows, cols // GROUP), generator=g, device="cuda")
    # as large as keeps the products of order one, some groups ten times others
    return packed, ((0.02 + 0.2 * scales) / math.sqrt(cols)).half()


def prepare(case, seed):
    kind, S, H = case["kind"], case["S"], case["H"]
    g = _gen(seed * 64 + 5)
    st = dict(case=case)
    if kind == "norm":
        # a residual stream: some channels far above the others
        st["h"] = torch.randn((S, H), generator=g, device="cuda") * (
            0.5 + 4.0 * torch.rand(H, generator=g, device="cuda") ** 8)
        st["add"] = torch.randn((S, H), generator=g, device="cuda") if case["add"] else None
        st["w"] = (1.0 + 0.2 * torch.randn(H, generator=g, device="cuda")).half()
        st["sum"] = torch.empty_like(st["h"]) if case["add"] else None
        st["out"] = torch.empty((S, H), dtype=torch.float16, device="cuda")
        return st
    E, k = case["E"], case["k"]
    if kind == "route":
        st["x"] = torch.randn((S, H), generator=g, device="cuda").half()
        st["gate"] = (torch.randn((E, H), generator=g, device="cuda") / math.sqrt(H)).half()
        st["bias"] = 0.1 * torch.randn(E, generator=g, device="cuda") if case["bias"] else None
        st["ids"] = torch.empty((S, k), dtype=torch.int32, device="cuda")
        st["weights"] = torch.empty((S, k), device="cuda")
        st["logits"] = torch.empty((S, E), device="cuda")
        return st
    F = case["F"]
    if case["E"] > 1:
        # experts' popularity as routers leave it, several times between first and last
        lean = 0.7 * torch.randn(E, generator=g, device="cuda")
        score = lean + torch.randn((S, E), generator=g, device="cuda")
        top, ids = score.topk(k, dim=1)
        st["ids"] = ids.int().contiguous()
        st["weights"] = torch.softmax(top, dim=1).contiguous()
        if case["pad"]:
            st["ids"][S - case["pad"]:] = -1
    else:
        st["ids"] = st["weights"] = None
    if kind == "up":
        st["x"] = torch.randn((S, H), generator=g, device="cuda").half()
        st["w1"], st["w3"] = _int4(g, E, F, H), _int4(g, E, F, H)
        st["act"] = torch.zeros((S, k, F), dtype=torch.float16, device="cuda")
    else:
        a, b = (torch.randn((S, k, F), generator=g, device="cuda") for _ in range(2))
        st["act"] = (a * torch.sigmoid(a) * b).half()
        st["w2"] = _int4(g, E, H, F)
        st["res"] = torch.randn((S, H), generator=g, device="cuda")
        st["out"] = torch.empty_like(st["res"])
    if own:
        from cuda_inf_amd import kernels
        st["ws"] = torch.zeros(kernels.moe_workspace_bytes(S, k, E, H, F), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ one pass
def _dense(w, e):
    """Expert e's INT4 weights as fp32 [rows, cols]."""
    packed, scales = w[0][e], w[1][e]
    nib = torch.stack((packed & 15, packed >> 4), dim=-1).view(packed.shape[0], -1, GROUP)
    return ((nib.float() - 8.0) * scales.float()[:, :, None]).view(packed.shape[0], -1)


def _choose(score, choice, case):
    """The k experts of largest choice (the lowest index first among equals), and their scores."""
    E, k, ng = case["E"], case["k"], case["n_group"]
    if ng > 1:
        # the groups by the sum of their two best choices, the other groups left out
        best = choice.view(-1, ng, E // ng).sort(dim=2, descending=True).values[..., :2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case["topk_group"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = choice.masked_fill(~mask.repeat_interleave(E // ng, dim=1), float("-inf"))
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    return ids, score.gather(1, ids)


def _plain_norm(st):
    h = st["h"] if st["add"] is None else st["h"] + st["add"]
    y = (h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * st["w"].float()).half()
    return [y] if st["add"] is None else [y, h]


def _plain_route(st):
    # in 64 bits: whether an expert is chosen must not hang on the order of a sum
    case = st["case"]
    logits = st["x"].double() @ st["gate"].double().t()
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        score = p / p.sum(1, keepdim=True)
    choice = score if st["bias"] is None else score + st["bias"].double()
    ids, w = _choose(score, choice, case)
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + RENORM)
    return [ids.int(), w.float(), logits.float()]


def _rows(st):
    """(expert, its rows of the S * k) for the experts that have any; a row's token is row // k."""
    case = st["case"]
    if st["ids"] is None:
        return [(0, torch.arange(case["S"], device="cuda"))]
    flat = st["ids"].view(-1)
    return [(e, torch.nonzero(flat == e).view(-1)) for e in torch.unique(flat).tolist() if e >= 0]


def _plain_up(st):
    case = st["case"]
    act = torch.zeros((case["S"] * case["k"], case["F"]), dtype=torch.float16, device="cuda")
    for e, rows in _rows(st):
        x = st["x"][rows // case["k"]].float()
        a, b = x @ _dense(st["w1"], e).t(), x @ _dense(st["w3"], e).t()
        act[rows] = (a / (1.0 + torch.exp(-a)) * b).half()
    return act.view(case["S"], case["k"], case["F"])


def _plain_down(st):
    case = st["case"]
    act = st["act"].view(-1, case["F"])
    y = torch.zeros((case["S"] * case["k"], case["H"]), device="cuda")
    for e, rows in _rows(st):
        y[rows] = act[rows].float() @ _dense(st["w2"], e).t()
    if st["weights"] is not None:
        y = y * st["weights"].view(-1, 1)
    return st["res"] + y.view(case["S"], case["k"], -1).sum(1)


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"norm": _plain_norm, "route": _plain_route, "up": _plain_up, "down": _plain_down}[kind](st)
    from cuda_inf_amd import kernels
    S, H = case["S"], case["H"]
    if kind == "norm":
        kernels.add_rmsnorm(st["h"], st["w"], st["out"], S, H, EPS, add=st["add"], hsum=st["sum"])
        return [st["out"]] if st["add"] is None else [st["out"], st["sum"]]
    if kind == "route":
        kernels.moe_route(st["x"], st["gate"], st["ids"], st["weights"], S, H, case["E"], case["k"],
                          bias=st["bias"], score=case["score"], n_group=case["n_group"],
                          topk_group=case["topk_group"], renorm=case["renorm"], eps=RENORM,
                          logits=st["logits"])
        return [st["ids"], st["weights"], st["logits"]]
    if kind == "up":
        kernels.moe_up_int4(st["x"], st["ids"], st["w1"], st["w3"], st["act"], S, case["k"], st["ws"])
        return st["act"]
    kernels.moe_down_int4(st["act"], st["ids"], st["weights"], st["w2"], st["res"], st["out"], S,
                          case["k"], st["ws"])
    return st["out"]


# ------------------------------------------------------------------ work
def _w_bytes(rows, cols):
    return rows * (cols // 2 + 2 * cols // GROUP)


def _active(S, E, k):
    """Experts that S tokens of k choices reach, on average, were all equally liked."""
    return E * (1.0 - (1.0 - k / E) ** S)


def work(case):
    kind, S, H = case["kind"], case["S"], case["H"]
    if kind == "norm":
        # h (and add) in, the norm (and the sum) out
        return dict(bytes=S * H * (4 + 2 + (8 if case["add"] else 0)) + 2 * H, flops=5.0 * S * H)
    E, k = case["E"], case["k"]
    if kind == "route":
        return dict(bytes=2 * S * H + 2 * E * H + S * (8 * k + 4 * E), flops=2.0 * S * H * E)
    F, rows = case["F"], (S - case["pad"]) * k
    n = _active(S - case["pad"], E, k)
    if kind == "up":
        return dict(bytes=n * _w_bytes(2 * F, H) + 2 * S * H + 2 * rows * F + 4 * S * k,
                    flops=2.0 * rows * 2 * F * H)
    return dict(bytes=n * _w_bytes(H, F) + 2 * rows * F + 8 * S * H + 8 * S * k,
                flops=2.0 * rows * F * H)


# ------------------------------------------------------------------ in 64 bits
def _groups(w, e, x):
    """x [n, cols] times expert e's weights, scale group by scale group."""
    packed, scales = (t[e] for t in w)
    y = torch.zeros((x.shape[0], packed.shape[0]), dtype=torch.float64, device="cuda")
    q = torch.empty((packed.shape[0], packed.shape[1] * 2), dtype=torch.float64, device="cuda")
    q[:, 0::2] = packed.bitwise_and(15)
    q[:, 1::2] = packed.bitwise_right_shift(4)
    q -= 8.0
    for i in range(scales.shape[1]):
        at = slice(i * GROUP, (i + 1) * GROUP)
        y += (x[:, at].double() @ q[:, at].t()) * scales[:, i].double()
    return y


def _by_expert(case, ids):
    """(expert, its rows) again, from the rows in order of their experts."""
    if ids is None:
        return [(0, torch.arange(case["S"], device="cuda"))]
    flat = ids.reshape(-1).long() + 1
    order = torch.argsort(flat, stable=True)
    parts = torch.split(order, torch.bincount(flat, minlength=case["E"] + 1).tolist())
    return [(e, r) for e, r in enumerate(parts[1:]) if r.numel()]


def exact(case, seed):
    st = prepare(case, seed)
    kind, S, k = case["kind"], case["S"], case.get("k", 1)
    if kind == "norm":
        h = st["h"].double() + (0.0 if st["add"] is None else st["add"].double())
        y = h / (h.pow(2).sum(1, keepdim=True) / case["H"] + EPS).sqrt() * st["w"].double()
        return [y] if st["add"] is None else [y, h]
    if kind == "route":
        x, gate = st["x"].double(), st["gate"].double()
        logits = (x[:, None, :] * gate[None]).sum(2) if S * case["E"] * case["H"] < 2 ** 27 else x @ gate.t()
        s = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, dim=1)
        c = s.clone() if st["bias"] is None else s + st["bias"].double()
        ng = case["n_group"]
        if ng > 1:
            per = case["E"] // ng
            of = torch.arange(case["E"], device="cuda") // per
            t = torch.stack([c[:, of == i].topk(min(2, per), dim=1).values.sum(1) for i in range(ng)], dim=1)
            keep = torch.zeros_like(t, dtype=torch.bool)
            for _ in range(case["topk_group"]):
                keep.scatter_(1, t.masked_fill(keep, float("-inf")).argmax(1, keepdim=True), True)
            c[~keep[:, of]] = float("-inf")
        w = c.new_empty((S, k))
        for j in range(k):
            at = c.argmax(1, keepdim=True)
            w[:, j:j + 1] = s.gather(1, at)
            c.scatter_(1, at, float("-inf"))
        if case["renorm"]:
            w = w / (w.sum(1, keepdim=True) + RENORM)
        return [None, w, logits]
    F = case["F"]
    if kind == "up":
        act = torch.zeros((S * k, F), dtype=torch.float64, device="cuda")
        for e, r in _by_expert(case, st["ids"]):
            x = st["x"][torch.div(r, k, rounding_mode="floor")]
            a = _groups(st["w1"], e, x)
            act[r] = a * torch.sigmoid(a) * _groups(st["w3"], e, x)
        return act.view(S, k, F)
    out = st["res"].double()
    for e, r in _by_expert(case, st["ids"]):
        y = _groups(st["w2"], e, st["act"].view(S * k, F)[r])
        if st["weights"] is not None:
            y *= st["weights"].reshape(-1)[r].double()[:, None]
        out.index_add_(0, torch.div(r, k, rounding_mode="floor"), y)
    return out
