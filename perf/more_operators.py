"""A batch's decode step as measurable calls: the paged key-value cache it writes
to and reads from, its attention over that cache, and the choice of each row's token.

Each case is a dict of plain values; ``prepare`` makes what the calling program
holds before the call (inputs, pages, tables, buffers), ``run`` makes one pass --
through the framework's entry points where ``own`` is true, in elementary torch
operations where it is not -- ``work`` states the bytes and operations such a
pass cannot do without, and ``exact`` computes the same outputs in 64 bits.

Kinds
  write   tokens' K and V to their places in the pages, quantised on the way
  read    tokens' K and V back from their places
  attn    one query token per row over the pages of its sequence
  sample  temperature, top-k, top-p and min-p, and a token from a given random number

Token (seq, pos) lies in row pos % page of page table[seq][pos / page].  Pages are
[page, kv head, row, dim] in e4m3, with an fp16 scale per row and kv head
(amax / 448 + 1e-12 before it is rounded), or in fp16.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the cases
def listed():
    # 32 query heads on 8 kv heads of 64, pages of 64 tokens, e4m3
    heads = dict(n_q=32, n_kv=8, D=64, page=64, type="e4m3")
    kv = dict(n_kv=8, D=64, page=64, type="e4m3")
    return [
        # the new token of a single conversation
        dict(name="write_1", kind="write", T=1, rows=1, longest=2000, pad=0, **kv),
        # prompts of several conversations at once, a few places of the batch empty
        dict(name="write_5001", kind="write", T=5001, rows=7, longest=3000, pad=5, **kv),
        # an early part of a conversation back for another turn, small fp16 pages
        dict(name="read_333_f16", kind="read", T=333, rows=1, longest=500, pad=0, n_kv=4, D=128, page=16, type="f16"),
        # a long prefix back
        dict(name="read_8192", kind="read", T=8192, rows=1, longest=8192, pad=0, **kv),
        # a decode token early in a conversation
        dict(name="attn_1_at_700", kind="attn", rows=1, shortest=700, longest=700, pad=0, window=0, **heads),
        # one conversation of 32k tokens
        dict(name="attn_1_at_32768", kind="attn", rows=1, shortest=32768, longest=32768, pad=0, window=0, **heads),
        # a serving batch, conversations of a few to some thousand tokens, three places empty
        dict(name="attn_61_ragged", kind="attn", rows=61, shortest=9, longest=9000, pad=3, window=0, **heads),
        # a large batch of ordinary conversations
        dict(name="attn_256", kind="attn", rows=256, shortest=900, longest=2048, pad=0, window=0, **heads),
        # wider heads in fp16 pages of 16 tokens, the last 1000 tokens attended
        dict(name="attn_33_f16_window", kind="attn", rows=33, shortest=100, longest=4000, pad=0, window=1000, n_q=24,
             n_kv=4, D=128, page=16, type="f16"),
        # a single conversation's token: all three filters
        dict(name="sample_1", kind="sample", rows=1, V=65536, type="f32", filters="kpm", greedy=0.0),
        # a batch of mixed requests, some greedy, over a ragged vocabulary in fp16
        dict(name="sample_47_f16", kind="sample", rows=47, V=50001, type="f16", filters="kp", greedy=0.3),
        # a large batch that samples from the nucleus of a large vocabulary
        dict(name="sample_256", kind="sample", rows=256, V=131072, type="f32", filters="p", greedy=0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "attn", "sample", "sample", "sample"])
    if kind == "sample":
        rows, V = _log_int(rng, 1, 256), _log_int(rng, 50, 131072)
        return dict(kind=kind, rows=rows, V=V, type=rng.choice(["f32", "f32", "f16"]),
                    filters=rng.choice(["", "k", "p", "m", "kp", "kpm"]), greedy=rng.choice([0.0, 0.0, 0.3]))
    n_kv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128])
    page, type = rng.choice([16, 32, 64, 128]), rng.choice(["e4m3", "e4m3", "f16"])
    if kind != "attn":
        T = _log_int(rng, 1, min(16384, 8192 * 512 // (n_kv * D)))
        rows = min(T, _log_int(rng, 1, 64))
        return dict(kind=kind, T=T, rows=rows, longest=-(-T // rows) + rng.randint(0, 2000),
                    pad=rng.randint(0, T // 8), n_kv=n_kv, D=D, page=page, type=type)
    # at most the bytes and the padded tokens of the largest listed case
    rows = _log_int(rng, 1, 256)
    most = 256 * 2048 * 8 * 64 // (n_kv * D * (1 if type == "e4m3" else 2))
    longest = _log_int(rng, 1, min(40000, max(1, most // rows)))
    return dict(kind=kind, rows=rows, shortest=_log_int(rng, 1, longest), longest=longest,
                pad=rng.randint(0, rows // 8), window=rng.choice([0, 0, rng.randint(1, longest)]),
                n_q=n_kv * rng.choice([1, 2, 4, 4, 6, 7, 8, 16]), n_kv=n_kv, D=D, page=page, type=type)


def _lengths(case):
    """Tokens of each row: spread over the logarithm between shortest and longest,
    both among them; none in the last `pad` rows."""
    n, lo, hi = case["rows"], math.log(case["shortest"]), math.log(case["longest"])
    at = [1.0] + [(i * 0.6180339887) % 1.0 for i in range(n - 1)]
    lens = [max(1, int(round(math.exp(lo + f * (hi - lo))))) for f in at]
    return [0 if i >= n - case["pad"] and i else x for i, x in enumerate(lens)]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 64 + 11)
    return g


def _values(g, *shape):
    """K or V as a projection and its norm leave them: some dims far above the others."""
    return torch.randn(shape, generator=g, device="cuda") * (
        0.4 + 3.0 * torch.rand(shape[-1], generator=g, device="cuda") ** 6)


def _pages(case, g, lens):
    """Filled pages in a shuffled order, and the table of lens' sequences (-1 behind a sequence's last)."""
    n_kv, D, page = case["n_kv"], case["D"], case["page"]
    need = [-(-n // page) for n in lens]
    n_pages, width = sum(need) + 4, max(max(need), 1) + 2
    st = dict(page=page)
    for name in "kv":
        x = _values(g, n_pages, n_kv, page, D)
        if case["type"] == "f16":
            st[name], st[name + "s"] = x.half(), None
        else:
            s = x.abs().amax(3) / E4M3_MAX
            st[name] = (x / s[..., None]).to(F8).view(torch.uint8)
            st[name + "s"] = s.half()
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    count = torch.tensor(need, device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    nth = (count.cumsum(0) - count)[:, None] + col
    st["table"] = torch.where(col < count[:, None], order[nth.clamp(max=n_pages - 1)], -1).int().contiguous()
    return st


def prepare(case, seed):
    kind = case["kind"]
    g = _gen(seed)
    if kind == "sample":
        return _prepare_sample(case, g)
    if kind == "attn":
        lens = _lengths(case)
        st = _pages(case, g, lens)
        st["case"] = case
        st["pos"] = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
        # scores of a few units about their mean
        st["q"] = (2.0 * torch.randn((case["rows"], case["n_q"], case["D"]), generator=g, device="cuda")).half()
        st["out"] = torch.empty_like(st["q"])
    else:
        T, rows, per = case["T"], case["rows"], -(-case["T"] // case["rows"])
        st = _pages(case, g, [case["longest"]] * rows)
        st["case"] = case
        # each sequence's last tokens; the places of the batch at its end empty
        t = torch.arange(T, device="cuda")
        st["seq"] = torch.div(t, per, rounding_mode="floor").int()
        pos = (case["longest"] - per + t % per).int()
        pos[T - case["pad"]:] = -1
        st["pos"] = pos
        for name in ("k_new", "v_new"):
            st[name] = _values(g, T, case["n_kv"], case["D"]).half()
    if own:
        from cuda_inf_amd import kernels
        st["pages"] = kernels.KvPages(st["k"], st["v"], st["table"], st["ks"], st["vs"])
        if kind == "attn":
            st["ws"] = kernels.new_attn_pages_workspace(st["pages"], case["n_q"])
    return st


def _prepare_sample(case, g):
    B, V = case["rows"], case["V"]
    r = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    st = dict(case=case)
    # most of a vocabulary is unlikely, a few tokens stand out; some rows surer than others
    x = torch.randn((B, V), generator=g, device="cuda") * (1.2 + 1.6 * r(B, 1))
    x += 6.0 * r(B, V) ** 400 - 3.0
    st["logits"] = x.half() if case["type"] == "f16" else x
    st["u"] = r(B)
    t = 0.6 + 0.7 * r(B)
    st["temperature"] = torch.where(r(B) < case["greedy"], torch.zeros_like(t), t)
    f = case["filters"]
    st["top_k"] = (10 + 190 * r(B)).int() if "k" in f else None
    st["top_p"] = 0.7 + 0.29 * r(B) if "p" in f else None
    st["min_p"] = 0.1 * r(B) if "m" in f else None
    st["ids"] = torch.empty(B, dtype=torch.int32, device="cuda")
    st["p"] = torch.empty(B, device="cuda")
    if own:
        from cuda_inf_amd import kernels
        st["ws"] = torch.empty(kernels.sample_workspace_bytes(B, V), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ one pass
def _place(st):
    """Page and row of each token, and whether it has one."""
    seq, pos, page = st["seq"].long(), st["pos"].long(), st["page"]
    at = torch.div(pos.clamp(min=0), page, rounding_mode="floor").clamp(max=st["table"].shape[1] - 1)
    pid = st["table"].long()[seq, at]
    return pid, pos % page, (pos >= 0) & (pid >= 0)


def _plain_write(st):
    pid, row, ok = _place(st)
    pid, row = pid[ok][:, None], row[ok][:, None]
    head = torch.arange(st["case"]["n_kv"], device="cuda")[None, :]
    outs = []
    for name in "kv":
        x = st[name + "_new"][ok]
        if st[name + "s"] is None:
            st[name][pid, head, row] = x
            outs.append(st[name])
            continue
        x = x.float()
        amax = x.abs().amax(2)
        s = amax / torch.full_like(amax, E4M3_MAX) + 1e-12
        st[name][pid, head, row] = (x / s[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(F8).view(torch.uint8)
        st[name + "s"][pid, head, row] = s.half()
        outs += [st[name].view(F8), st[name + "s"]]
    return outs


def _plain_read(st):
    pid, row, ok = _place(st)
    pid, row = pid[ok][:, None], row[ok][:, None]
    head = torch.arange(st["case"]["n_kv"], device="cuda")[None, :]
    for name in "kv":
        x = st[name][pid, head, row]
        if st[name + "s"] is not None:
            x = (x.view(F8).float() * st[name + "s"][pid, head, row].float()[..., None]).half()
        st[name + "_new"][ok] = x
    return [st["k_new"], st["v_new"]]


def _dense(st, name):
    """Every row's K or V in fp32, [rows, kv heads, tokens, dims], as long as the longest."""
    case, page = st["case"], st["page"]
    idx = st["table"].clamp(min=0).long()
    x = st[name][idx]
    x = x.float() if st[name + "s"] is None else x.view(F8).float() * st[name + "s"][idx].float()[..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(idx.shape[0], case["n_kv"], idx.shape[1] * page, case["D"])


def _plain_attn(st):
    case = st["case"]
    n, n_q, n_kv, D = case["rows"], case["n_q"], case["n_kv"], case["D"]
    q = st["q"].float().view(n, n_kv, n_q // n_kv, D)
    s = torch.matmul(q, _dense(st, "k").transpose(2, 3)) * (1.0 / math.sqrt(D))
    at, pos = torch.arange(s.shape[3], device="cuda")[None, :], st["pos"].long()[:, None]
    ok = at <= pos
    if case["window"]:
        ok &= at > pos - case["window"]
    ok = ok[:, None, None, :]
    s = s.masked_fill(~ok, float("-inf"))
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - top).masked_fill(~ok, 0.0)
    o = torch.matmul(e, _dense(st, "v")) / e.sum(3, keepdim=True).clamp(min=1e-30)
    return o.view(n, n_q, D).half()


def _plain_sample(st):
    # in 64 bits: which token it is must not hang on the order of a sum
    l = st["logits"].double()
    B, V = l.shape
    t = st["temperature"].double()[:, None]
    greedy = t == 0
    l, order = l.sort(dim=1, descending=True, stable=True)
    w = torch.exp((l - l[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    run = w.cumsum(1)
    at = torch.arange(V, device="cuda")[None, :]
    last = torch.full((B, 1), V - 1, device="cuda")
    if st["top_k"] is not None:
        last = torch.minimum(last, st["top_k"].long()[:, None] - 1)
    if st["top_p"] is not None:
        need = st["top_p"].double()[:, None] * run.gather(1, last)
        last = torch.minimum(last, (run < need).sum(1, keepdim=True))
    if st["min_p"] is not None:
        last = torch.minimum(last, (w >= st["min_p"].double()[:, None]).sum(1, keepdim=True) - 1)
    total = run.gather(1, last)
    nth = (run <= st["u"].double()[:, None] * total).sum(1, keepdim=True)
    nth = torch.where(greedy, 0, torch.minimum(nth, last))
    p = torch.where(greedy, 1.0, w.gather(1, nth) / total)
    return [order.gather(1, nth).view(-1).int(), p.view(-1).float()]


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn, "sample": _plain_sample}[kind](st)
    from cuda_inf_amd import kernels
    if kind == "write":
        kernels.kv_pages_write(st["pages"], st["k_new"], st["v_new"], st["pos"], seq=st["seq"])
        if st["ks"] is None:
            return [st["k"], st["v"]]
        return [st["k"].view(F8), st["ks"], st["v"].view(F8), st["vs"]]
    if kind == "read":
        kernels.kv_pages_read(st["pages"], st["k_new"], st["v_new"], st["pos"], seq=st["seq"])
        return [st["k_new"], st["v_new"]]
    if kind == "attn":
        kernels.attn_pages(st["pages"], st["q"], st["out"], st["pos"], st["ws"], scale=1.0 / math.sqrt(case["D"]),
                           window=case["window"])
        return st["out"]
    kernels.sample(st["logits"], st["u"], st["ids"], st["ws"], temperature=st["temperature"], top_k=st["top_k"],
                   top_p=st["top_p"], min_p=st["min_p"], p=st["p"])
    return [st["ids"], st["p"]]


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["V"]
        return dict(bytes=n * (4 if case["type"] == "f32" else 2) + 28 * case["rows"], flops=4.0 * n)
    n_kv, D = case["n_kv"], case["D"]
    token = n_kv * (2 * D + 4 if case["type"] == "e4m3" else 4 * D)  # K and V of a token in the pages
    if kind != "attn":
        n = case["T"] - case["pad"]
        return dict(bytes=n * (4 * n_kv * D + token + 12), flops=4.0 * n * n_kv * D)
    n = sum(min(x, case["window"] or x) for x in _lengths(case))
    return dict(bytes=n * token + 4 * case["rows"] * case["n_q"] * D + n / case["page"] * 4,
                flops=4.0 * n * case["n_q"] * D)


# ------------------------------------------------------------------ in 64 bits
def _stored(st, name):
    """Pages as 64-bit numbers."""
    if st[name + "s"] is None:
        return st[name].double()
    return st[name].view(F8).double() * st[name + "s"].double()[..., None]


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(case, st)
    n_kv, D, page = case["n_kv"], case["D"], case["page"]
    if kind == "attn":
        k, v = _stored(st, "k"), _stored(st, "v")
        out = torch.zeros((case["rows"], n_kv, case["n_q"] // n_kv, D), dtype=torch.float64, device="cuda")
        for i, n in enumerate(_lengths(case)):
            first = max(0, n - case["window"]) if case["window"] else 0
            if n == 0:
                continue
            ids = st["table"][i, first // page:(n - 1) // page + 1].long()
            cut = slice(first % page, first % page + n - first)
            ki, vi = (x[ids].transpose(0, 1).reshape(n_kv, -1, D)[:, cut].contiguous() for x in (k, v))
            q = st["q"][i].double().view(n_kv, -1, D) / D ** 0.5
            a = torch.softmax((q.unsqueeze(2) * ki.unsqueeze(1)).sum(3) if n < 64 else torch.bmm(
                q, ki.transpose(1, 2).contiguous()), dim=2)
            out[i] = torch.bmm(a, vi)
        return out.view(case["rows"], case["n_q"], D)
    live = st["pos"] >= 0
    pos, seq = st["pos"][live].long(), st["seq"][live].long()
    pid, row = st["table"][seq, pos // page].long(), pos % page
    if kind == "read":
        outs = []
        for name in "kv":
            y = st[name + "_new"].double()
            y[live] = _stored(st, name).permute(0, 2, 1, 3)[pid, row]
            outs.append(y)
        return outs
    outs = []
    for name in "kv":
        x = st[name + "_new"][live].double()
        if case["type"] == "f16":
            y = st[name].double()
            y.permute(0, 2, 1, 3)[pid, row] = x
            outs.append(y)
            continue
        s = x.abs().max(dim=2).values / 448 + 1e-12
        y, ys = st[name].view(F8).double(), st[name + "s"].double()
        y.permute(0, 2, 1, 3)[pid, row] = x / s.unsqueeze(2)
        ys.permute(0, 2, 1)[pid, row] = s
        outs += [y, ys]
    return outs


def _exact_sample(case, st):
    l, B = st["logits"].double(), case["rows"]
    p = torch.ones(B, dtype=torch.float64, device="cuda")
    for b in range(B):
        t = float(st["temperature"][b])
        if t == 0:
            continue
        q, _ = torch.sort(torch.softmax(l[b] / t, dim=0), descending=True)
        if st["top_k"] is not None:
            q = q[:int(st["top_k"][b])]
        if st["top_p"] is not None:
            q = q / q.sum()
            before = q.cumsum(0) - q
            q = q[before < float(st["top_p"][b])]
        if st["min_p"] is not None:
            q = q[q >= float(st["min_p"][b]) * q[0]]
        q = q / q.sum()
        p[b] = q[min(int((q.cumsum(0) <= float(st["u"][b])).sum()), q.numel() - 1)]
    return [None, p]
