"""Every kernel and shape of the experts' products on the GPU, against 64-bit forms
computed there, at the sizes of ffn_sizes.py."""
import numpy as np
import pytest
import torch

import ffn_sizes
from ffn_ref import U11, U24

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cia, dev):
    from cuda_inf_amd import kernels
    return kernels


def int4(g, E, rows, cols):
    packed = torch.randint(0, 256, (E, rows, cols // 2), generator=g, device=g.device, dtype=torch.uint8)
    scales = torch.rand((E, rows, cols // 128), generator=g, device=g.device)
    return packed, ((0.02 + 0.2 * scales) / cols ** 0.5).half()


def wide(w, e):
    packed, scales = w[0][e], w[1][e].double()
    nib = torch.stack((packed & 15, packed >> 4), -1).view(packed.shape[0], -1).double() - 8.0
    return nib * scales.repeat_interleave(128, 1)


def by_expert(ids, P, E):
    if ids is None:
        return [(0, torch.arange(P, device="cuda"))]
    flat = ids.view(-1)
    return [(e, r) for e in range(E) if (r := torch.nonzero(flat == e).view(-1)).numel()]


def inside(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[0].tolist()}"


def name(size):
    P, k, E, K, N, rows = size
    return f"{P}of{E}-{K}x{N}" + ("-dense" if rows == "dense" else "-ladder" if rows else "")


def setup(dev, P, k, E, rows, seed):
    ids = ffn_sizes.pair_ids(P, k, E, rows)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    order = torch.randperm(P // k, generator=g, device=dev)
    return None if ids is None else torch.from_numpy(ids).to(dev), g, order


# Bounds: a group's 128 products, a fused add for each of the K / 128 groups, at most
# 16 partial sums that meet (up: half steps of the magnitudes' sum; an fp16 step at the
# end; exp of an argument rounded to fp32 is |g| 2^-23 off, |silu'| <= 1.1).
@pytest.mark.parametrize("size", ffn_sizes.UP, ids=name)
def test_up(K, dev, size):
    P, k, E, H, F, rows = size
    S = P // k
    ids, g, order = setup(dev, P, k, E, rows, P + H + F)
    x = torch.randn((S, H), generator=g, device=dev).half()
    w1, w3 = int4(g, E, F, H), int4(g, E, F, H)
    ws = torch.full((K.moe_workspace_bytes(S, k, E, H, F),), 0xAB, dtype=torch.uint8, device=dev)
    act = torch.full((S, k, F), 3.0, dtype=torch.float16, device=dev)
    K.moe_up_int4(x, ids, w1, w3, act, S, k, ws)
    n = (128 + H / 128 + 20) * U24
    live = torch.zeros(P, dtype=torch.bool, device=dev)
    for e, r in by_expert(ids, P, E):
        live[r] = True
        xd, A, B = x[r // k].double(), wide(w1, e), wide(w3, e)
        a, u = xd @ A.t(), xd @ B.t()
        da, du = n * (xd.abs() @ A.abs().t()), n * (xd.abs() @ B.abs().t())
        silu = a / (1.0 + torch.exp(-a))
        want = silu * u
        bound = (want.abs() * (U11 * 1.001 + (a.abs() + 8.0) * 2 * U24) + 1.1 * da * (u.abs() + du)
                 + (silu.abs() + 1.1 * da) * du + 2.0 ** -25)
        inside(act.view(P, F)[r], want, bound, f"expert {e}")
    assert (act.view(P, F)[~live] == 3.0).all(), "rows of pairs that take no part were written"
    # the same tokens in another order: the same bits for each
    act2 = torch.full_like(act, 3.0)
    K.moe_up_int4(x[order], None if ids is None else ids[order].contiguous(), w1, w3, act2, S, k, ws)
    assert torch.equal(act2, act[order])


@pytest.mark.parametrize("size", ffn_sizes.DOWN, ids=name)
@pytest.mark.parametrize("weighted", [True, False])
def test_down(K, dev, size, weighted):
    P, k, E, F, H, rows = size
    S = P // k
    ids, g, order = setup(dev, P, k, E, rows, P + H + F + 1)
    act = torch.randn((S, k, F), generator=g, device=dev).half()
    w2 = int4(g, E, H, F)
    wt = torch.randn((S, k), generator=g, device=dev) if weighted else None
    res = torch.randn((S, H), generator=g, device=dev)
    ws = torch.full((K.moe_workspace_bytes(S, k, E, H, F),), 0xFF, dtype=torch.uint8, device=dev)
    want, mag, bound = res.double(), res.double().abs(), torch.zeros((S, H), dtype=torch.float64, device=dev)
    n = (128 + F / 128 + 20) * U24
    live = torch.zeros(P, dtype=torch.bool, device=dev)
    for e, r in by_expert(ids, P, E):
        live[r] = True
        a, W = act.view(P, F)[r].double(), wide(w2, e)
        c = torch.ones((len(r), 1), device=dev).double() if wt is None else wt.view(-1)[r].double()[:, None]
        y, b = c * (a @ W.t()), n * c.abs() * (a.abs() @ W.abs().t())
        for t, v in ((want, y), (mag, y.abs()), (bound, b)):
            t.index_add_(0, r // k, v)
    act.view(P, F)[~live] = float("nan")
    out = torch.full((S, H), 5.0, device=dev)
    K.moe_down_int4(act, ids, wt, w2, res, out, S, k, ws)
    inside(out, want, bound + (k + 3) * U24 * mag, "out")
    out2 = res[order]  # in place, the tokens in another order
    K.moe_down_int4(act[order], None if ids is None else ids[order].contiguous(), None if wt is None else wt[order],
                    w2, out2, out2, S, k, ws)
    assert torch.equal(out2, out[order])
