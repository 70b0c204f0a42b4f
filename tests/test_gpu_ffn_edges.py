"""Calls of the feed-forward branch at the edges of what its header allows."""
import numpy as np
import pytest
import torch

import ffn_ref as ref
from test_gpu_ffn import block, t, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(cia, dev):
    from cuda_inf_amd import kernels
    return kernels


@pytest.mark.parametrize("S", [1025, 1040])
@pytest.mark.parametrize("E,H,kw", [
    (1, 8, dict(k=1)), (2, 24, dict(k=2)), (16, 520, dict(k=16)), (63, 8, dict(k=5, score="softmax")),
    (64, 520, dict(k=4, score="softmax", renorm=False)), (65, 136, dict(k=7)), (256, 264, dict(k=8)),
    (256, 40, dict(k=16, score="softmax")), (64, 136, dict(k=6, n_group=64, topk_group=6)),
    (256, 264, dict(k=3, n_group=128, topk_group=9, score="softmax")), (72, 520, dict(k=6, n_group=6, topk_group=6))])
@pytest.mark.parametrize("bias", [None, "some", "shut"])
def test_route_of_many_tokens(K, dev, S, E, H, kw, bias):
    """Half of the experts' rows equal to the other half's, or 2^-26 apart; experts that a
    bias shuts or prefers.  Sums are exact in 64 bits, in any order."""
    kw = dict(kw)
    k = kw.pop("k")
    rng = np.random.default_rng(S + E + H)
    x = rng.integers(-2047, 2048, (S, H)) / 1024.0
    gate = rng.integers(-2047, 2048, (E, H)) / 65536.0
    x[:, 3] = rng.integers(-1, 2, S) / 1024.0
    twin = rng.permutation(E)
    gate[twin[E // 2:2 * (E // 2)]] = gate[twin[:E // 2]]
    gate[twin[E // 2:], 3] += rng.integers(0, 2, E - E // 2) / 65536.0
    gate[:, 3] = np.clip(gate[:, 3], -2047 / 65536.0, 2047 / 65536.0)
    x[5] = 0
    x, gate = x.astype(np.float16), gate.astype(np.float16)
    b = None
    if bias:
        b = np.zeros(E, np.float32)
        b[twin[:E // 2]] = b[twin[E // 2:2 * (E // 2)]] = 0.1 * rng.standard_normal(E // 2)
    if bias == "shut":
        b[rng.random(E) < 0.5] = -np.inf
        b[rng.random(E) < 0.1] = 4.0
    l = (x.astype(np.float64) * 2.0 ** 10) @ (gate.astype(np.float64) * 2.0 ** 16).T * 2.0 ** -26
    ids, wt = ref.choose(l, b, k, **kw)
    gi, gw = torch.full((S, k), -7, dtype=torch.int32, device=dev), torch.zeros((S, k), device=dev)
    gl = torch.zeros((S, E), device=dev)
    K.moe_route(t(x, dev), t(gate, dev), gi, gw, S, H, E, k, bias=t(b, dev), logits=gl, **kw)
    wrong = (gi.cpu().numpy() != ids).any(1)
    assert not wrong.any(), f"{wrong.sum()} of {S} tokens, first {np.flatnonzero(wrong)[0]}"
    far = 32 * ref.U24 * (np.abs(x.astype(np.float64)) @ np.abs(gate.astype(np.float64)).T)
    within(gl.cpu().numpy(), l, ref.U24 * np.abs(l) + far, "logits")
    within(gw.cpu().numpy(), wt, ref.weights_bound(l, far, ids, wt, **kw), "weights")


@pytest.mark.parametrize("S,H", [(3, 2048), (2, 8192), (2, 8200), (5, 40)])
def test_norm_sum_into_the_addend(K, dev, S, H):
    g = torch.Generator(device=dev)
    g.manual_seed(S)
    h, b = (torch.randn((S, H), generator=g, device=dev) for _ in range(2))
    w = torch.ones(H, dtype=torch.float16, device=dev)
    out, out2, want = torch.empty((S, H), dtype=torch.float16, device=dev), torch.empty((S, H), dtype=torch.float16, device=dev), h + b
    K.add_rmsnorm(h, w, out, S, H, add=b)
    K.add_rmsnorm(h, w, out2, S, H, add=b, hsum=b)
    assert torch.equal(out, out2) and torch.equal(b, want)


@pytest.mark.parametrize("S,E,k", [(1100, 8, 2), (1100, 1, 1), (5000, 6, 4)])
def test_long_branch_captured(K, dev, S, E, k):
    """The router of many tokens and the plan of many pairs in a graph, replayed with
    eager calls of the same branch between."""
    rng = np.random.default_rng(S + E)
    B, _ = block(dev, rng, E, k, 256, 384, max_batch=S)
    hs = [t(rng.standard_normal((S, 256)).astype(np.float32), dev) for _ in range(3)]
    want = [h.clone() for h in hs]
    for o in want:
        B.forward(o)
    buf, g = hs[0].clone(), torch.cuda.CUDAGraph()
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
