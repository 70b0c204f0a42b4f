"""The feed-forward branch's C-ABI on the CPU: declared symbols, refusals before
any use of a device, workspace sizes, and the Python wrappers' checks."""
import ctypes
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # aligned non-null address: validation must fail before any use
NULL, ALIGN, ARG, OK = 1, 2, 3, 0


@pytest.fixture(scope="module")
def L(cia):
    from cuda_inf_amd import _lib
    return _lib.lib()


def test_every_declared_symbol(L):
    from cuda_inf_amd import _lib
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cuda_inf_ffn.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(cia_[a-z0-9_]+)\s*\(", text))
    assert len(names) == 8
    assert all(hasattr(L, n) for n in names) and names <= set(_lib.SIGNATURES)


@pytest.mark.parametrize("args,code", [
    ((A, None, A, 1e-5, None, A, 0, 64), OK),
    ((None, None, None, 1e-5, None, None, 0, 64), OK),
    ((None, None, A, 1e-5, None, A, 1, 64), NULL),
    ((A, None, None, 1e-5, None, A, 1, 64), NULL),
    ((A, None, A, 1e-5, None, None, 1, 64), NULL),
    ((A, None, A, 1e-5, None, A, -1, 64), ARG),
    ((A, None, A, 1e-5, None, A, 1, 0), ARG),
    ((A, None, A, 1e-5, None, A, 1, 60), ARG),
    ((A, None, A, 1e-5, None, A, 1, (1 << 24) + 8), ARG),
    ((A, None, A, 1e-5, None, A, (1 << 22) + 1, 64), ARG),
    ((A, None, A, -1e-5, None, A, 1, 64), ARG),
    ((A, None, A, float("nan"), None, A, 1, 64), ARG),
    ((A + 8, None, A, 1e-5, None, A, 1, 64), ALIGN),
    ((A, A + 4, A, 1e-5, None, A, 1, 64), ALIGN),
    ((A, None, A + 2, 1e-5, None, A, 1, 64), ALIGN),
    ((A, None, A, 1e-5, A + 4, A, 1, 64), ALIGN),
    ((A, None, A, 1e-5, None, A + 2, 1, 64), ALIGN),
])
def test_norm_refusals(L, args, code):
    assert L.cia_add_rmsnorm(*args, None) == code


GOOD = dict(E=32, k=4, score=0, n_group=1, topk_group=1, renorm=1, eps=1e-6, scale=1.0)


@pytest.mark.parametrize("kw,code", [
    (dict(E=0), ARG), (dict(E=257), ARG), (dict(k=0), ARG), (dict(k=17), ARG), (dict(E=3, k=4), ARG),
    (dict(score=2), ARG), (dict(score=-1), ARG), (dict(n_group=0), ARG), (dict(n_group=5), ARG),
    (dict(n_group=8, topk_group=0), ARG), (dict(n_group=8, topk_group=9), ARG),
    (dict(n_group=16, topk_group=1), ARG),          # 2 experts to choose 4 from
    (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG), (dict(eps=float("inf")), ARG),
    (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG), (dict(), OK),
    (dict(n_group=8, topk_group=1), OK), (dict(scale=-2.0, eps=0.0, renorm=0), OK),
])
def test_gating_refusals(L, kw, code):
    from cuda_inf_amd import _lib
    g = _lib.cia_moe_gating(*{**GOOD, **kw}.values())
    assert L.cia_moe_route(A, A, None, ctypes.byref(g), A, A, None, 0, 64, None) == code
    assert L.cia_moe_select(A, None, ctypes.byref(g), A, A, 0, None) == code


@pytest.mark.parametrize("args,code", [
    ((None, A, None, A, A, None, 1, 64), NULL), ((A, None, None, A, A, None, 1, 64), NULL),
    ((A, A, None, None, A, None, 1, 64), NULL), ((A, A, None, A, None, None, 1, 64), NULL),
    ((A, A, None, A, A, None, -1, 64), ARG), ((A, A, None, A, A, None, 1, 0), ARG),
    ((A, A, None, A, A, None, 1, 68), ARG), ((A, A, None, A, A, None, 1, (1 << 24) + 8), ARG), ((A + 8, A, None, A, A, None, 1, 64), ALIGN),
    ((A, A + 2, None, A, A, None, 1, 64), ALIGN), ((A, A, A + 2, A, A, None, 1, 64), ALIGN),
    ((A, A, None, A + 2, A, None, 1, 64), ALIGN), ((A, A, None, A, A + 1, None, 1, 64), ALIGN),
    ((A, A, None, A, A, A + 2, 1, 64), ALIGN), ((None, None, None, None, None, None, 0, 64), OK),
])
def test_route_refusals(L, args, code):
    from cuda_inf_amd import _lib
    x, gate, bias, ids, w, logits, S, H = args
    g = _lib.cia_moe_gating(*GOOD.values())
    assert L.cia_moe_route(x, gate, bias, ctypes.byref(g), ids, w, logits, S, H, None) == code
    assert L.cia_moe_route(x, gate, bias, None, ids, w, logits, S, H, None) == NULL


@pytest.mark.parametrize("args,code", [
    ((None, None, A, A, 1), NULL), ((A, None, None, A, 1), NULL), ((A, None, A, None, 1), NULL),
    ((A + 2, None, A, A, 1), ALIGN), ((A, A + 1, A, A, 1), ALIGN), ((A, None, A, A, -1), ARG),
])
def test_select_refusals(L, args, code):
    from cuda_inf_amd import _lib
    l, bias, ids, w, S = args
    g = _lib.cia_moe_gating(*GOOD.values())
    assert L.cia_moe_select(l, bias, ctypes.byref(g), ids, w, S, None) == code


def q4(E, rows, cols, **kw):
    from cuda_inf_amd import _lib
    d = dict(packed=A, scales=A, packed_stride=rows * cols // 2, scales_stride=rows * cols // 128)
    return _lib.cia_q4_experts(*{**d, **kw}.values())


EXPERTS = [
    (dict(S=0), OK), (dict(S=0, x=None, act=None, ws=None), OK), (dict(S=-1), ARG), (dict(k=0), ARG),
    (dict(k=17), ARG), (dict(E=0), ARG), (dict(E=257), ARG), (dict(H=0), ARG), (dict(H=192), ARG),
    (dict(F=64), ARG), (dict(F=(1 << 20) + 128), ARG), (dict(S=1 << 23, k=4), ARG),
    (dict(ids=None), ARG),                                 # experts, but nothing chooses
    (dict(x=None), NULL), (dict(act=None), NULL), (dict(ws=None), NULL),
    (dict(x=A + 8), ALIGN), (dict(ids=A + 2), ALIGN), (dict(act=A + 4), ALIGN), (dict(ws=A + 8), ALIGN),
    (dict(ws_less=1), ARG),
    (dict(w=dict(packed=None)), NULL), (dict(w=dict(scales=None)), NULL), (dict(w=dict(packed=A + 8)), ALIGN),
    (dict(w=dict(scales=A + 1)), ALIGN), (dict(w=dict(packed_stride=256 * 128 // 2 + 8)), ALIGN),
    (dict(w=dict(packed_stride=256 * 128 // 2 - 16)), ARG), (dict(w=dict(scales_stride=255)), ARG),
    (dict(w=dict(packed_stride=-(1 << 20))), ARG),
]


def put(kw):
    d = dict(S=3, k=2, E=4, H=256, F=128, ids=A, x=A, act=A, ws=A, ws_less=0, w={}, res=A, out=A, weights=A)
    d.update(kw)
    return d


@pytest.mark.parametrize("kw,code", EXPERTS)
def test_up_refusals(L, kw, code):
    d = put(kw)
    n = L.cia_moe_workspace_bytes(*(d[i] for i in "SkEHF")) - d["ws_less"]
    good, bad = q4(4, 128, 256), q4(4, 128, 256, **d["w"])
    for w1, w3 in ((good, bad), (bad, good)):
        assert L.cia_moe_up_int4(d["x"], d["ids"], ctypes.byref(w1), ctypes.byref(w3), d["act"], d["S"], d["k"],
                                 d["E"], d["H"], d["F"], d["ws"], n, None) == code
    if code == OK:
        return
    assert L.cia_moe_up_int4(A, A, None, ctypes.byref(good), A, 3, 2, 4, 256, 128, A, 1 << 30, None) == NULL


@pytest.mark.parametrize("kw,code", EXPERTS + [
    (dict(res=None), NULL), (dict(out=None), NULL), (dict(res=A + 4), ALIGN), (dict(out=A + 8), ALIGN),
    (dict(weights=A + 2), ALIGN)])
def test_down_refusals(L, kw, code):
    d = put(kw)
    n = L.cia_moe_workspace_bytes(*(d[i] for i in "SkEHF")) - d["ws_less"]
    w2 = q4(4, 256, 128, **d["w"])
    # (up's x is not among down's pointers)
    act = d["act"] if d["x"] == A else d["x"]
    assert L.cia_moe_down_int4(act, d["ids"], d["weights"], ctypes.byref(w2), d["res"], d["out"], d["S"], d["k"],
                               d["E"], d["H"], d["F"], d["ws"], n, None) == code
    assert L.cia_moe_down_int4(A, A, A, None, A, A, 3, 2, 4, 256, 128, A, 1 << 30, None) == NULL


@pytest.mark.parametrize("kw,code", [
    (dict(H=32768, F=32768), OK), (dict(H=32768 + 128), ARG), (dict(F=32768 + 128), ARG), (dict(E=256, k=16), OK),
    (dict(S=1 << 19, k=2, ws_less=1), ARG), (dict(S=(1 << 19) + 1, k=2), ARG)])
def test_limits_of_the_products(L, kw, code):
    """The largest of each argument (of no tokens, or refused for what is looked at
    later), and one more."""
    d = put({"S": 0, **kw})
    n = L.cia_moe_workspace_bytes(*(d[i] for i in "SkEHF")) - d["ws_less"]
    assert (n > 0) == (d["H"] <= 32768 and d["F"] <= 32768)
    w, w2 = q4(d["E"], d["F"], d["H"]), q4(d["E"], d["H"], d["F"])
    sizes = [d[i] for i in "SkEHF"]
    assert L.cia_moe_up_int4(A, A, ctypes.byref(w), ctypes.byref(w), A, *sizes, A, n, None) == code
    assert L.cia_moe_down_int4(A, A, A, ctypes.byref(w2), A, A, *sizes, A, n, None) == code


def test_workspace_bytes(L):
    f = L.cia_moe_workspace_bytes
    assert f(-1, 4, 32, 2048, 1792) == 0 and f(1, 0, 32, 2048, 1792) == 0 and f(1, 4, 0, 2048, 1792) == 0
    assert f(1, 17, 32, 2048, 1792) == f(1, 4, 257, 2048, 1792) == f(1, 4, 32, 40000, 1792) == 0
    # more tokens never need less, and sizes past 32 bits are whole
    last = 0
    for S in (0, 1, 2, 7, 100, 5000, 1 << 20):
        n = f(S, 4, 32, 2048, 1792)
        assert n >= last
        last = n
    assert last > 1 << 32


@pytest.mark.parametrize("H,F", [(192, 1792), (2048, 64), (2049, 128), (2048, 32768 + 128), (32768 + 128, 128)])
def test_workspace_bytes_of_widths_that_no_call_takes(L, H, F):
    from cuda_inf_amd import _lib
    assert L.cia_moe_workspace_bytes(1, 4, 32, H, F) == 0
    M = _lib.cia_moe(H=H, F=F, gate=A, gating=_lib.cia_moe_gating(*GOOD.values()))
    assert L.cia_moe_block_workspace_bytes(ctypes.byref(M), 8) == 0
    M.H, M.F = 32768, 32768  # the widest
    assert L.cia_moe_workspace_bytes(1, 4, 32, 32768, 32768) > 0
    assert L.cia_moe_block_workspace_bytes(ctypes.byref(M), 8) > 0


def test_block_workspace_bytes_of_batches_that_no_call_takes(L):
    from cuda_inf_amd import _lib
    M = _lib.cia_moe(H=2048, F=1792, gate=A, gating=_lib.cia_moe_gating(*GOOD.values()))
    f = L.cia_moe_block_workspace_bytes
    assert f(ctypes.byref(M), 1 << 18) > 1 << 32 and f(ctypes.byref(M), (1 << 18) + 1) == 0
    M.gate = None  # a dense layer: a row a token
    assert f(ctypes.byref(M), 1 << 20) > 1 << 32 and f(ctypes.byref(M), (1 << 20) + 1) == 0


def test_strides_of_one_expert_are_not_read(L):
    w = q4(1, 128, 256, packed_stride=-7, scales_stride=-1)
    n = L.cia_moe_workspace_bytes(1, 1, 1, 256, 128)
    w2 = q4(1, 256, 128, packed_stride=1, scales_stride=0)
    # (refused for what is looked at after the strides)
    assert L.cia_moe_up_int4(A, None, ctypes.byref(w), ctypes.byref(w), A, 1, 1, 1, 256, 128, A, n - 1, None) == ARG
    assert L.cia_moe_down_int4(A, None, None, ctypes.byref(w2), A, A, 1, 1, 1, 256, 128, A, n - 1, None) == ARG


def test_block_refusals(L):
    from cuda_inf_amd import _lib

    def block(**kw):
        M = _lib.cia_moe(norm_w=A, norm_eps=1e-5, H=256, F=128, gate=A, bias=None,
                         gating=_lib.cia_moe_gating(*{**GOOD, "E": 4, "k": 2}.values()), w1=q4(4, 128, 256),
                         w3=q4(4, 128, 256), w2=q4(4, 256, 128), ws=A, cap=8)
        M.ws_bytes = L.cia_moe_block_workspace_bytes(ctypes.byref(M), 8)
        for n, v in kw.items():
            setattr(M, n, v)
        return ctypes.byref(M)

    fwd = L.cia_moe_block_forward
    assert fwd(block(), A, 0, None) == OK
    assert fwd(None, A, 1, None) == NULL and fwd(block(), None, 1, None) == NULL
    assert fwd(block(), A, -1, None) == ARG and fwd(block(), A, 9, None) == ARG
    assert fwd(block(ws=None), A, 1, None) == NULL and fwd(block(ws=A + 8), A, 1, None) == ALIGN
    assert fwd(block(ws_bytes=1), A, 8, None) == ARG
    assert fwd(block(w2=q4(4, 256, 128, packed=None)), A, 1, None) == NULL
    assert fwd(block(w3=q4(4, 256, 128, scales_stride=1)), A, 1, None) == ARG
    assert fwd(block(H=200), A, 1, None) == ARG
    assert fwd(block(norm_w=None), A, 1, None) == NULL
    assert fwd(block(norm_eps=-1.0), A, 1, None) == ARG
    assert fwd(block(gating=_lib.cia_moe_gating(4, 2, 7, 1, 1, 1, 0.0, 1.0)), A, 1, None) == ARG
    assert L.cia_moe_block_workspace_bytes(None, 8) == 0
    assert L.cia_moe_block_workspace_bytes(block(), -1) == 0


def test_block_refuses_a_router_out_of_place_before_any_launch(L):
    from cuda_inf_amd import _lib
    M = _lib.cia_moe(norm_w=A, norm_eps=1e-5, H=256, F=128, gating=_lib.cia_moe_gating(*{**GOOD, "E": 4, "k": 2}.values()),
                     w1=q4(4, 128, 256), w3=q4(4, 128, 256), w2=q4(4, 256, 128), ws=A, ws_bytes=1 << 30, cap=8)
    for gate, bias in ((A + 8, None), (A, A + 2)):
        M.gate, M.bias = gate, bias
        assert L.cia_moe_block_forward(ctypes.byref(M), A, 1, None) == ALIGN


def test_wrapper_refusals(cia):
    import torch

    from cuda_inf_amd import kernels as K
    x = torch.zeros((2, 256), dtype=torch.float16)
    with pytest.raises(ValueError, match="x: must be a device tensor"):
        K.moe_route(x, x, None, None, 2, 256, 4, 2)
    with pytest.raises(ValueError, match="score"):
        K.moe_gating(4, 2, score="tanh")
    with pytest.raises(ValueError, match=r"w1: need two tensors \[experts"):
        K.moe_up_int4(x, None, (x, x), (x, x), x, 2, 1, x)
    with pytest.raises(ValueError, match="w2.packed: must be a device tensor"):
        K.moe_down_int4(x, None, None, (torch.zeros((1, 2, 64), dtype=torch.uint8), x[None]), x, x, 2, 1, x)


def test_choice_oracle():
    """The tests' own choice: hand-made rows."""
    import ffn_ref as ref
    l = np.log(np.array([[0.1, 0.2, 0.3, 0.4]]))
    ids, w = ref.choose(l, None, 2, score="softmax", renorm=False)
    assert ids.tolist() == [[3, 2]] and np.allclose(w, [[0.4, 0.3]])
    ids, w = ref.choose(l, np.array([1, 0, 0, 0], np.float32), 2, score="softmax", eps=0.0)
    assert ids.tolist() == [[0, 3]] and np.allclose(w, [[0.2, 0.8]])
    # groups {0.1, 0.2}, {0.3, 0.4}: the second by its sum
    ids, _ = ref.choose(l, None, 2, score="softmax", n_group=2, topk_group=1)
    assert ids.tolist() == [[3, 2]]
    ids, _ = ref.choose(np.zeros((1, 4)), None, 3)
    assert ids.tolist() == [[0, 1, 2]]


def test_tensors_of_another_device(cia, monkeypatch):
    import torch

    from cuda_inf_amd import kernels as K

    class On(torch.Tensor):  # a tensor that says it is on a device
        is_cuda = True
        index = 0

        def get_device(self):
            return self.index

    def on(t, index):
        t = t.as_subclass(On)
        t.index = index
        return t

    x = on(torch.zeros((2, 256)), 0)
    assert K._at(x, "x", (torch.float32,), 512, 0) == x.data_ptr()
    with pytest.raises(ValueError, match="x: on .*other tensors of the call on cuda:1"):
        K._at(x, "x", (torch.float32,), 512, 1)
    with pytest.raises(ValueError, match="x: needs at least 513"):
        K._at(x, "x", (torch.float32,), 513, 0)
    with pytest.raises(TypeError, match="x: expected a torch.Tensor"):
        K._at(None, "x", (torch.float32,), 512, 0)
    packed, scales = torch.zeros((2, 4, 64), dtype=torch.uint8), torch.zeros((2, 4, 1), dtype=torch.float16)
    q, E, rows, cols = K.q4_experts((on(packed, 0), on(scales, 0)), "w")
    assert (E, rows, cols, q.packed_stride, q.scales_stride) == (2, 4, 128, 256, 4)
    for a, b, dev in ((0, 1, None), (1, 1, 0)):
        with pytest.raises(ValueError, match="w: packed is on"):
            K._q4((on(packed, a), on(scales, b)), "w", dev)
    monkeypatch.setattr(K, "_current_device", lambda: 1)
    with pytest.raises(ValueError, match="the current device is cuda:1"):
        K._stream_on(0)
