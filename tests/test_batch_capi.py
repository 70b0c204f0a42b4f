"""The paged cache, its attention and sampling on the CPU: declared symbols, refusals
before any use of a device, workspace sizes, the Python wrappers' checks, and the
tests' own plain forms."""
import ctypes
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # aligned non-null address: validation must fail before any use
OK, NULL, ALIGN, ARG = 0, 1, 2, 3
GOOD = dict(k=A, v=A, ks=A, vs=A, type=0, n_pages=10, page=64, n_kv=8, head_dim=64, n_seq=4, max_pages=6, table=A,
            table_stride=6)


@pytest.fixture(scope="module")
def L(cia):
    from cuda_inf_amd import _lib
    return _lib.lib()


def pages(**kw):
    from cuda_inf_amd import _lib
    return ctypes.byref(_lib.cia_kv_pages(*{**GOOD, **kw}.values()))


def test_every_declared_symbol(L):
    from cuda_inf_amd import _lib
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cuda_inf_batch.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(cia_[a-z0-9_]+)\s*\(", text))
    assert len(names) == 6
    assert all(hasattr(L, n) for n in names) and names <= set(_lib.SIGNATURES)


def calls(L, P, T=1):
    """The status of each call over P with good other arguments."""
    big = 1 << 40
    return [L.cia_kv_pages_write(P, A, 512 * 32, A, 512 * 32, A, A, T, None),
            L.cia_kv_pages_read(P, A, 512 * 32, A, 512 * 32, A, A, T, None),
            L.cia_attn_pages(P, A, 4096 * 32, A, A, T, 32, 0.125, 0, A, A, big, None)]


@pytest.mark.parametrize("kw,code", [
    (dict(type=2), ARG), (dict(type=-1), ARG), (dict(n_pages=0), ARG), (dict(n_seq=0), ARG), (dict(max_pages=0), ARG),
    (dict(page=8), ARG), (dict(page=48), ARG), (dict(page=2048), ARG), (dict(page=0), ARG), (dict(page=-16), ARG),
    (dict(n_kv=0), ARG), (dict(n_kv=129), ARG), (dict(head_dim=32), ARG), (dict(head_dim=96), ARG),
    (dict(table_stride=5), ARG), (dict(max_pages=1 << 20, table_stride=1 << 20), ARG),
    (dict(max_pages=2 ** 31 - 1, table_stride=2 ** 31), ARG),
])
def test_pages_refused_in_every_call(L, kw, code):
    # (also where there is no work)
    assert calls(L, pages(**kw)) == [code] * 3
    assert calls(L, pages(**kw), T=0) == [code] * 3


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(ks=None), NULL), (dict(vs=None), NULL), (dict(table=None), NULL),
    (dict(k=A + 8), ALIGN), (dict(v=A + 4), ALIGN), (dict(ks=A + 1), ALIGN), (dict(vs=A + 1), ALIGN), (dict(table=A + 2), ALIGN),
])
def test_pages_pointers(L, kw, code):
    assert calls(L, pages(**kw)) == [code] * 3
    assert calls(L, pages(**kw), T=0) == [OK] * 3
    assert calls(L, None) == [NULL] * 3


def test_largest_cache_without_work(L):
    assert calls(L, pages(max_pages=1 << 15, page=1024, table_stride=1 << 40, n_kv=8, n_pages=2 ** 31 - 1), T=0) == [OK] * 3


@pytest.mark.parametrize("args,code", [
    ((A, 512, A, 512, A, A, -1), ARG), ((A, 512, A, 512, A, A, (1 << 22) + 1), ARG),
    ((A, 504, A, 512, A, A, 1), ARG), ((A, 512, A, 504, A, A, 1), ARG), ((A, 516, A, 512, A, A, 1), ARG),
    ((A, 512, A, 516, A, A, 1), ARG), ((A, -512, A, 512, A, A, 1), ARG),
    ((A, 512, A, 512, None, A, 5), ARG),  # token t of sequence t: 4 sequences
    ((None, 512, A, 512, A, A, 1), NULL), ((A, 512, None, 512, A, A, 1), NULL), ((A, 512, A, 512, A, None, 1), NULL),
    ((A + 8, 512, A, 512, A, A, 1), ALIGN), ((A, 512, A + 2, 512, A, A, 1), ALIGN),
    ((A, 512, A, 512, A + 2, A, 1), ALIGN), ((A, 512, A, 512, A, A + 1, 1), ALIGN),
    ((None, 512, None, 512, None, None, 0), OK),
])
def test_move_refusals(L, args, code):
    assert L.cia_kv_pages_write(pages(), *args, None) == code
    assert L.cia_kv_pages_read(pages(), *args, None) == code


def test_attn_refusals(L):
    n = L.cia_attn_pages_workspace_bytes(32, 8, 64)
    good = dict(q=A, q_stride=2048, seq=A, pos=A, T=1, n_q=32, scale=0.125, window=0, out=A, ws=A, ws_bytes=n)
    f = lambda **kw: L.cia_attn_pages(pages(), *{**good, **kw}.values(), None)  # noqa: E731
    for kw in (dict(T=-1), dict(T=4097), dict(n_q=0), dict(n_q=33), dict(n_q=4), dict(n_q=-8), dict(n_q=8 * 65, q_stride=1 << 20),
               dict(q_stride=2040), dict(q_stride=2052), dict(window=-1), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(scale=float("-inf")), dict(scale=1.0001 * 2.0 ** 64), dict(scale=-1e30),
               dict(ws_bytes=n - 1), dict(ws_bytes=0),
               dict(seq=None, T=5)):
        assert f(**kw) == ARG, kw
    for kw in (dict(q=None), dict(pos=None), dict(out=None), dict(ws=None)):
        assert f(**kw) == NULL, kw
    for kw in (dict(q=A + 8), dict(seq=A + 1), dict(pos=A + 2), dict(out=A + 2), dict(ws=A + 4)):
        assert f(**kw) == ALIGN, kw
    assert f(T=0, q=None, seq=None, pos=None, out=None, ws=None, ws_bytes=0) == OK


def test_attn_workspace(L):
    f = L.cia_attn_pages_workspace_bytes
    for n_q, n_kv, D in ((0, 1, 64), (8, 0, 64), (8, 129, 64), (8, 3, 64), (65, 1, 64), (8, 8, 32), (-8, 8, 64),
                         (8, -8, 64), (4, 8, 64)):
        assert f(n_q, n_kv, D) == 0
    for n_q, n_kv, D in ((1, 1, 64), (64, 1, 128), (128 * 64, 128, 128), (32, 8, 64)):
        assert f(n_q, n_kv, D) > 0


def test_sample_refusals(L):
    n = L.cia_sample_workspace_bytes(3, 100)
    good = dict(logits=A, type=0, stride=100, temperature=A, top_k=A, top_p=A, min_p=A, u=A, ids=A, p=A, B=3, V=100,
                ws=A, ws_bytes=n)
    f = lambda **kw: L.cia_sample(*{**good, **kw}.values(), None)  # noqa: E731
    for kw in (dict(type=2), dict(type=-1), dict(stride=99), dict(stride=-100), dict(B=-1), dict(B=(1 << 16) + 1),
               dict(V=0), dict(V=-1), dict(B=1 << 16, V=(1 << 18) + 1, stride=1 << 20), dict(V=(1 << 22) + 1, stride=1 << 23), dict(ws_bytes=n - 1)):
        assert f(**kw) == ARG, kw
    for kw in (dict(logits=None), dict(u=None), dict(ids=None), dict(ws=None)):
        assert f(**kw) == NULL, kw
    for kw in (dict(logits=A + 2), dict(logits=A + 1, type=1), dict(temperature=A + 1), dict(top_k=A + 2), dict(top_p=A + 2),
               dict(min_p=A + 2), dict(u=A + 2), dict(ids=A + 2), dict(p=A + 2), dict(ws=A + 8)):
        assert f(**kw) == ALIGN, kw
    assert f(B=0, logits=None, u=None, ids=None, ws=None, ws_bytes=L.cia_sample_workspace_bytes(0, 100)) == OK


def test_sample_workspace(L):
    f = L.cia_sample_workspace_bytes
    assert f(-1, 10) == f(1, 0) == f((1 << 16) + 1, 10) == f(1, (1 << 22) + 1) == 0
    assert f(1, 1) > 0 and f(1 << 12, 1 << 22) >= f(1 << 10, 1 << 22) >= f(1, 1 << 22) > 0 and f(1 << 16, 1 << 18) > 0
    assert f((1 << 12) + 1, 1 << 22) == f(1 << 16, (1 << 18) + 1) == 0  # (more than 2^34 logits)
    # (a smaller batch of the same rows fits what a larger one was given)
    for V in (1, 17, 4096, 16385, 65536, 131073):
        last = 0
        for B in range(1, 1100):
            n = f(B, V)
            assert n >= last
            last = n


def test_wrapper_checks(cia, monkeypatch):
    import torch

    from cuda_inf_amd import kernels as K
    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="k: need a tensor"):
        K.KvPages(k[0], k, None)
    with pytest.raises(ValueError, match="k: need a tensor"):
        K.KvPages(None, k, None)
    with pytest.raises(TypeError, match="k: dtype"):
        K.KvPages(k.float(), k, None)
    with pytest.raises(ValueError, match="k: must be a device tensor"):
        K.KvPages(k, k, torch.zeros((1, 1), dtype=torch.int32))
    for bad in (None, k[0, 0, 0], k.int()[0, 0], k[0, 0].double()):
        with pytest.raises(ValueError, match="logits: need a device tensor"):
            K.sample(bad, None, None, None)
    with pytest.raises(ValueError, match="logits: need a device tensor"):
        K.sample(torch.zeros((2, 8)), None, None, None)

    class On(torch.Tensor):  # a tensor that says it is on device 0
        is_cuda = True

        def get_device(self):
            return 0

    def on(t):
        return t.as_subclass(On)

    t = on(torch.zeros((3, 5), dtype=torch.int32))
    u8, sc = on(torch.zeros((4, 2, 16, 64), dtype=torch.uint8)), on(torch.zeros((4, 2, 16), dtype=torch.float16))
    P = K.KvPages(on(k), on(k), t[:, :4])
    assert (P._s.type, P._s.n_pages, P._s.page, P._s.n_kv, P._s.head_dim, P._s.n_seq, P._s.max_pages,
            P._s.table_stride) == (1, 4, 16, 2, 64, 3, 4, 5)
    P = K.KvPages(u8, u8, t[:1], sc, sc)
    assert (P._s.type, P._s.table_stride, P._s.ks) == (0, 5, sc.data_ptr())
    with pytest.raises(ValueError, match="fp16 pages have no scales"):
        K.KvPages(on(k), on(k), t, sc, sc)
    with pytest.raises((TypeError, ValueError), match="ks"):
        K.KvPages(u8, u8, t)
    with pytest.raises(ValueError, match="v: "):
        K.KvPages(u8, on(torch.zeros((4, 2, 32, 32), dtype=torch.uint8)), t, sc, sc)
    with pytest.raises(ValueError, match="vs: "):
        K.KvPages(u8, u8, t, sc, on(torch.zeros((4, 16, 2), dtype=torch.float16)))
    for bad in (None, t[0], on(t.long()), on(torch.zeros((5, 3), dtype=torch.int32)).t()):
        with pytest.raises(ValueError, match="table: need an int32"):
            K.KvPages(on(k), on(k), bad)
    with pytest.raises(ValueError, match="table: on"):
        K.KvPages(on(k), on(k), torch.zeros((3, 5), dtype=torch.int32))
    # rows apart, and not contiguous
    x = on(torch.zeros((3, 6, 64), dtype=torch.float16))
    assert K._rows(x[:, 2:4], "k", 2, 64, 3, 0) == (x.data_ptr() + 256, 384)
    assert K._rows(x[:1, 2:4], "k", 2, 64, 1, 0) == (x.data_ptr() + 256, 128)
    for bad in (x, x[:, ::3], x[:2, :2], x[:, :2].transpose(0, 1)):
        with pytest.raises(ValueError, match="k: "):
            K._rows(bad, "k", 2, 64, 3, 0)
    with pytest.raises(TypeError, match="k: dtype"):
        K._rows(on(torch.zeros((3, 2, 64))), "k", 2, 64, 3, 0)
    with pytest.raises(TypeError, match="k: expected"):
        K._rows(None, "k", 2, 64, 3, 0)
    with pytest.raises(ValueError, match="beyond what a call takes"):
        K.new_attn_pages_workspace(P, 3)


def test_more_wrapper_checks(cia):
    import torch

    from cuda_inf_amd import kernels as K

    class On(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 0

    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16).as_subclass(On)
    P = K.KvPages(k, k, torch.zeros((3, 5), dtype=torch.int32).as_subclass(On))
    pos, row = torch.zeros(2, dtype=torch.int32).as_subclass(On), torch.zeros((2, 2, 64), dtype=torch.float16).as_subclass(On)
    for f in (K.kv_pages_write, K.kv_pages_read):
        with pytest.raises(TypeError, match="pos: expected"):
            f(P, row, row, None)
        with pytest.raises(TypeError, match="pos: dtype"):
            f(P, row, row, pos.long())
        with pytest.raises(ValueError, match="v: "):
            f(P, row, row[:1], pos)
        with pytest.raises(ValueError, match="seq: needs at least 2"):
            f(P, row, row, pos, seq=pos[:1])
        with pytest.raises(ValueError, match="pos: must be a device tensor"):
            f(P, row, row, torch.zeros(2, dtype=torch.int32))
    q = torch.zeros((2, 4, 64), dtype=torch.float16).as_subclass(On)
    ws = torch.zeros(8, dtype=torch.uint8).as_subclass(On)
    for bad in (None, q[0], q[:, :, :32], q[:1]):
        with pytest.raises((TypeError, ValueError), match="q: "):
            K.attn_pages(P, bad, q, pos, ws)
    with pytest.raises(ValueError, match="out: needs at least"):
        K.attn_pages(P, q, q[:1], pos, ws)
    with pytest.raises(TypeError, match="ws: dtype"):
        K.attn_pages(P, q, q, pos, q)
    l, f = torch.zeros((2, 8)).as_subclass(On), torch.zeros(2).as_subclass(On)
    with pytest.raises(TypeError, match="u: dtype"):
        K.sample(l, f.half(), pos, ws)
    with pytest.raises(TypeError, match="top_k: dtype"):
        K.sample(l, f, pos, ws, top_k=f)
    with pytest.raises(ValueError, match="top_p: needs at least 2"):
        K.sample(l, f, pos, ws, top_p=f[:1])
    with pytest.raises(ValueError, match="logits: need a device tensor"):
        K.sample(l.t(), f, pos, ws)


def test_pages_of_no_elements(cia):
    import torch

    from cuda_inf_amd import kernels as K
    for shape in ((4, 2, 16, 0), (0, 2, 16, 64), (4, 0, 16, 64)):
        k = torch.zeros(shape, dtype=torch.float16)
        with pytest.raises(ValueError, match="k: need a tensor"):
            K.KvPages(k, k, torch.zeros((1, 1), dtype=torch.int32))


def test_page_table(cia):
    from cuda_inf_amd.layer import PageTable
    t = PageTable(3, 100, 8, page=16, device="cpu")
    assert t.table.shape == (3, 7) and (t.table == -1).all() and t.free_pages == 8
    t.reserve(0, 17)
    t.reserve(1, 0)
    t.reserve(2, 64)
    assert t.free_pages == 2
    got = t.table.tolist()
    assert got[1] == [-1] * 7 and got[0][2:] == [-1] * 5 and got[2][4:] == [-1] * 3
    assert sorted(got[0][:2] + got[2][:4]) == [0, 1, 2, 3, 4, 5]
    t.reserve(0, 20)  # (what it has already)
    assert t.table.tolist() == got
    with pytest.raises(RuntimeError, match="3 pages needed, 2 free"):
        t.reserve(1, 33)
    with pytest.raises(ValueError, match="a sequence holds 112"):
        t.reserve(0, 113)
    for seq in (-1, 3):
        with pytest.raises(ValueError, match="the table has 3"):
            t.reserve(seq, 1)
        with pytest.raises(ValueError, match="the table has 3"):
            t.release(seq)
    assert t.table.tolist() == got and t.free_pages == 2
    t.release(2)
    assert t.free_pages == 6 and (t.table[2] == -1).all()
    t.reserve(1, 96)
    assert t.free_pages == 0 and len(set(t.table[1, :6].tolist() + got[0][:2])) == 8


def test_page_table_refusals(cia):
    """What the calls over its pages would refuse, it refuses when it is made."""
    from cuda_inf_amd import _lib
    from cuda_inf_amd.layer import PageTable
    text = open(os.path.join(ROOT, "include", "cuda_inf_batch.h")).read()
    assert [int(re.search(rf"{n} (\d+)", text)[1]) for n in ("CIA_PAGE_MIN", "CIA_PAGE_MAX")] == [_lib.PAGE_MIN, _lib.PAGE_MAX]
    assert "CIA_PAGES_MAX_TOKENS (1 << 25)" in text and _lib.PAGES_MAX_TOKENS == 1 << 25
    for page in (0, 1, 8, 24, 48, 2048, -16):
        with pytest.raises(ValueError, match="page="):
            PageTable(2, 100, 4, page=page, device="cpu")
    for kw in (dict(max_seqs=0), dict(max_seqs=-1), dict(n_pages=0), dict(max_tokens=0), dict(max_tokens=(1 << 25) + 1)):
        with pytest.raises(ValueError, match=f"{list(kw)[0]}="):
            PageTable(**{**dict(max_seqs=2, max_tokens=100, n_pages=4), **kw}, device="cpu")
    for page in (16, 1024):
        assert PageTable(1, 1 << 25, 1, page=page, device="cpu").table.shape == (1, (1 << 25) // page)


def test_page_table_keeps_its_count(cia):
    """A table that cannot be written (its device out of memory, a stream that captures) leaves the pages where they were."""
    import torch

    from cuda_inf_amd.layer import PageTable
    t = PageTable(2, 100, 8, page=16, device="cpu")
    t.reserve(0, 40)
    whole = t.table

    class Closed(torch.Tensor):
        def __setitem__(self, at, what):
            raise RuntimeError("closed")

    t.table = whole.as_subclass(Closed)
    with pytest.raises(RuntimeError, match="closed"):
        t.reserve(1, 80)
    with pytest.raises(RuntimeError, match="closed"):
        t.reserve(0, 90)
    with pytest.raises(RuntimeError, match="closed"):
        t.release(0)
    t.table = whole
    assert t.free_pages == 5
    t.reserve(0, 48)  # (what it has)
    assert t.free_pages == 5 and (t.table[0, :3] >= 0).all() and (t.table[0, 3:] == -1).all() and (t.table[1] == -1).all()
    t.reserve(1, 80)
    assert t.free_pages == 0 and sorted(t.table[t.table >= 0].tolist()) == list(range(8))
    t.release(0)
    t.release(1)
    assert t.free_pages == 8 and (t.table == -1).all()


def test_choice_oracle():
    """The tests' own choice: hand-made rows."""
    import batch_ref as ref
    l = np.log(np.array([[0.1, 0.4, 0.2, 0.3]]))
    for u, kw, want, p in ((0.0, {}, 1, 0.4), (0.39, {}, 1, 0.4), (0.41, {}, 3, 0.3), (0.71, {}, 2, 0.2), (0.95, {}, 0, 0.1),
                           (0.95, dict(top_k=[3]), 2, 2 / 9), (0.95, dict(top_p=[0.65]), 3, 3 / 7),
                           (0.95, dict(top_p=[0.75]), 2, 2 / 9), (0.95, dict(min_p=[0.6]), 3, 3 / 7),
                           (0.95, dict(top_p=[0.0]), 1, 1.0), (0.5, dict(temperature=[0.0]), 1, 1.0),
                           (0.95, dict(top_k=[2], top_p=[0.5]), 1, 1.0), (2.0, {}, 0, 0.1), (-1.0, {}, 1, 0.4)):
        ids, q, _ = ref.choose(l, [u], **kw)
        assert ids[0] == want and abs(q[0] - p) < 1e-12, (u, kw)
    nan, inf = np.nan, np.inf
    assert ref.choose(np.array([[nan, -inf]]), [0.5])[0][0] == -1
    assert ref.choose(np.array([[nan, 1, 1, -inf]]), [0.6])[0][0] == 2
    assert ref.choose(np.array([[5, inf, 1, inf]]), [0.6])[0][0] == 3
    assert ref.choose(np.array([[1, 2, 2.0]]), [0.6], temperature=[0])[0][0] == 1


def test_attention_oracle():
    import batch_ref as ref
    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 5, 1, 16, 8))
    table = np.array([[3, 1], [0, -1]], np.int32)
    q = rng.standard_normal((2, 2, 8))
    out, _ = ref.attend(q, k, v, table, 16, [0, 1], [20, 30], 0.5, 0)
    kk, vv = (np.concatenate([x[3, 0], x[1, 0, :5]]) for x in (k, v))
    w = np.exp(0.5 * kk @ q[0, 1])
    assert np.allclose(out[0, 1], w @ vv / w.sum())
    # the second page is not there: 16 of the 31 tokens
    w = np.exp(0.5 * k[0, 0] @ q[1, 0])
    assert np.allclose(out[1, 0], w @ v[0, 0] / w.sum())
    out, _ = ref.attend(q, k, v, table, 16, [0, 1], [20, 30], 0.5, 4)
    w = np.exp(0.5 * k[1, 0, 1:5] @ q[0, 0])
    assert np.allclose(out[0, 0], w @ v[1, 0, 1:5] / w.sum()) and not out[1].any()
