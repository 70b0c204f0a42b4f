"""The paged cache, its attention and sampling on the GPU against plain forms."""
import numpy as np
import pytest
import torch

import batch_ref as ref

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


class Cache:
    """Pages of random rows on both sides; `stale` fills every byte and scale that no token of lens has."""

    def __init__(self, K, orc, dev, rng, lens, n_kv, D, page, quant, spare=3, width=None, stale=0x7F, scale=1.0):
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        width = width or max(max(need), 1) + 1
        self.table = ref.table_of(rng, n_pages, need, width)
        self.page, self.n_pages = page, n_pages
        self.num, self.raw = {}, {}
        shape = (n_pages, n_kv, page, D)
        live = np.zeros((n_pages, page), bool)
        for i, n in enumerate(lens):
            for j in range(0, n, page):
                live[self.table[i, j // page], :min(page, n - j)] = True
        for name in "kv":
            x = (scale * rng.standard_normal(shape) * (0.3 + 3 * rng.random(D) ** 4)).astype(np.float16)
            if quant:
                b, s = ref.quant(orc, x)
                b[~live.repeat(n_kv, 0).reshape(n_pages, n_kv, page)] = stale
                s[~live.repeat(n_kv, 0).reshape(n_pages, n_kv, page)] = np.nan
                self.raw[name], self.raw[name + "s"] = t(b, dev), t(s, dev)
                self.num[name] = orc.e4m3_decode_table()[b].astype(np.float64) * s.astype(np.float64)[..., None]
            else:
                x[~live.repeat(n_kv, 0).reshape(n_pages, n_kv, page)] = np.nan if stale == 0x7F else np.inf
                self.raw[name], self.raw[name + "s"] = t(x, dev), None
                self.num[name] = x.astype(np.float64)
        self.dev_table = t(self.table, dev)
        self.P = K.KvPages(self.raw["k"], self.raw["v"], self.dev_table, self.raw["ks"], self.raw["vs"])


# ------------------------------------------------------------------ write and read
MOVES = [(1, 8, 64, 64, True), (1, 1, 128, 16, True), (33, 3, 64, 16, True), (100, 8, 64, 32, False),
         (257, 2, 128, 128, True), (17, 5, 128, 16, False), (700, 1, 64, 1024, True)]


@pytest.mark.parametrize("T,n_kv,D,page,quant", MOVES)
@pytest.mark.parametrize("apart", [0, 24])
def test_write_and_read(K, orc, dev, T, n_kv, D, page, quant, apart):
    """Tokens of several sequences in any order, rows apart, some without a place: bytes
    and scales of their places as kv_quant_write stores them, every other one as it was;
    and back, rows without a place as they were."""
    rng = np.random.default_rng(T + D + apart)
    n_seq, width = 5, max(2, -(-T // page))
    n_pages = n_seq * width + 2
    table = ref.table_of(rng, n_pages, [width] * n_seq, width)
    table[2, width - 1] = -1
    table[3, 0] = n_pages  # beyond the cache
    order = rng.permutation(n_seq * width * page)[:T]
    seq, pos = (order // (width * page)).astype(np.int32), (order % (width * page)).astype(np.int32)
    if T > 8:
        pos[3], pos[5], seq[6], seq[7] = -1, width * page, n_seq, -1
        pos[2], seq[4] = 2 ** 31 - 1, -2 ** 31
    x = [(rng.standard_normal((T, n_kv, D)) * (1 + 30 * (rng.random(D) < 0.05))).astype(np.float16) for _ in "kv"]
    if T > 20:
        x[0][8], x[1][9] = 0, -0.0
        x[0][10, 0, 1], x[1][11, 0, 3], x[1][12, 0, 7] = np.nan, np.inf, -6e-8
    wide = [torch.full((T, n_kv * D + apart), 3.0, dtype=torch.float16, device=dev) for _ in x]
    rows = [w[:, :n_kv * D].unflatten(1, (n_kv, D)) for w in wide]
    for r, a in zip(rows, x):
        r.copy_(t(a, dev))
    if quant:
        raw = [torch.full((n_pages, n_kv, page, D), 0x55, dtype=torch.uint8, device=dev) for _ in x]
        sc = [torch.full((n_pages, n_kv, page), 7.0, dtype=torch.float16, device=dev) for _ in x]
    else:
        raw = [torch.full((n_pages, n_kv, page, D), 7.0, dtype=torch.float16, device=dev) for _ in x]
        sc = [None, None]
    tab = torch.full((n_seq, width + 3), 0, dtype=torch.int32, device=dev)
    tab[:, :width] = t(table, dev)
    P = K.KvPages(*raw, tab[:, :width], *sc)
    K.kv_pages_write(P, *rows, t(pos, dev), seq=t(seq, dev))
    pid, row, ok = ref.places(table, n_pages, page, seq, pos)
    assert T < 8 or (ok.any() and not ok.all())
    back = [np.full((T, n_kv, D), 9.0, np.float16) for _ in x]
    for a, r, s, z in zip(x, raw, sc, back):
        if quant:
            want, ws = np.full(r.shape, 0x55, np.uint8), np.full(s.shape, 7.0, np.float16)
            b, bs = ref.quant(orc, a)
            want[pid[ok], :, row[ok]], ws[pid[ok], :, row[ok]] = b[ok], bs[ok]
            got = r.cpu().numpy()
            # (a row with an infinity: inf / inf is a NaN of either sign)
            both = np.isnan(orc.e4m3_decode_table()[want]) & np.isnan(orc.e4m3_decode_table()[got])
            assert np.array_equal(np.where(both, 0, got), np.where(both, 0, want))
            assert np.array_equal(s.cpu().numpy().view(np.uint16), ws.view(np.uint16))
            with np.errstate(invalid="ignore"):
                z[ok] = (orc.e4m3_decode_table()[b] * bs.astype(np.float32)[..., None]).astype(np.float16)[ok]
        else:
            want = np.full(r.shape, 7.0, np.float16)
            want[pid[ok], :, row[ok]] = a[ok]
            assert np.array_equal(r.cpu().numpy().view(np.uint16), want.view(np.uint16))
            z[ok] = a[ok]
    for r in rows:
        r.fill_(9.0)
    K.kv_pages_read(P, *rows, t(pos, dev), seq=t(seq, dev))
    for r, w, z in zip(rows, wide, back):
        assert np.array_equal(r.cpu().numpy(), z, equal_nan=True)
        assert (w[:, n_kv * D:] == 3.0).all()


def test_write_matches_kv_quant_write(K, dev):
    """The reference's slots and a one-page cache of one head hold the same rows."""
    g = torch.Generator(device="cpu").manual_seed(3)
    k, v = (torch.randn((16, 8, 64), generator=g).half().to(dev) for _ in range(2))
    f = [torch.zeros((16, 8, 64), dtype=torch.uint8, device=dev) for _ in range(2)]
    s = [torch.zeros((16, 8), dtype=torch.float16, device=dev) for _ in range(2)]
    at = torch.arange(16, dtype=torch.int32, device=dev)
    K.kv_quant_write(k, v, *f, *s, at, 16)
    raw = [torch.zeros((1, 8, 16, 64), dtype=torch.uint8, device=dev) for _ in range(2)]
    sc = [torch.zeros((1, 8, 16), dtype=torch.float16, device=dev) for _ in range(2)]
    P = K.KvPages(*raw, torch.zeros((1, 1), dtype=torch.int32, device=dev), *sc)
    K.kv_pages_write(P, k, v, at, seq=torch.zeros_like(at))
    for a, b, c, d in zip(f, raw, s, sc):
        assert torch.equal(a, b[0].transpose(0, 1)) and torch.equal(c, d[0].t())


def test_sequence_t_is_token_ts(K, dev):
    k = torch.randn((3, 2, 64), device=dev).half()
    raw = [torch.zeros((3, 2, 16, 64), dtype=torch.float16, device=dev) for _ in range(2)]
    table = torch.tensor([[2], [0], [1], [1]], dtype=torch.int32, device=dev)
    P = K.KvPages(*raw, table)
    K.kv_pages_write(P, k, -k, torch.tensor([4, 0, 15], dtype=torch.int32, device=dev))
    for i, (page, row) in enumerate(((2, 4), (0, 0), (1, 15))):
        assert torch.equal(raw[0][page, :, row], k[i]) and torch.equal(raw[1][page, :, row], -k[i])
    assert raw[0].count_nonzero() == k.count_nonzero()


# ------------------------------------------------------------------ attention
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 127, 128, 129, 0, 191, 255, 257, 500, 1000]


def attend(K, c, dev, q, seq, pos, scale, window, ws=None):
    T, n_q, D = q.shape
    out = torch.full((T, n_q, D), 7.0, dtype=torch.float16, device=dev)
    ws = K.new_attn_pages_workspace(c.P, n_q) if ws is None else ws
    K.attn_pages(c.P, t(q, dev), out, t(pos, dev), ws, seq=t(seq, dev), scale=scale, window=window)
    return out


def check(K, c, dev, q, seq, pos, scale, window, ws=None, what=""):
    out = attend(K, c, dev, q, seq, pos, scale, window, ws)
    want, bound = ref.attend(q, c.num["k"], c.num["v"], c.table, c.page, np.arange(len(pos)) if seq is None else seq, pos,
                             scale, window)
    within(out.cpu().numpy(), want, bound, what)
    return out


@pytest.mark.parametrize("n_q,n_kv,D,page,quant", [
    (32, 8, 64, 64, True), (4, 4, 64, 16, True), (6, 3, 128, 32, True), (7, 1, 64, 128, True), (16, 2, 128, 16, True),
    (16, 1, 64, 16, True), (17, 1, 64, 64, True), (64, 1, 128, 64, True), (40, 2, 64, 32, True), (1, 1, 64, 1024, True),
    (32, 8, 64, 64, False), (5, 5, 128, 16, False), (12, 2, 64, 16, False), (14, 2, 128, 32, False), (36, 1, 128, 64, False),
    (3, 1, 64, 16, False)])
@pytest.mark.parametrize("window", [0, 1, 50, 300])
def test_attention_of_all_lengths(K, orc, dev, n_q, n_kv, D, page, quant, window):
    """Every length about a tile's, a page's and a unit's edge, an empty row among them; places behind a
    sequence's last token hold NaN."""
    rng = np.random.default_rng(n_q + 10 * D + page)
    c = Cache(K, orc, dev, rng, EDGES, n_kv, D, page, quant)
    q = (2 * rng.standard_normal((len(EDGES), n_q, D))).astype(np.float16)
    pos = np.array(EDGES, np.int32) - 1
    out = check(K, c, dev, q, None, pos, D ** -0.5, window, what=f"window {window}")
    assert (out[EDGES.index(0)] == 0).all()


@pytest.mark.parametrize("quant", [True, False])
def test_attention_rows_of_any_sequence(K, orc, dev, quant):
    """Rows of a sequence at several positions, in any order, q rows apart; sequences and positions that are none."""
    rng = np.random.default_rng(5)
    lens = [300, 40, 513]
    c = Cache(K, orc, dev, rng, lens, 2, 64, 32, quant)
    seq = np.array([2, 0, 2, 1, 2, 0, -1, 3, 1, 2 ** 31 - 1, 2], np.int32)
    pos = np.array([512, 299, 0, 39, 255, 5, 3, 3, -1, 3, -2 ** 31], np.int32)
    wide = (2 * rng.standard_normal((11, 9, 64))).astype(np.float16)
    q = t(wide, dev)[:, 1:7]
    out = torch.full((11, 6, 64), 7.0, dtype=torch.float16, device=dev)
    K.attn_pages(c.P, q, out, t(pos, dev), K.new_attn_pages_workspace(c.P, 6), seq=t(seq, dev), scale=0.2)
    want, bound = ref.attend(wide[:, 1:7], c.num["k"], c.num["v"], c.table, 32, seq, pos, 0.2, 0)
    within(out.cpu().numpy(), want, bound, "rows")
    assert (out[[6, 7, 8, 9, 10]] == 0).all()


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_attention_without_some_pages(K, orc, dev, quant, page):
    """Pages that are not there take no part; a row of none, and one whose window holds none, are 0; a position
    behind the table's last column attends to what the table holds."""
    rng = np.random.default_rng(page)
    n = 10 * page
    c = Cache(K, orc, dev, rng, [n, n, n, n, n], 2, 64, page, quant, width=10)
    c.table[0, [0, 3, 9]] = -1
    c.table[1, :] = [-1, c.n_pages, 2 ** 31 - 1, -2 ** 31, -1, -5, c.n_pages + 7, -1, -1, -1]
    c.table[2, 4:] = -1
    c.table[3, 1:9] = c.n_pages
    c.dev_table.copy_(t(c.table, dev))
    q = (2 * rng.standard_normal((5, 8, 64))).astype(np.float16)
    pos = np.array([n - 1, n - 1, n - 1, n - 1, n + 1000], np.int32)
    out = check(K, c, dev, q, None, pos, 0.125, 0, what="pages")
    assert (out[1] == 0).all() and (out[4] != 0).any()
    out = check(K, c, dev, q, None, np.minimum(pos, n - 1), 0.125, 2 * page, what="window")
    assert (out[1] == 0).all() and (out[2] == 0).all()


def test_attention_over_long_caches(K, orc, dev):
    """One long sequence among short ones, split over many workgroups; and the same alone."""
    rng = np.random.default_rng(9)
    lens = [40000, 3, 700, 20001]
    c = Cache(K, orc, dev, rng, lens, 2, 64, 64, True)
    q = (2 * rng.standard_normal((4, 8, 64))).astype(np.float16)
    pos = np.array(lens, np.int32) - 1
    ws = K.new_attn_pages_workspace(c.P, 8)
    check(K, c, dev, q, None, pos, 0.125, 0, ws, "long")
    check(K, c, dev, q[:1], None, pos[:1], 0.125, 0, ws, "one")
    check(K, c, dev, q, None, pos, 0.125, 9000, ws, "window")
    a = attend(K, c, dev, q, None, pos, 0.125, 0, ws)
    for _ in range(3):
        assert torch.equal(a, attend(K, c, dev, q, None, pos, 0.125, 0, ws))


@pytest.mark.parametrize("T", [255, 256, 257, 1000, 4096])
def test_attention_of_many_rows(K, orc, dev, T):
    """Batches about and above a workgroup's threads, most rows short, some empty; the largest call."""
    rng = np.random.default_rng(T)
    lens = [5, 130, 64, 900]
    c = Cache(K, orc, dev, rng, lens, 1, 64, 16, True)
    seq = rng.integers(0, 4, T).astype(np.int32)
    pos = (rng.random(T) * np.array(lens)[seq]).astype(np.int32)
    pos[rng.random(T) < 0.1] = -1
    q = (2 * rng.standard_normal((T, 2, 64))).astype(np.float16)
    check(K, c, dev, q, seq, pos, 0.125, 0, what=f"{T} rows")


@pytest.mark.parametrize("n_q,n_kv,D,quant", [(128 * 64, 128, 64, True), (128, 128, 128, False), (64 * 5, 5, 64, True),
                                              (33 * 7, 7, 128, True)])
def test_attention_of_many_heads(K, orc, dev, n_q, n_kv, D, quant):
    """Heads at their limits: one workgroup for a kv head and 16 query heads, parts of 16 that are not full."""
    rng = np.random.default_rng(n_q)
    lens = [200, 1, 0, 777]
    c = Cache(K, orc, dev, rng, lens, n_kv, D, 32, quant)
    q = rng.standard_normal((4, n_q, D)).astype(np.float16)
    check(K, c, dev, q, None, np.array(lens, np.int32) - 1, D ** -0.5, 0, what="heads")


def test_attention_of_the_most_rows_of_wide_heads(K, orc, dev):
    """4096 rows whose list and joins take the most of a workgroup's LDS."""
    rng = np.random.default_rng(77)
    lens = [700, 90]
    c = Cache(K, orc, dev, rng, lens, 1, 128, 64, False)
    seq = rng.integers(0, 2, 4096).astype(np.int32)
    pos = np.where(seq == 0, rng.integers(-1, 700, 4096), rng.integers(-1, 90, 4096)).astype(np.int32)
    q = rng.standard_normal((4096, 16, 128)).astype(np.float16)
    out = attend(K, c, dev, q, seq, pos, 0.09, 130)
    some = np.r_[0:40, 2000:2040, 4056:4096]
    want, bound = ref.attend(q[some], c.num["k"], c.num["v"], c.table, 64, seq[some], pos[some], 0.09, 130)
    within(out.cpu().numpy()[some], want, bound, "rows")
    assert not out.isnan().any() and (out[torch.from_numpy(pos < 0)] == 0).all()


@pytest.mark.parametrize("quant", [True, False])
def test_attention_values(K, orc, dev, quant):
    """Scores far apart and far from zero, all alike, scales of a few steps of fp16's least, rows of zeros."""
    rng = np.random.default_rng(2)
    lens = [300, 300, 300, 300]
    for scale in (1.0, 1e-4, 3e-7, 60.0):
        c = Cache(K, orc, dev, rng, lens, 1, 64, 64, quant, scale=scale)
        q = (np.array([0.0, 3.0, 200.0, -9.0])[:, None, None] * rng.standard_normal((4, 3, 64))).astype(np.float16)
        check(K, c, dev, q, None, np.array(lens, np.int32) - 1, 0.125, 0, what=f"scale {scale}")
        check(K, c, dev, q, None, np.array(lens, np.int32) - 1, -0.125, 0, what=f"scale {scale}, negative")
        check(K, c, dev, q, None, np.array(lens, np.int32) - 1, 0.0, 0, what="mean")


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("gap", [8.0, 14.0, 17.0, 19.0])
def test_attention_of_many_small_weights(K, orc, dev, quant, gap):
    """One token with nearly all the weight and a V of zeros, at the start or the end, 12000 others that the output
    is made of, each of a weight down to 6e-9 of it; so many rows that a workgroup has all of a row."""
    rng = np.random.default_rng(1)
    n, D, T = 12000, 64, 2048
    c = Cache(K, orc, dev, rng, [n, n], 1, D, 64, quant)
    q = np.zeros((T, 4, D), np.float16)
    q[:, :, 0] = 8.0 * gap  # score gap with scale 1/8 for a key of 1 against one of 0
    for name in "kv":
        x = np.zeros((c.n_pages, 1, 64, D), np.float16)
        for s, at in ((0, 0), (1, n - 1)):
            page = int(c.table[s, at // 64])
            if name == "v":
                x[c.table[s, :-(-n // 64)]] = (1 + rng.random((-(-n // 64), 1, 64, D))).astype(np.float16)
                x[page, 0, at % 64] = 0
            else:
                x[page, 0, at % 64, 0] = 1.0
        if quant:
            b, sc = ref.quant(orc, x)
            c.raw[name].copy_(t(b, dev))
            c.raw[name + "s"].copy_(t(sc, dev))
            c.num[name] = orc.e4m3_decode_table()[b].astype(np.float64) * sc.astype(np.float64)[..., None]
        else:
            c.raw[name].copy_(t(x, dev))
            c.num[name] = x.astype(np.float64)
    seq = np.arange(T, dtype=np.int32) % 2
    pos = np.full(T, n - 1, np.int32)
    out = attend(K, c, dev, q, seq, pos, 0.125, 0).cpu().numpy()
    want, bound = ref.attend(q[:2], c.num["k"], c.num["v"], c.table, 64, seq[:2], pos[:2], 0.125, 0)
    for s in range(2):
        within(out[s::2], want[s], bound[s], f"gap {gap}, {s}")


def test_attention_of_numbers_that_are_none(K, orc, dev):
    """A NaN in a token that is attended to reaches its kv head's rows alone; one outside the window nothing."""
    rng = np.random.default_rng(3)
    c = Cache(K, orc, dev, rng, [200, 200], 2, 64, 16, True)
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    c.raw["v"][int(c.table[0, 2]), 1, 5, 7] = 0x7F  # token 37 of sequence 0, kv head 1, dimension 7
    c.raw["k"][int(c.table[1, 0]), 0, 0, 0] = 0x7F  # token 0 of sequence 1, kv head 0
    pos = np.array([199, 199], np.int32)
    out = attend(K, c, dev, q, None, pos, 0.125, 0).cpu()
    bad = out.isnan()
    assert bad[0, 2:, 7].all() and bad[0].sum() == 2 and bad[1, :2].all() and bad[1].sum() == 2 * 64
    assert not attend(K, c, dev, q, None, pos, 0.125, 162).isnan().any()


@pytest.mark.parametrize("group", [1, 4, 8, 16])
def test_attention_to_an_infinity(K, orc, dev, group):
    rng = np.random.default_rng(5)
    c = Cache(K, orc, dev, rng, [50, 50], 1, 64, 16, False)
    q = rng.standard_normal((2, group, 64)).astype(np.float16)
    c.raw["v"][int(c.table[0, 1]), 0, 3, 9] = float("inf")  # token 19 of sequence 0, dimension 9
    pos = np.array([49, 49], np.int32)
    bad = ~attend(K, c, dev, q, None, pos, 0.125, 0).cpu().isfinite()
    assert bad[0, :, 9].all() and bad.sum() == group
    assert attend(K, c, dev, q, None, pos, 0.125, 30).isfinite().all()


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("scale", [2.0 ** 64, -(2.0 ** 64), 2.0 ** 40])
def test_attention_at_the_largest_scales(K, orc, dev, quant, scale):
    """Only the largest score's token is left: its V, rounded once (2^-11 of it, or half of the least step)."""
    rng = np.random.default_rng(6)
    c = Cache(K, orc, dev, rng, [700, 31], 2, 64, 16, quant)
    q = rng.standard_normal((2, 8, 64)).astype(np.float16)
    pos = np.array([699, 30], np.int32)
    out = attend(K, c, dev, q, None, pos, scale, 0).cpu().numpy()
    for s in range(2):
        at = [(int(c.table[s, j // 16]), j % 16) for j in range(pos[s] + 1)]
        k, v = (np.stack([c.num[name][p, :, r] for p, r in at]) for name in "kv")  # [tokens, kv heads, D]
        for h in range(8):
            best = np.argmax(np.sign(scale) * (k[:, h // 4] @ q[s, h].astype(np.float64)))
            want = v[best, h // 4]
            within(out[s, h], want, np.abs(want) * 2.0 ** -11 + 2.0 ** -25, f"sequence {s}, head {h}")


@pytest.mark.parametrize("sizes", [(-10, 7), (-16, -15), (-8, -7), (6, 7)])
@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("units", [2.0 ** 20, *(f * 2.0 ** e for e in (21, 22, 23, 24, 25, 26, 27, 28, 29) for f in (1.02, 1.11, 1.3, 1.47, 1.7, 1.83)), 2.0 ** 40])
def test_attention_of_equals_among_large_scores(K, orc, dev, quant, units, sizes):
    """Scores of `units` powers of 2, where fp32's steps reach and pass those that numerators are kept within.  All alike:
    the mean of V, whose tokens' sizes (e4m3: scales) lie 2^16 apart or are all of one; weights are equal, so that only the sums' terms
    of ref.attend's bound count.  The later ones higher by 16 or more, and still so where both are rounded to steps of
    up to 16: their mean, and 128 / 100 * 2^-16 of the first ones' at most.  A call of two rows, and of so many that a
    workgroup has all units of a row."""
    rng = np.random.default_rng(8)
    n, D = 228, 64
    c = Cache(K, orc, dev, rng, [n, n], 1, D, 16, quant)
    shape = (c.n_pages, 1, 16)
    size = (2.0 ** rng.integers(*sizes, shape)).astype(np.float16)
    v = rng.integers(-16, 17, (*shape, D)).astype(np.float32)  # (whole numbers to 16: exact in e4m3)
    k = np.zeros((*shape, D), np.float32)
    k[..., 0] = 448.0
    step = 2.0 ** min(7.0, max(0.0, 27 - np.floor(np.log2(units))))
    for j in range(128, n):  # 448 and 2^-14 `step`: 2^-22.8 of it higher for a step of 1
        k[int(c.table[1, j // 16]), 0, j % 16, 1] = step
    if quant:
        for name, x, s in (("k", k, np.ones(shape, np.float16)), ("v", v, size)):
            c.raw[name].copy_(t(orc.e4m3_encode(x.reshape(-1)).reshape(x.shape), dev))
            c.raw[name + "s"].copy_(t(s, dev))
    else:
        c.raw["k"].copy_(t(k.astype(np.float16), dev))
        c.raw["v"].copy_(t((v * size[..., None]).astype(np.float16), dev))
    num = v.astype(np.float64) * size.astype(np.float64)[..., None]
    rows = [np.stack([num[int(c.table[s, j // 16]), 0, j % 16] for j in range(n)]) for s in range(2)]
    apart = units * step * 2.0 ** -14 / 448 >= 16
    for T in (2, 1024):
        q = np.zeros((T, 4, D), np.float16)
        q[..., 0], q[..., 1] = 1.0, 2.0 ** -14
        out = attend(K, c, dev, q, np.arange(T, dtype=np.int32) % 2, np.full(T, n - 1, np.int32),
                     units * np.log(2.0) / 448, 0).cpu().numpy()
        for s in range(2 if apart else 1):
            x = rows[s][128:] if s else rows[s]
            want, mass = x.mean(0), np.abs(x).mean(0)
            bound = mass * ((n / 16 + 64) * 2 * ref.U24 + 2.0 ** -22) + n * 2.0 ** -37 * np.abs(x).max()
            if s:
                bound = bound + 1.28 * 2.0 ** -16 * (mass + np.abs(rows[s][:128]).mean(0))
            within(out[s::2], want, bound + np.abs(want) * ref.U11 * 1.001 + 2.0 ** -25, f"{T} rows, sequence {s}")


def test_pages_beyond_32_bits(K, orc, dev):
    """Rows of pages whose bytes lie past 2^32: written, attended and read."""
    n_pages, page, n_kv, D = 2100, 1024, 8, 128
    raw = [torch.empty((n_pages, n_kv, page, D), dtype=torch.float16, device=dev) for _ in range(2)]
    table = np.array([[n_pages - 1, 3], [2070, n_pages - 2]], np.int32)
    P = K.KvPages(*raw, t(table, dev))
    rng = np.random.default_rng(4)
    n = [1500, 1100]
    T = sum(n)
    seq, pos = np.repeat([0, 1], n).astype(np.int32), np.concatenate([np.arange(x) for x in n]).astype(np.int32)
    x = [rng.standard_normal((T, n_kv, D)).astype(np.float16) for _ in "kv"]
    K.kv_pages_write(P, *(t(a, dev) for a in x), t(pos, dev), seq=t(seq, dev))
    back = [torch.zeros((T, n_kv, D), dtype=torch.float16, device=dev) for _ in x]
    K.kv_pages_read(P, *back, t(pos, dev), seq=t(seq, dev))
    for a, b in zip(x, back):
        assert np.array_equal(a, b.cpu().numpy())
    num = [np.zeros((4, n_kv, page, D), np.float16) for _ in x]
    small = np.array([[0, 1], [2, 3]], np.int32)
    for a, b in zip(x, num):
        p, r, _ = ref.places(small, 4, page, seq, pos)
        b[p, :, r] = a
    q = rng.standard_normal((2, 8, D)).astype(np.float16)
    out = torch.empty((2, 8, D), dtype=torch.float16, device=dev)
    last = np.array(n, np.int32) - 1
    K.attn_pages(P, t(q, dev), out, t(last, dev), K.new_attn_pages_workspace(P, 8), scale=D ** -0.5)
    want, bound = ref.attend(q, *num, small, page, [0, 1], last, D ** -0.5, 0)
    within(out.cpu().numpy(), want, bound, "far pages")


# ------------------------------------------------------------------ sampling
def sample(K, dev, l, u, V=None, **f):
    B = l.shape[0]
    ids = torch.full((B,), -7, dtype=torch.int32, device=dev)
    p = torch.full((B,), -7.0, device=dev)
    x = l if isinstance(l, torch.Tensor) else t(l, dev)
    ws = torch.empty(K.sample_workspace_bytes(B, x.shape[1]), dtype=torch.uint8, device=dev)
    f = {k: t(np.asarray(v, np.int32 if k == "top_k" else np.float32), dev) for k, v in f.items()}
    K.sample(x, t(np.asarray(u, np.float32), dev), ids, ws, p=p, **f)
    return ids.cpu().numpy(), p.cpu().numpy()


def check_sample(K, dev, l, u, what="", **f):
    """Tokens equal, but where the draw fell within 1e-9 of the border to another: sums are good to 2^-34 of
    themselves and the weights left out are below 2^-41; p half an fp32 step and as much."""
    ids, p = sample(K, dev, l, u, **f)
    g = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in f.items()}
    want, q, near = ref.choose(np.asarray(l), np.asarray(u, np.float32), **g)
    sure = near > 1e-9
    assert sure.mean() > 0.9, what
    assert np.array_equal(ids[sure], want[sure]), f"{what}: rows {np.nonzero((ids != want) & sure)[0]}"
    within(p[sure], q[sure], q[sure] * (ref.U24 + 1e-9), what)


FILTERS = [dict(), dict(top_k=1), dict(top_k=3), dict(top_k=50), dict(top_k=1000), dict(top_p=0.9), dict(top_p=0.2),
           dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0), dict(min_p=1e-6), dict(top_k=40, top_p=0.9, min_p=0.02),
           dict(top_k=200, top_p=0.5), dict(temperature=0.3), dict(temperature=4.0, top_p=0.95), dict(temperature=0.01),
           dict(temperature=30.0), dict(temperature=0.0), dict(temperature=1.5, min_p=0.1, top_k=5000)]


@pytest.mark.parametrize("B,V", [(7, 1), (5, 2), (9, 63), (6, 257), (12, 1500), (4, 4095), (5, 16385), (3, 65536),
                                 (2, 131073)])
@pytest.mark.parametrize("half", [False, True])
def test_sample(K, dev, B, V, half):
    rng = np.random.default_rng(V + half)
    l = (2.5 * rng.standard_normal((B, V)) + 6 * rng.random((B, V)) ** 200).astype(np.float16 if half else np.float32)
    for i, f in enumerate(FILTERS):
        u = rng.random(B).astype(np.float32)
        check_sample(K, dev, l, u, f"{V} {f}", **{k: np.full(B, v) for k, v in f.items()})


def test_sample_of_mixed_rows(K, dev):
    """Each row its own parameters, rows of the logits apart and not aligned, no p wanted."""
    rng = np.random.default_rng(8)
    B, V = 300, 777
    wide = (3 * rng.standard_normal((B, 779))).astype(np.float32)
    f = dict(temperature=rng.choice([0.0, 0.2, 0.7, 1.0, 2.0], B), top_k=rng.choice([-1, 0, 1, 2, 30, 777, 5000], B),
             top_p=rng.choice([0.1, 0.5, 0.9, 0.99, 1.0, 1.5], B), min_p=rng.choice([-1.0, 0.0, 0.01, 0.3, 1.0], B))
    u = rng.random(B)
    for dtype in (np.float32, np.float16):
        x = t(wide.astype(dtype), dev)[:, 1:778]
        ids, p = sample(K, dev, x, u, **f)
        g = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in f.items()}
        want, q, near = ref.choose(wide.astype(dtype)[:, 1:778], u.astype(np.float32), **g)
        assert np.array_equal(ids, want) and near.min() > 1e-9
        within(p, q, q * (ref.U24 + 1e-9), "p")
        ids2 = torch.empty(B, dtype=torch.int32, device=dev)
        ws = torch.empty(K.sample_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
        K.sample(x, t(u.astype(np.float32), dev), ids2, ws,
                 **{k: t(v, dev) for k, v in g.items()})
        assert np.array_equal(ids, ids2.cpu().numpy())


@pytest.mark.parametrize("V", [5, 5000, 70000])
@pytest.mark.parametrize("half", [False, True])
def test_sample_of_ties(K, dev, V, half):
    """Logits of a few values each, more equals than are put in order at once: the lowest index first."""
    rng = np.random.default_rng(V)
    dtype = np.float16 if half else np.float32
    kinds = [np.zeros(V), rng.integers(0, 2, V), rng.integers(0, 3, V) * 1e-3, np.where(rng.random(V) < 0.5, 0.0, -0.0),
             -5 + rng.integers(0, 4, V) * 0.25, np.full(V, 1e4), np.where(np.arange(V) % 2, 3.0, -np.inf),
             np.linspace(0, 1e-2, V)]
    l = np.stack(kinds).astype(dtype)
    B = len(kinds)
    for f in (dict(), dict(top_k=3), dict(top_k=V // 2 + 1), dict(top_p=0.37), dict(top_p=0.9, top_k=V - 1), dict(min_p=0.9),
              dict(min_p=1.0), dict(temperature=1e-3), dict(temperature=np.inf)):
        u = (rng.integers(0, 2 ** 20, B) + 0.37) / 2 ** 20
        check_sample(K, dev, l, u, f"{f}", **{k: np.full(B, v) for k, v in f.items()})


def test_sample_of_numbers_that_are_none(K, dev):
    nan, inf = np.nan, np.inf
    V = 300
    l = np.full((10, V), -inf, np.float32)
    l[1, 7], l[2, [3, 250]], l[3, 9], l[4] = 2.0, inf, nan, nan
    l[5], l[5, 4], l[5, 5] = 1.0, nan, -inf
    l[6], l[6, [1, 299]] = 5.0, inf
    l[7] = 3.4e38
    l[8] = -3.4e38
    l[8, 17] = 3.4e38
    l[9] = 1e-45
    u = np.array([0.5, 0.9, 0.7, 0.5, 0.5, 0.0149, 0.3, 0.5, 0.5, 0.999], np.float32)
    for half in (False, True):
        with np.errstate(over="ignore"):
            x = l.astype(np.float16) if half else l
        for f in (dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.3), dict(temperature=0.0), dict(temperature=1e-44)):
            f = {k: np.full(10, v) for k, v in f.items()}
            ids, p = sample(K, dev, x, u, **f)
            want, q, _ = ref.choose(x, u, **{k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in f.items()})
            assert np.array_equal(ids, want), (half, f)
            within(p, q, q * (ref.U24 + 1e-9), f"{f}")
    # parameters that are none
    l = np.random.default_rng(1).standard_normal((6, 40)).astype(np.float32)
    bad = np.array([nan, inf, -inf, -1.0, 2.0, 0.5], np.float32)
    for name in ("temperature", "top_p", "min_p"):
        check_sample(K, dev, l, np.full(6, 0.6), name, **{name: bad})
    for u, same in ((nan, 0.0), (-3.0, 0.0), (-inf, 0.0), (1.0, 1 - 2.0 ** -24), (inf, 1 - 2.0 ** -24)):
        a, b = sample(K, dev, l, np.full(6, u)), sample(K, dev, l, np.full(6, same))
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("V", [1000, 16384, 16385, 20000, 65536, 70000, 262144, 262145, 270000])
@pytest.mark.parametrize("half", [False, True])
def test_sample_of_rows_with_infinities(K, dev, V, half):
    """+inf in rows of one chunk and of many, of both sizes, beside finite logits far above 0: one, a few of one
    chunk, some of all chunks, more in one chunk than it lists, more than are put in order at once, and a row of
    them alone; a NaN and -inf between them.  They are the choice, all alike; a row without any is as ever."""
    rng = np.random.default_rng(V + half)
    dtype = np.float16 if half else np.float32
    spots = [[V // 2], [V - 1], [0, 3, 250], rng.permutation(V)[:40], rng.permutation(min(V, 8192))[:700],
             rng.permutation(V)[:900], np.arange(0, V, max(1, V // 1500)), rng.permutation(V)[:V // 3], np.arange(V), []]
    l = (2 * rng.standard_normal((len(spots), V)) + np.linspace(-30, 30, len(spots))[:, None]).astype(dtype)
    for row, at in zip(l, spots):
        row[at] = np.inf
    l[1:3, 5], l[1:3, 7] = np.nan, -np.inf
    B = len(spots)
    for f in (dict(), dict(top_k=1), dict(top_k=2), dict(top_k=500), dict(top_p=0.6), dict(min_p=0.3),
              dict(top_k=650, top_p=0.7, min_p=0.5), dict(temperature=0.0), dict(temperature=np.inf, top_k=100),
              dict(temperature=1e-3)):
        f = {k: np.full(B, v) for k, v in f.items()}
        u = (rng.integers(0, 2 ** 20, B) + 0.37) / 2 ** 20
        ids, _ = sample(K, dev, l, u, **f)
        assert (ids >= 0).all() and (ids < V).all(), f"{V} {f}"
        check_sample(K, dev, l, u, f"{V} {f}", **f)


def test_sample_of_the_longest_rows(K, dev):
    rng = np.random.default_rng(6)
    V = 1 << 22
    l = (1.5 * rng.standard_normal((2, V))).astype(np.float32)
    for f in (dict(), dict(top_k=100), dict(top_p=0.9), dict(temperature=0.0), dict(temperature=8.0, top_k=1 << 21)):
        check_sample(K, dev, l, [0.83, 0.21], f"{f}", **{k: np.full(2, v) for k, v in f.items()})


def sample_within(K, dev, l, u, temperature, bound, what):
    """Tokens equal where the draw is further than `bound` (of the kept mass) from a border, valid everywhere; p half
    an fp32 step and twice the bound, once for the weight and once for the sum."""
    ids, p = sample(K, dev, l, u, temperature=temperature)
    want, q, near = ref.choose(l, np.asarray(u, np.float32), temperature=temperature.astype(np.float32))
    sure = near > bound
    assert np.array_equal(ids[sure], want[sure]), what
    assert ((ids >= 0) & (ids < l.shape[1])).all()
    same = ids == want
    within(p[same], q[same], q[same] * (ref.U24 + 2 * bound), what)
    return sure


@pytest.mark.parametrize("V", [16384, 131072, 262144, 1 << 22])
def test_sample_of_a_peak_and_a_far_tail(K, dev, V):
    """One token and V - 1 alike far below it, on both sides of the weight from which on they may count as 0."""
    gaps = np.array([20.0, 28.0, 28.4, 28.6, 29.0, 29.07, 29.2, 30.0])
    l = np.repeat(-gaps[:, None].astype(np.float32), V, 1)
    l[:, V // 3] = 0.0
    far = 2.0 ** -34 + V * 2.0 ** -41
    for u in (0.5, 1 - 2.0 ** -24):
        sure = sample_within(K, dev, l, np.full(8, u), np.ones(8), far, f"{V} {u}")
        assert u > 0.5 or sure.all()
        # weights of 2^-41 and more (e^-28.4) count: bounds of their own alone
        sample_within(K, dev, l[:3], np.full(3, u), np.ones(3), 2.0 ** -33, f"{V} {u}, counted")


@pytest.mark.parametrize("V", [50, 20000])
def test_sample_of_cold_rows(K, dev, V):
    """Temperatures down to 2^-28 beside logits of 1, whose neighbours' weights are e^-1 to e^-16."""
    rng = np.random.default_rng(V)
    for e in (10, 18, 20, 22, 24, 26, 28):
        T = 2.0 ** -e
        l = np.zeros((6, V), np.float32)
        for row in l:
            row[rng.permutation(V)[:40]] = 1.0 - np.arange(40) * max(T, 2.0 ** -23)
        if e == 10:
            l[l == 0] = -1.0
        assert sample_within(K, dev, l, rng.random(6), np.full(6, T), 2.0 ** -34 + 2.0 ** (e - 52) + V * 2.0 ** -41, f"2^-{e}").all()


def test_sample_frequencies(K, dev):
    """Equally spaced numbers draw every token as often as its probability says."""
    rng = np.random.default_rng(0)
    l = np.repeat((1.5 * rng.standard_normal(11)).astype(np.float32)[None], 5000, 0)
    ids, _ = sample(K, dev, l, (np.arange(5000) + 0.5) / 5000, temperature=np.full(5000, 0.8), top_k=np.full(5000, 9))
    w = np.exp((l[0].astype(np.float64) - l[0].max()) / np.float32(0.8))
    w[np.argsort(l[0])[:2]] = 0
    assert (np.abs(np.bincount(ids, minlength=11) - 5000 * w / w.sum()) <= 1).all()


@pytest.mark.parametrize("B,V", [(3, 8191), (3, 8192), (3, 8193), (2, 262144), (2, 262145), (70, 65536), (300, 20001),
                                 (520, 16384), (600, 3), (256, 65536), (257, 65536)])
@pytest.mark.parametrize("half", [False, True])
def test_sample_about_a_chunks_edge(K, dev, B, V, half):
    """Rows of one chunk and of many, of both sizes, one more logit and one less, batches on both sides of the
    choice between them; rows in descending and ascending order, whose largest tokens all lie in one chunk."""
    rng = np.random.default_rng(B + V)
    n = min(B, 6)
    l = np.zeros((B, V), np.float16 if half else np.float32)
    l[:] = (2 * rng.standard_normal((n, V)))[np.arange(B) % n]
    l[0] = np.sort(l[0])
    l[1] = np.sort(l[1])[::-1]
    l[2 % B, V // 2:] = -np.inf
    check = np.unique(np.r_[0:n, rng.integers(0, B, 3), B - 1])
    x = t(l, dev)
    for f in (dict(top_k=30), dict(top_k=800, top_p=0.95), dict(top_p=0.6), dict(min_p=0.2), dict(), dict(temperature=0.0)):
        u = rng.random(B).astype(np.float32)
        f = {k: np.full(B, v, np.int32 if k == "top_k" else np.float32) for k, v in f.items()}
        ids, p = sample(K, dev, x, u, **f)
        want, q, near = ref.choose(l[check], u[check], **{k: v[check] for k, v in f.items()})
        sure = near > 1e-9
        assert sure.mean() > 0.6 and np.array_equal(ids[check][sure], want[sure]), f
        within(p[check][sure], q[sure], q[sure] * (ref.U24 + 1e-9), f"{f}")


def test_sample_of_tokens_that_one_thread_meets(K, dev):
    """The likely tokens 2048 apart, and 8192 and 512: more of them a thread than it keeps."""
    rng = np.random.default_rng(4)
    V = 1 << 19
    l = (rng.standard_normal((6, V)) - 30).astype(np.float32)
    for b, (step, n) in enumerate(((2048, 256), (8192, 64), (512, 1024), (2048, 200), (2048, 256), (4, 1000))):
        l[b, 5:5 + step * n:step] = 2 * rng.standard_normal(n)
    l[4, 5::2048] = 1.0  # (equals)
    for f in (dict(top_k=60), dict(top_p=0.9), dict(top_k=150, top_p=0.7, min_p=0.01), dict(min_p=0.05), dict(),
              dict(temperature=0.5, top_k=1000)):
        check_sample(K, dev, l, rng.random(6), f"{f}", **{k: np.full(6, v) for k, v in f.items()})


@pytest.mark.parametrize("V", [3, 4, 5, 1023, 1025, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385, 270000])
@pytest.mark.parametrize("half", [False, True])
def test_sample_of_rows_about_the_limits_of_their_kernels(K, dev, V, half):
    """Broad and narrow rows, one whose likely tokens are the last, one of equals, one with numbers that are none."""
    rng = np.random.default_rng(V)
    l = np.stack([1.5 * rng.standard_normal(V), 9 * rng.standard_normal(V), np.where(np.arange(V) >= V - 5, 7.0, 0.0) + rng.random(V),
                  np.full(V, -3.0), rng.standard_normal(V), -20 * rng.random(V)]).astype(np.float16 if half else np.float32)
    l[4, V // 2], l[4, 0], l[4, -1] = np.nan, -np.inf, -np.inf
    for f in (dict(), dict(top_k=1), dict(top_k=40), dict(top_k=1200), dict(top_p=0.8), dict(top_p=0.99, top_k=700), dict(min_p=0.2),
              dict(top_k=50, top_p=0.6, min_p=0.1), dict(temperature=0.0), dict(temperature=0.3, min_p=0.01)):
        check_sample(K, dev, l, rng.random(6), f"{f}", **{k: np.full(6, v) for k, v in f.items()})


@pytest.mark.parametrize("V", [1, 8, 1000, 70000, 140000])
def test_sample_at_the_border_between_equals(K, dev, V):
    """Sums of equals are whole: a number on the border between two of them draws the second."""
    at = np.unique(np.minimum(V - 1, np.array([0, 1, 2, V // 8, V // 4, V // 2, V - 1])))
    u = (at / V).astype(np.float32)
    keep = (u.astype(np.float64) * V == at)  # those that fp32 holds
    at, u = at[keep], u[keep]
    assert at.size
    for level, temp in ((0.3, 1.0), (-7.25, 0.7), (1e4, 1.3)):
        l = np.full((at.size, V), level, np.float32)
        ids, p = sample(K, dev, l, u, temperature=np.full(at.size, temp))
        assert np.array_equal(ids, at)
        assert (p == np.float32(1 / V)).all()


def test_calls_of_other_sizes_on_the_same_workspaces(K, orc, dev):
    """A workspace that a larger call has filled, and one whose contents are anything."""
    rng = np.random.default_rng(2)
    l = (2 * rng.standard_normal((40, 30000))).astype(np.float32)
    x, u = t(l, dev), rng.random(40).astype(np.float32)
    ws = torch.full((K.sample_workspace_bytes(40, 30000),), 0xFF, dtype=torch.uint8, device=dev)
    ids = torch.zeros(40, dtype=torch.int32, device=dev)
    tp = torch.full((40,), 0.8, device=dev)
    for B, V in ((40, 30000), (3, 29999), (40, 100), (1, 30000), (40, 30000)):
        K.sample(x[:B, :V], t(u, dev), ids, ws, top_p=tp)
        want, _, near = ref.choose(l[:B, :V], u[:B], top_p=np.full(B, 0.8, np.float32))
        assert near.min() > 1e-9 and np.array_equal(ids[:B].cpu().numpy(), want)
    lens = [3000, 5, 600]
    c = Cache(K, orc, dev, rng, lens, 2, 64, 16, True)
    ws = torch.zeros(max(K.attn_pages_workspace_bytes(n, 2, 64) for n in (2, 8, 32)), dtype=torch.uint8, device=dev)
    for n_q, rows in ((32, 3), (2, 1), (8, 3), (32, 2), (2, 3)):
        q = rng.standard_normal((rows, n_q, 64)).astype(np.float16)
        check(K, c, dev, q, None, np.array(lens[:rows], np.int32) - 1, 0.125, 0, ws, f"{n_q} heads")


@pytest.mark.parametrize("B,V", [(1, 300), (5, 16384), (1, 16385), (3, 20000), (31, 65536), (65, 262144), (3, 262145), (300, 70000)])
def test_sample_stays_in_its_workspace(K, dev, B, V):
    """A workspace of the stated size, odd numbers of chunks among them, with nothing written beside it."""
    n, edge = K.sample_workspace_bytes(B, V), 4096
    assert V > 16384 or n <= 64  # (rows of one launch need none)
    whole = torch.full((edge + n + edge,), 0xA5, dtype=torch.uint8, device=dev)
    rng = np.random.default_rng(V)
    l = (2 * rng.standard_normal((min(B, 7), V))).astype(np.float32)[np.arange(B) % 7]
    x, u = t(l, dev), rng.random(B).astype(np.float32)
    ids = torch.empty(B, dtype=torch.int32, device=dev)
    for f in (dict(top_k=40), dict(top_p=0.9)):
        f = {k: np.full(B, v, np.int32 if k == "top_k" else np.float32) for k, v in f.items()}
        K.sample(x, t(u, dev), ids, whole[edge:edge + n], **{k: t(v, dev) for k, v in f.items()})
        some = np.unique(np.r_[0:min(B, 3), B - 1])
        want, _, near = ref.choose(l[some], u[some], **{k: v[some] for k, v in f.items()})
        assert near.min() > 1e-9 and np.array_equal(ids.cpu().numpy()[some], want)
        assert (whole[:edge] == 0xA5).all() and (whole[edge + n:] == 0xA5).all()


def test_two_streams_at_once(K, orc, dev):
    """The same calls on two streams, each with its workspaces, one cache between them."""
    rng = np.random.default_rng(14)
    lens = [5000, 900, 20]
    c = Cache(K, orc, dev, rng, lens, 2, 64, 64, True)
    pos = t(np.array(lens, np.int32) - 1, dev)
    q = [t((2 * rng.standard_normal((3, 8, 64))).astype(np.float16), dev) for _ in range(2)]
    l = [t((2 * rng.standard_normal((3, 50000))).astype(np.float32), dev) for _ in range(2)]
    u = t(rng.random(3).astype(np.float32), dev)
    ws = [(K.new_attn_pages_workspace(c.P, 8), torch.empty(K.sample_workspace_bytes(3, 50000), dtype=torch.uint8, device=dev))
          for _ in range(2)]
    tp = torch.full((3,), 0.9, device=dev)

    def run(i):
        out, ids = torch.empty_like(q[i]), torch.empty(3, dtype=torch.int32, device=dev)
        for _ in range(10):
            K.attn_pages(c.P, q[i], out, pos, ws[i][0])
            K.sample(l[i], u, ids, ws[i][1], top_p=tp)
        return out, ids

    alone = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            both.append(run(i))
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ together, streams, graphs
@pytest.mark.parametrize("V", [9000, 40000, 300000])
def test_on_another_stream_and_captured(K, orc, dev, V):
    """Write, attention and sampling captured on a fresh stream, replayed with other inputs and eager work
    between: every replay is the eager result."""
    rng = np.random.default_rng(12)
    lens = [700, 33, 0, 2100]
    c = Cache(K, orc, dev, rng, [x + 8 for x in lens], 2, 64, 16, True, stale=0)
    B, n_q = 4, 8
    q = torch.zeros((B, n_q, 64), dtype=torch.float16, device=dev)
    kv = [torch.zeros((B, 2, 64), dtype=torch.float16, device=dev) for _ in range(2)]
    pos, u = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, device=dev)
    logits = torch.zeros((B, V), device=dev)
    tp = torch.full((B,), 0.9, device=dev)
    out, ids, p = torch.zeros_like(q), torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, device=dev)
    ws = K.new_attn_pages_workspace(c.P, n_q)
    ws2 = torch.empty(K.sample_workspace_bytes(B, V), dtype=torch.uint8, device=dev)

    def step():
        K.kv_pages_write(c.P, *kv, pos)
        K.attn_pages(c.P, q, out, pos, ws)
        K.sample(logits, u, ids, ws2, top_p=tp, p=p)

    def inputs(i):
        g = torch.Generator(device="cpu").manual_seed(i)
        for x in (q, *kv, logits):
            x.copy_(torch.randn(x.shape, generator=g).to(x.dtype) * 2)
        u.copy_(torch.rand(B, generator=g))
        pos.copy_(torch.tensor([x - 1 + i if x else -1 + (i > 2) for x in lens], dtype=torch.int32))

    state = {k: v.clone() for k, v in c.raw.items()}
    eager = []
    for i in range(5):
        inputs(i)
        step()
        eager.append([x.clone() for x in (out, ids, p)])
    torch.cuda.synchronize()
    after = {k: v.clone() for k, v in c.raw.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    inputs(0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(2):
        for k, v in state.items():
            c.raw[k].copy_(v)
        for i in range(5):
            inputs(i)
            graph.replay()
            for a, b in zip(eager[i], (out, ids, p)):
                assert torch.equal(a, b)
            torch.cuda.synchronize()
        for k, v in after.items():
            assert torch.equal(c.raw[k].view(torch.uint8), v.view(torch.uint8))
        step()  # eager work on the same workspaces
        for a, b in zip(eager[4], (out, ids, p)):
            assert torch.equal(a, b)
    # eager on another stream
    for x in (out, ids, p):
        x.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    for a, b in zip(eager[4], (out, ids, p)):
        assert torch.equal(a, b)


def test_pages_change_hands_outside_a_capture(cia, dev):
    from cuda_inf_amd.layer import PageTable
    table = PageTable(2, 100, 8, page=16, device=dev)
    table.reserve(0, 40)
    x = torch.zeros(4, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        for change in (lambda: table.reserve(1, 40), lambda: table.release(0)):
            with pytest.raises(RuntimeError, match="outside a graph's capture"):
                change()
    graph.replay()
    table.reserve(1, 80)
    assert (x == 1).all() and table.free_pages == 0
    assert sorted(table.table[table.table >= 0].tolist()) == list(range(8)) and (table.table[0, 3:] == -1).all()


def int4(rng, rows, cols, dev):
    packed = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    scales = ((0.5 + rng.random((rows, cols // 128))) * 0.35 / np.sqrt(cols)).astype(np.float16)
    return t(packed, dev), t(scales, dev)


@pytest.mark.parametrize("quant", [True, False])
def test_a_batch_decodes(K, orc, dev, quant):
    """The decode loop of a batch: embedding rows, and in each of two layers norm, q/k/v, producers, pages, attention,
    out_proj and the dense branch; then logits and a token each, which is the next step's.  Sequences of
    several lengths, one that ends and one that begins on the way.  Each step's attention and tokens are those of the
    plain forms on the step's own cache, queries and logits."""
    from cuda_inf_amd.layer import MoeBlock, PagedAttn, PageTable
    rng = np.random.default_rng(21)
    H, V, B, steps = 2048, 1000, 5, 6
    table = PageTable(B, 400, 12, page=64, device=dev)
    layers = []
    for _ in range(2):
        w = dict(norm=t((1 + 0.1 * rng.standard_normal(H)).astype(np.float16), dev),
                 q=int4(rng, 2048, H, dev), k=int4(rng, 512, H, dev), v=int4(rng, 512, H, dev), o=int4(rng, H, 2048, dev),
                 qw=t((1 + 0.1 * rng.standard_normal(64)).astype(np.float16), dev),
                 kw=t((1 + 0.1 * rng.standard_normal(64)).astype(np.float16), dev))
        ffn = [int4(rng, *s, dev) for s in ((512, H), (512, H), (H, 512))]
        w["ffn"] = MoeBlock(w["norm"], *[(p[None], s[None]) for p, s in ffn], max_batch=B, device=dev)
        w["attn"] = PagedAttn(table, quant=quant)
        layers.append(w)
    head, embed = int4(rng, V, H, dev), t(rng.standard_normal((V, H)).astype(np.float32), dev)
    lens = [100, 3, 64, 0, 300]
    for s, n in enumerate(lens):
        if not n:
            continue
        table.reserve(s, n + steps)
        at = torch.arange(n, dtype=torch.int32, device=dev)
        for w in layers:
            w["attn"].write(*(t(rng.standard_normal((n, 8, 64)).astype(np.float16), dev) for _ in range(2)), at,
                            seq=torch.full_like(at, s))
    assert table.free_pages == 12 - 2 - 1 - 2 - 5
    with pytest.raises(RuntimeError, match="pages needed"):
        table.reserve(3, 400)
    pos = torch.tensor(lens, dtype=torch.int32, device=dev)
    pos[3] = -1
    ids = torch.zeros(B, dtype=torch.int32, device=dev)
    p, u = torch.zeros(B, device=dev), torch.zeros(B, device=dev)
    ws = torch.empty(K.sample_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
    f = dict(temperature=np.array([0.7, 0.0, 1.2, 1.0, 0.9], np.float32), top_k=np.array([40, 0, 0, 5, 0], np.int32),
             top_p=np.array([0.9, 1, 0.95, 1, 1], np.float32), min_p=np.array([0, 0, 0.02, 0, 0.1], np.float32))
    fd = {k: t(v, dev) for k, v in f.items()}
    x = torch.zeros((B, H), dtype=torch.float16, device=dev)
    q = torch.zeros((B, 32, 64), dtype=torch.float16, device=dev)
    k, v, out = torch.zeros((B, 8, 64), dtype=torch.float16, device=dev), torch.zeros((B, 8, 64), dtype=torch.float16, device=dev), torch.zeros_like(q)
    logits = torch.zeros((B, V), device=dev)
    codes = orc.e4m3_decode_table().astype(np.float64)
    for step in range(steps):
        if step == 3:
            table.release(4)
            pos[4] = -1
            table.reserve(3, steps)
            pos[3] = 0
        h = embed[ids.long()].clone()
        for w in layers:
            K.add_rmsnorm(h, w["norm"], x, B, H)
            K.qkv_proj_int4(x, w["q"], w["k"], w["v"], q, k, v, B)
            K.qk_norm_rope(q, k, w["qw"], w["kw"], pos.clamp(min=0), B)
            w["attn"].decode(q, k, v, pos, out=out)
            P = w["attn"].pages
            num = [codes[c.cpu().numpy()] * s.cpu().numpy().astype(np.float64)[..., None] if quant else c.cpu().numpy()
                   for c, s in ((P.k, P.ks), (P.v, P.vs))]
            want, bound = ref.attend(q.cpu().numpy(), *num, table.table.cpu().numpy(), 64, np.arange(B), pos.cpu().numpy(), 0.125, 0)
            within(out.cpu().numpy(), want, bound, f"step {step}")
            back = [torch.full_like(k, 9.0) for _ in range(2)]
            w["attn"].read(*back, pos)
            live = pos >= 0
            for got, new in zip(back, (k, v)):
                assert (got[~live] == 9).all()
                # a step of e4m3 is 2^-3 of a value at most, half of it the bytes', and a 2^-11 each of scale and result;
                # below 2^-6 of 448 scales steps are 2^-9 of the scale
                far = (got[live].double() - new[live].double()).abs()
                amax = new[live].double().abs().amax(2, keepdim=True)
                assert (far <= (new[live].double().abs() * (2.0 ** -4 + 2.0 ** -10) + amax / 448 * 2.0 ** -10 if quant else 0 * amax)).all()
            K.gemv_int4(out, *w["o"], h, H, 2048, B, add=True)
            w["ffn"].forward(h)
        K.add_rmsnorm(h, layers[0]["norm"], x, B, H)
        K.gemv_int4(x, *head, logits, V, H, B)
        un = rng.random(B).astype(np.float32)
        u.copy_(t(un, dev))
        K.sample(logits, u, ids, ws, p=p, **fd)
        assert logits.isfinite().all()
        want, pw, near = ref.choose(logits.cpu().numpy(), un, **f)
        assert near.min() > 1e-9 and np.array_equal(ids.cpu().numpy(), want)
        within(p.cpu().numpy(), pw, pw * (ref.U24 + 1e-9), f"p of step {step}")
        pos += (pos >= 0).int()
    assert table.free_pages == 12 - 2 - 1 - 2 - 1
