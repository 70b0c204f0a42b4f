"""One attention layer of the cuda_inf engine: its device cache, the host state
the reference keeps beside it, and the attention branch of ``layer_forward``
(engine.cu:802-857), run by the C++ driver ``cia_layer_forward``.

Also exposes the host-only policy helpers (append planner, H2O clamps and
slot picker) which need no GPU.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import (D, KVGROUP, NH, NKV, NSPLIT_DEFAULT, PAGE_MAX, PAGE_MIN, PAGES_MAX_TOKENS, call,
                   cia_append_op, cia_attn_proj, cia_layer, cia_moe)
from .kernels import (KvPages, _stream_on, attn_pages, decode_workspace_bytes, h2o_workspace_bytes,
                      kv_pages_read, kv_pages_write, moe_gating, new_attn_pages_workspace, q4_experts,
                      stream_handle)

HIDDEN = _lib.HIDDEN


# ------------------------------------------------------------ host policy
def kv_append_plan(committed: int, S: int, past: int):
    """engine.cu:830-845 as a list of ops; returns (ops, new_committed)."""
    max_ops = S // KVGROUP + 2
    ops = (cia_append_op * max_ops)()
    c = ctypes.c_int(committed)
    n = ctypes.c_int(0)
    call("cia_kv_append_plan", ctypes.byref(c), S, past, ops, max_ops, ctypes.byref(n))
    out = [dict(src_token=o.src_token, slot=o.slot, cnt=o.cnt, commit=bool(o.commit),
                commit_base=o.commit_base, commit_grp=o.commit_grp) for o in ops[:n.value]]
    return out, c.value


def h2o_clamp(budget: int, window: int, prompt_len: int, maxT: int):
    """engine.cu:752-756; returns (budget, window)."""
    b, w = ctypes.c_int(budget), ctypes.c_int(window)
    _lib.lib().cia_h2o_clamp(ctypes.byref(b), ctypes.byref(w), prompt_len, maxT)
    return b.value, w.value


def h2o_pick_slots(n_live: int, C: int, W: int, slotpos: np.ndarray, attn_host: np.ndarray,
                   S: int, past: int):
    """engine.cu:808-823 on host arrays (updated in place).

    Returns (n_live, dst[S], zeroed[S], evictions)."""
    assert slotpos.dtype == np.int32 and attn_host.dtype == np.float32
    dst = np.zeros(S, np.int32)
    zeroed = np.zeros(S, np.int32)
    nl = ctypes.c_int(n_live)
    ev = _lib.lib().cia_h2o_pick_slots(ctypes.byref(nl), C, W, slotpos.ctypes.data,
                                       attn_host.ctypes.data, S, past, dst.ctypes.data,
                                       zeroed.ctypes.data)
    if ev < 0:
        _lib.check("cia_h2o_pick_slots", -ev)
    return nl.value, dst, zeroed, ev


# ------------------------------------------------------------ the layer
class AttnLayer:
    """Device buffers of one attention layer (engine.cu:596-613, 731-770).

    ``nsplit`` > 0 runs the reference's flash-decoding split + combine with
    that split count; ``nsplit`` = 0 runs the matrix-core decode with the
    library's own split (and the tail write fused into it).  ``budget`` > 0
    enables H2O eviction with a ``budget``-slot buffer and local ``window``
    (0 -> budget/2, clamped as the reference does against ``prompt_len``).
    ``qk_norm`` = (q weight, k weight), fp16 [64] each: q and k passed to
    ``forward`` are raw and the layer runs the QK producers (per-head
    RMSNorm with ``eps``, RoPE at ``theta``; engine.cu:799-801) itself --
    inside the decode kernels for single-token steps, else one launch into a
    ``max_batch``-token scratch.
    """

    def __init__(self, max_tokens: int, *, nsplit: int = NSPLIT_DEFAULT, budget: int = 0,
                 window: int = 0, prompt_len: int = 0, max_batch: int = 4096,
                 qk_norm=None, eps: float = 1e-5, theta: float = 5.0e6, device="cuda"):
        dev = torch.device(device)
        self.device = dev
        self.maxT = max_tokens
        u8, f16, f32, i32 = torch.uint8, torch.float16, torch.float32, torch.int32
        ng = max_tokens // KVGROUP + 2
        self.kc8 = torch.zeros((max_tokens, NKV, D), dtype=u8, device=dev)
        self.vc8 = torch.zeros((max_tokens, NKV, D), dtype=u8, device=dev)
        self.ksc = torch.zeros((ng, NKV), dtype=f16, device=dev)
        self.vsc = torch.zeros((ng, NKV), dtype=f16, device=dev)
        self.ktail = torch.zeros((KVGROUP, NKV, D), dtype=f16, device=dev)
        self.vtail = torch.zeros((KVGROUP, NKV, D), dtype=f16, device=dev)
        self.nsplit = nsplit
        ns = max(nsplit, 1)
        self.pm = torch.zeros(NH * ns, dtype=f32, device=dev)
        self.pl = torch.zeros(NH * ns, dtype=f32, device=dev)
        self.po = torch.zeros(NH * ns * D, dtype=f32, device=dev)
        self.ws_decode = torch.zeros(decode_workspace_bytes(max_tokens), dtype=u8, device=dev)
        s = cia_layer()
        for name in ("kc8", "vc8", "ksc", "vsc", "ktail", "vtail", "pm", "pl", "po", "ws_decode"):
            setattr(s, name, getattr(self, name).data_ptr())
        s.maxT, s.committed, s.nsplit = max_tokens, 0, nsplit
        self.budget = 0
        if budget > 0:
            budget, window = h2o_clamp(budget, window, prompt_len, max_tokens)
            self.budget, self.window = budget, window
            C = budget
            self.kf = torch.zeros((C, NKV, D), dtype=u8, device=dev)
            self.vf = torch.zeros((C, NKV, D), dtype=u8, device=dev)
            self.ks = torch.zeros((C, NKV), dtype=f16, device=dev)
            self.vs = torch.zeros((C, NKV), dtype=f16, device=dev)
            self.hattn = torch.zeros(C, dtype=f32, device=dev)
            self.d_slotpos = torch.full((C,), -1, dtype=i32, device=dev)
            self.d_dst = torch.zeros(max_batch, dtype=i32, device=dev)
            self.ws_mass = torch.zeros(h2o_workspace_bytes(max_batch, C), dtype=u8, device=dev)
            s.budget, s.window = budget, window
            for name in ("kf", "vf", "ks", "vs", "hattn", "d_slotpos", "d_dst", "ws_mass"):
                setattr(s, name, getattr(self, name).data_ptr())
            s.n_live = 0
        if qk_norm is not None:
            qw, kw = qk_norm
            self.qw = torch.as_tensor(qw).to(device=dev, dtype=f16).contiguous()
            self.kw = torch.as_tensor(kw).to(device=dev, dtype=f16).contiguous()
            assert self.qw.numel() == D and self.kw.numel() == D
            self.prep_ws = torch.zeros(max_batch * (NH + NKV) * D, dtype=f16, device=dev)
            s.qw, s.kw = self.qw.data_ptr(), self.kw.data_ptr()
            s.eps, s.theta = float(eps), float(theta)
            s.prep_ws, s.prep_cap = self.prep_ws.data_ptr(), max_batch
        self.max_batch = max_batch
        self._s = s

    @property
    def committed(self) -> int:
        return self._s.committed

    @property
    def n_live(self) -> int:
        return self._s.n_live

    def forward(self, q, k, v, past: int, out=None, scale: float = 0.125, evicted: bool = True):
        """Append k, v [S,8,64] at positions past.. and attend q [S,32,64].

        Returns (out [S,32,64] fp16, evicted slot of the last token or -1).
        On an H2O layer the evicted slot is read back from the device, which
        waits for the stream; ``evicted=False`` skips that (returns None)."""
        S = k.shape[0]
        if (self.budget or self._s.qw) and S > self.max_batch:
            raise ValueError(f"S={S} exceeds max_batch={self.max_batch}")
        for t, name, n in ((q, "q", S * NH * D), (k, "k", S * NKV * D), (v, "v", S * NKV * D)):
            if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous() or t.numel() != n:
                raise ValueError(f"{name}: need a contiguous device fp16 tensor of {n} elements")
        if out is None:
            out = torch.empty((S, NH, D), dtype=torch.float16, device=self.device)
        ev = ctypes.c_int(-1)
        call("cia_layer_forward", ctypes.byref(self._s), q.data_ptr(), k.data_ptr(), v.data_ptr(),
             out.data_ptr(), S, past, float(scale), ctypes.byref(ev) if evicted else None,
             stream_handle())
        return out, (ev.value if evicted else None)

    # -------------------------------------------------------- projections
    def set_projections(self, wq, wk, wv, wo):
        """INT4 group-128 weights of q/k/v/out_proj (engine.cu:792-797, 858):
        each a (packed u8 [N, 1024], scales fp16 [N, 16]) pair of device
        tensors, N = 2048 / 512 / 512 / 2048."""
        P = cia_attn_proj()
        self._proj_w = []
        for name, (pk, sc), N in (("q", wq, NH * D), ("k", wk, NKV * D), ("v", wv, NKV * D),
                                  ("o", wo, HIDDEN)):
            if (pk.dtype != torch.uint8 or not pk.is_cuda or not pk.is_contiguous()
                    or pk.numel() != N * HIDDEN // 2):
                raise ValueError(f"{name}_proj packed: need contiguous device uint8 [{N}, {HIDDEN // 2}]")
            if (sc.dtype not in (torch.float16, torch.int16) or not sc.is_cuda
                    or not sc.is_contiguous() or sc.numel() != N * HIDDEN // 128):
                raise ValueError(f"{name}_proj scales: need contiguous device fp16 [{N}, {HIDDEN // 128}]")
            setattr(P, name + "_packed", pk.data_ptr())
            setattr(P, name + "_scales", sc.data_ptr())
            self._proj_w += [pk, sc]
        self.proj_ws = torch.zeros(self.max_batch * (2 * NH * D + 2 * NKV * D), dtype=torch.float16,
                                   device=self.device)
        P.ws, P.cap = self.proj_ws.data_ptr(), self.max_batch
        self._p = P

    def block_forward(self, x, h, past: int, scale: float = 0.125, evicted: bool = True):
        """engine.cu:792-859: x fp16 [S, 2048] (normalised hidden state) through
        q/k/v_proj, the QK producers (when the layer has qk_norm), attention
        and out_proj, added into the residual h fp32 [S, 2048] in place.
        Returns the evicted slot of the last token on an H2O layer (or -1;
        None with evicted=False)."""
        S = x.numel() // HIDDEN
        if x.dtype != torch.float16 or not x.is_cuda or not x.is_contiguous() or x.numel() != S * HIDDEN:
            raise ValueError("x: need a contiguous device fp16 tensor [S, 2048]")
        if h.dtype != torch.float32 or not h.is_cuda or not h.is_contiguous() or h.numel() != S * HIDDEN:
            raise ValueError("h: need a contiguous device fp32 tensor [S, 2048]")
        ev = ctypes.c_int(-1)
        call("cia_attn_block_forward", ctypes.byref(self._s), ctypes.byref(self._p), x.data_ptr(),
             h.data_ptr(), S, past, float(scale), ctypes.byref(ev) if evicted else None,
             stream_handle())
        return ev.value if evicted else None


def attn_block_loop(layers, x, h, past: int, steps: int, scale: float = 0.125, events=None):
    """cia_attn_block_loop: steps decode steps through the attention branches
    of ``layers`` (AttnLayer with projections).  x fp16 [steps, n_layers, 2048],
    h fp32 [2048] (the residual stream, added into in place)."""
    n = len(layers)
    arr = (cia_layer * n)(*[L._s for L in layers])
    parr = (cia_attn_proj * n)(*[L._p for L in layers])
    ev = None
    if events is not None:
        for e in events:  # the hipEvent_t handles exist once recorded
            e.record()
        ev = (ctypes.c_void_p * len(events))(*[e.cuda_event for e in events])
    try:
        call("cia_attn_block_loop", arr, parr, n, x.data_ptr(), h.data_ptr(), past, steps,
             float(scale), ev, stream_handle())
    finally:
        for L, s in zip(layers, arr):  # host counters advance in the copies
            L._s.committed, L._s.n_live = s.committed, s.n_live


# ------------------------------------------------------------ the feed-forward branch
class MoeBlock:
    """The feed-forward branch of one layer (engine.cu:869-905): ffn_norm, the
    router, and the chosen experts' INT4 products, into the residual.

    ``norm_w``: fp16 [H].  ``w1``, ``w3`` ([E, F, H]) and ``w2`` ([E, H, F]):
    INT4 group-128 experts as (packed u8 [E, rows, cols / 2], scales fp16
    [E, rows, cols / 128]) pairs of device tensors.  ``gate`` (fp16 [E, H]) with
    ``top_k``, ``renorm_eps`` and the other arguments of ``kernels.moe_gating``
    routes; without it the layer is dense (E = 1).  ``bias``: fp32 [E], for the
    choice alone.  ``eps``: the norm's.  ``max_batch``: tokens a call may bring.
    """

    def __init__(self, norm_w, w1, w3, w2, *, gate=None, bias=None, top_k: int = 1, eps: float = 1e-5,
                 renorm_eps: float = 1e-6, max_batch: int = 4096, device="cuda", **gating):
        dev = torch.device(device)
        M = cia_moe()
        M.w1, E, F, H = q4_experts(w1, "w1")
        M.w3, *s3 = q4_experts(w3, "w3")
        M.w2, *s2 = q4_experts(w2, "w2")
        if s3 != [E, F, H] or s2 != [E, H, F]:
            raise ValueError(f"w3 {s3} and w2 {s2} do not go with w1 {[E, F, H]}")
        if gate is None and (E != 1 or bias is not None or top_k != 1 or gating):
            raise ValueError("experts need a gate (a dense layer has one expert and no router)")
        for t, name, dtype, shape in ((norm_w, "norm_w", torch.float16, (H,)),
                                      (gate, "gate", torch.float16, (E, H)),
                                      (bias, "bias", torch.float32, (E,))):
            if t is not None and (t.dtype != dtype or not t.is_cuda or not t.is_contiguous()
                                  or tuple(t.shape) != shape):
                raise ValueError(f"{name}: need a contiguous device {dtype} tensor {shape}")
        if dev.index is None:
            dev = norm_w.device
        for t in (norm_w, *w1, *w3, *w2, gate, bias):
            if t is not None and t.device != dev:
                raise ValueError(f"a weight is on {t.device}, the layer on {dev}")
        self.H, self.max_batch = H, max_batch
        self._keep = (norm_w, w1, w3, w2, gate, bias)
        M.norm_w, M.norm_eps, M.H, M.F = norm_w.data_ptr(), float(eps), H, F
        if gate is not None:
            M.gate = gate.data_ptr()
            M.bias = None if bias is None else bias.data_ptr()
            M.gating = moe_gating(E, top_k, eps=renorm_eps, **gating)
        M.cap = max_batch
        M.ws_bytes = _lib.lib().cia_moe_block_workspace_bytes(ctypes.byref(M), max_batch)
        if not M.ws_bytes:
            raise ValueError(f"max_batch={max_batch}, top_k={top_k}, {E} experts of {F}, H={H}: beyond what a call takes")
        self.ws = torch.empty(M.ws_bytes, dtype=torch.uint8, device=dev)
        M.ws = self.ws.data_ptr()
        self._m = M

    def forward(self, h) -> None:
        """h fp32 [S, H], the residual, in place; S up to max_batch."""
        S = h.numel() // self.H
        if (h.dtype != torch.float32 or not h.is_cuda or not h.is_contiguous()
                or h.numel() != S * self.H):
            raise ValueError(f"h: need a contiguous device fp32 tensor [S, {self.H}]")
        if S > self.max_batch:
            raise ValueError(f"S={S} exceeds max_batch={self.max_batch}")
        if h.device != self.ws.device:
            raise ValueError(f"h is on {h.device}, the layer on {self.ws.device}")
        call("cia_moe_block_forward", ctypes.byref(self._m), h.data_ptr(), S, _stream_on(h.get_device()))


# ------------------------------------------------------------ many sequences
class PageTable:
    """Which pages hold the tokens of each of ``max_seqs`` sequences: token ``pos`` of
    sequence ``s`` lies in page ``table[s, pos // page]``, -1 where it has none.  The
    layers of a model share one: ``n_pages`` pages of ``page`` tokens in each of them,
    given out and taken back on the host, and written to ``table`` on the current stream,
    which must not be capturing a graph."""

    def __init__(self, max_seqs: int, max_tokens: int, n_pages: int, *, page: int = 64, device="cuda"):
        if not PAGE_MIN <= page <= PAGE_MAX or page & (page - 1):
            raise ValueError(f"page={page}: need a power of two, {PAGE_MIN} to {PAGE_MAX}")
        for n, name in ((max_seqs, "max_seqs"), (max_tokens, "max_tokens"), (n_pages, "n_pages")):
            if n < 1:
                raise ValueError(f"{name}={n}: need 1 or more")
        if max_tokens > PAGES_MAX_TOKENS:
            raise ValueError(f"max_tokens={max_tokens}: a sequence holds {PAGES_MAX_TOKENS} at most")
        self.page, self.n_pages = page, n_pages
        width = -(-max_tokens // page)
        self.table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=device)
        self._held = [[] for _ in range(max_seqs)]
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _row(self, seq: int):
        if not 0 <= seq < len(self._held):
            raise ValueError(f"seq={seq}: the table has {len(self._held)} sequences")
        return self._held[seq]

    def _no_capture(self) -> None:
        if self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages change hands outside a graph's capture: a replay would do it again")

    def reserve(self, seq: int, tokens: int) -> None:
        """Pages for the first ``tokens`` tokens of a sequence, those it has among them.
        Raises RuntimeError, with nothing changed, where not enough are free."""
        held = self._row(seq)
        need = -(-tokens // self.page) - len(held)
        if need <= 0:
            return
        if len(held) + need > self.table.shape[1]:
            raise ValueError(f"tokens={tokens}: a sequence holds {self.table.shape[1] * self.page}")
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} free")
        new = self._free[:-need - 1:-1]
        self._no_capture()
        self.table[seq, len(held):len(held) + need] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        del self._free[-need:]  # (once they are in the table)
        held += new

    def release(self, seq: int) -> None:
        """A sequence's pages back; its row of the table is -1.  Work that still reads
        them has to lie before what writes them next (the same stream, or events)."""
        held = self._row(seq)
        self._no_capture()
        self.table[seq] = -1
        self._free += reversed(held)
        self._held[seq] = []


class PagedAttn:
    """Attention of one layer for a batch of sequences, over pages that ``table`` gives
    out: e4m3 with an fp16 scale per token and kv head (engine.cu:317-333), or fp16
    with ``quant=False``.  ``scale``: of the scores, 1 / sqrt(head_dim) if None;
    ``window``: tokens attended to, 0 for all.  Positions are int32 device tensors, -1
    for an empty place of a batch; ``seq`` is the tokens' sequences, None: token t is
    sequence t's.  The layer's making, which clears its buffers, and its calls must be
    ordered on one stream."""

    def __init__(self, table: PageTable, *, n_q: int = NH, n_kv: int = NKV, head_dim: int = D, quant: bool = True,
                 scale=None, window: int = 0):
        dev, shape = table.table.device, (table.n_pages, n_kv, table.page, head_dim)
        new = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=dev)  # noqa: E731
        kv = [new(shape, torch.uint8 if quant else torch.float16) for _ in range(2)]
        scales = [new(shape[:3], torch.float16) for _ in range(2)] if quant else [None, None]
        self.table = table
        self.pages = KvPages(*kv, table.table, *scales)
        self.ws = new_attn_pages_workspace(self.pages, n_q)
        self.scale, self.window = head_dim ** -0.5 if scale is None else float(scale), window

    def write(self, k, v, pos, seq=None) -> None:
        """k, v fp16 [T, kv heads, dim] to their places."""
        kv_pages_write(self.pages, k, v, pos, seq=seq)

    def read(self, k, v, pos, seq=None) -> None:
        """Rows of k, v fp16 [T, kv heads, dim] from their places."""
        kv_pages_read(self.pages, k, v, pos, seq=seq)

    def attend(self, q, pos, seq=None, out=None):
        """out fp16 [T, query heads, dim] of q over its sequences' tokens up to pos."""
        if out is None:
            out = torch.empty(q.shape, dtype=torch.float16, device=q.device)
        attn_pages(self.pages, q, out, pos, self.ws, seq=seq, scale=self.scale, window=self.window)
        return out

    def decode(self, q, k, v, pos, seq=None, out=None):
        """One token of each sequence: its k and v written, then q attended."""
        self.write(k, v, pos, seq=seq)
        return self.attend(q, pos, seq=seq, out=out)
