"""The reference engine's attention kernels as Python calls on torch tensors.

Each function keeps the name, argument order and meaning of one kernel of
g023/cuda_inf ``src/engine.cu`` and runs the gfx950 implementation through the
C-ABI of libcuda_inf_attn.so on torch's current stream.  fp16 tensors may be
``torch.float16`` or ``torch.int16``/``torch.uint16`` bit patterns.  Errors
raise ``CiaError``; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import D, KVGROUP, NH, NKV, NSPLIT_DEFAULT, call

_F16 = (torch.float16, torch.int16, torch.uint16)


# torch's own short way to the current stream's handle; no public name, so a
# build of torch without it takes the long way
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle() -> int:
    """The hipStream_t of torch's current stream on the current device: the
    value of ``torch.cuda.current_stream().cuda_stream`` without the stream
    object (2.8 -> 0.3 us, of an 8.3 us gemv_int4 call of one row, whose
    kernel takes 2.9).  Read on every call, like that one."""
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _dev(t: torch.Tensor, name: str, dtypes=None, numel=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if numel is not None and t.numel() < numel:
        raise ValueError(f"{name}: needs at least {numel} elements, has {t.numel()}")
    return t.data_ptr()


def _opt(t, name, dtypes=None, numel=None):
    return None if t is None else _dev(t, name, dtypes, numel)


def e4m3_encode_range(first_bits: int, n: int, out) -> None:
    """Device E4M3 encoder on the fp32 bit patterns first_bits .. first_bits+n-1."""
    call("cia_e4m3_encode_range", first_bits, n, _dev(out, "out", (torch.uint8,), n), stream_handle())


# ------------------------------------------------------------ group-64 cache
def kv_write_tail(k, v, ktail, vtail, slot: int, cnt: int) -> None:
    """engine.cu:190-198: tail rows slot..slot+cnt-1 <- k, v [cnt, 8, 64]."""
    n = cnt * NKV * D
    call("cia_kv_write_tail", _dev(k, "k", _F16, n), _dev(v, "v", _F16, n),
         _dev(ktail, "ktail", _F16, KVGROUP * NKV * D), _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         slot, cnt, stream_handle())


def kv_commit_group(ktail, vtail, kc8, vc8, ksc, vsc, dst_tok_base: int, grp: int) -> None:
    """engine.cu:202-228: commit the full tail group to FP8 with fp16 scales."""
    call("cia_kv_commit_group", _dev(ktail, "ktail", _F16, KVGROUP * NKV * D),
         _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         _dev(kc8, "kc8", (torch.uint8,), (dst_tok_base + KVGROUP) * NKV * D),
         _dev(vc8, "vc8", (torch.uint8,), (dst_tok_base + KVGROUP) * NKV * D),
         _dev(ksc, "ksc", _F16, (grp + 1) * NKV), _dev(vsc, "vsc", _F16, (grp + 1) * NKV),
         dst_tok_base, grp, stream_handle())


# ------------------------------------------------------------ attention
def attention_fused(q, kc8, vc8, ksc, vsc, ktail, vtail, committed: int, out, attn_sum,
                    S: int, past: int, scale: float, ws=None) -> None:
    """engine.cu:236-308: causal attention of S queries at past..past+S-1."""
    T = past + S
    call("cia_attention_fused", _dev(q, "q", _F16, S * NH * D),
         _dev(kc8, "kc8", (torch.uint8,), min(T, committed) * NKV * D),
         _dev(vc8, "vc8", (torch.uint8,), min(T, committed) * NKV * D),
         _dev(ksc, "ksc", _F16), _dev(vsc, "vsc", _F16),
         _dev(ktail, "ktail", _F16, KVGROUP * NKV * D), _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         committed, _dev(out, "out", _F16, S * NH * D),
         _opt(attn_sum, "attn_sum", (torch.float32,), T), S, past, float(scale),
         _opt(ws, "ws", None, mass_workspace_bytes(S) if attn_sum is not None else None),
         ws.numel() * ws.element_size() if ws is not None else 0, stream_handle())


def attention_fused_fp8(q, kc8, vc8, ksc, vsc, ktail, vtail, committed: int, out, S: int,
                        past: int, scale: float) -> None:
    """attention_fused's causal attention on the OCP-fp8 matrix cores (Q and
    the softmax numerators rounded to fp8; error reported, not bounded by
    the fp16 path's tolerance)."""
    T = past + S
    call("cia_attention_fused_fp8", _dev(q, "q", _F16, S * NH * D),
         _dev(kc8, "kc8", (torch.uint8,), min(T, committed) * NKV * D),
         _dev(vc8, "vc8", (torch.uint8,), min(T, committed) * NKV * D),
         _dev(ksc, "ksc", _F16), _dev(vsc, "vsc", _F16),
         _dev(ktail, "ktail", _F16, KVGROUP * NKV * D), _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         committed, _dev(out, "out", _F16, S * NH * D), S, past, float(scale), stream_handle())


def attn_decode_split(q, kc8, vc8, ksc, vsc, ktail, vtail, committed: int, qpos: int,
                      scale: float, pm, pl, po, nsplit: int = NSPLIT_DEFAULT, ws=None) -> None:
    """engine.cu:396-464 with a runtime split count.  ws (optional): a
    workspace of split_workspace_bytes(nsplit) bytes, zeroed before its first
    use, in place of the library's fixed device array."""
    args = (_dev(q, "q", _F16, NH * D),
            _dev(kc8, "kc8", (torch.uint8,)), _dev(vc8, "vc8", (torch.uint8,)),
            _dev(ksc, "ksc", _F16), _dev(vsc, "vsc", _F16),
            _dev(ktail, "ktail", _F16, KVGROUP * NKV * D),
            _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
            committed, qpos, float(scale),
            _dev(pm, "pm", (torch.float32,), NH * nsplit),
            _dev(pl, "pl", (torch.float32,), NH * nsplit),
            _dev(po, "po", (torch.float32,), NH * nsplit * D), nsplit)
    if ws is None:
        call("cia_attn_decode_split", *args, stream_handle())
    else:
        call("cia_attn_decode_split_ws", *args,
             _dev(ws, "ws", (torch.uint8,), split_workspace_bytes(nsplit)), ws.numel(), stream_handle())


def split_workspace_bytes(nsplit: int) -> int:
    """Workspace bytes of attn_decode_split's caller-workspace form."""
    return int(_lib.lib().cia_split_workspace_bytes(nsplit))


def attn_decode_combine(pm, pl, po, out, nsplit: int = NSPLIT_DEFAULT) -> None:
    """engine.cu:467-480 with a runtime split count."""
    call("cia_attn_decode_combine", _dev(pm, "pm", (torch.float32,), NH * nsplit),
         _dev(pl, "pl", (torch.float32,), NH * nsplit),
         _dev(po, "po", (torch.float32,), NH * nsplit * D), _dev(out, "out", _F16, NH * D),
         nsplit, stream_handle())


def decode_workspace_bytes(max_tokens: int) -> int:
    """Scratch bytes of attn_decode for contexts of up to max_tokens keys."""
    return int(_lib.lib().cia_decode_workspace_bytes(max_tokens))


def new_decode_workspace(max_tokens: int, device="cuda") -> torch.Tensor:
    """Workspace of attn_decode: partial softmax states and per-kv-head
    arrival counters.  Zeroed here; every call leaves the counters at zero."""
    return torch.zeros(decode_workspace_bytes(max_tokens), dtype=torch.uint8, device=device)


def attn_decode(q, kc8, vc8, ksc, vsc, ktail, vtail, committed: int, qpos: int, scale: float,
                out, ws) -> None:
    """Flash-decoding on the matrix cores with the library's own split, one
    launch (replaces engine.cu:848-852's split + combine launches).  Calls
    sharing ws must be ordered on one stream."""
    call("cia_attn_decode", _dev(q, "q", _F16, NH * D),
         _dev(kc8, "kc8", (torch.uint8,)), _dev(vc8, "vc8", (torch.uint8,)),
         _dev(ksc, "ksc", _F16), _dev(vsc, "vsc", _F16),
         _dev(ktail, "ktail", _F16, KVGROUP * NKV * D), _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         committed, qpos, float(scale), _dev(out, "out", _F16, NH * D),
         _dev(ws, "ws", (torch.uint8,), decode_workspace_bytes(qpos + 1)), ws.numel(), stream_handle())


def attn_decode_noalloc(q, kc8, vc8, ksc, vsc, ktail, vtail, committed: int, qpos: int,
                        scale: float, out) -> None:
    """attn_decode with the library's own fixed workspace (allocates
    nothing; calls overlapping on one GPU race)."""
    call("cia_attn_decode_noalloc", _dev(q, "q", _F16, NH * D),
         _dev(kc8, "kc8", (torch.uint8,)), _dev(vc8, "vc8", (torch.uint8,)),
         _dev(ksc, "ksc", _F16), _dev(vsc, "vsc", _F16),
         _dev(ktail, "ktail", _F16, KVGROUP * NKV * D), _dev(vtail, "vtail", _F16, KVGROUP * NKV * D),
         committed, qpos, float(scale), _dev(out, "out", _F16, NH * D), stream_handle())


# ------------------------------------------------------------ H2O
def kv_quant_write(k, v, kf, vf, ks, vs, dst_slots, S: int) -> None:
    """engine.cu:317-333: per-token FP8 quantisation into slots dst_slots[j]."""
    call("cia_kv_quant_write", _dev(k, "k", _F16, S * NKV * D), _dev(v, "v", _F16, S * NKV * D),
         _dev(kf, "kf", (torch.uint8,)), _dev(vf, "vf", (torch.uint8,)),
         _dev(ks, "ks", _F16), _dev(vs, "vs", _F16),
         _dev(dst_slots, "dst_slots", (torch.int32,), S), S, stream_handle())


def h2o_place(k, v, kf, vf, ks, vs, attn_sum, slot_pos, dst_slots, n_live: int, C: int, W: int,
              S: int, past: int) -> int:
    """engine.cu:808-826 on the device: slot choice + per-token quantisation.

    Updates attn_sum, slot_pos, dst_slots in place; returns the new n_live."""
    nl = ctypes.c_int(n_live)
    call("cia_h2o_place", _dev(k, "k", _F16, S * NKV * D), _dev(v, "v", _F16, S * NKV * D),
         _dev(kf, "kf", (torch.uint8,), C * NKV * D), _dev(vf, "vf", (torch.uint8,), C * NKV * D),
         _dev(ks, "ks", _F16, C * NKV), _dev(vs, "vs", _F16, C * NKV),
         _dev(attn_sum, "attn_sum", (torch.float32,), C),
         _dev(slot_pos, "slot_pos", (torch.int32,), C),
         _dev(dst_slots, "dst_slots", (torch.int32,), S), ctypes.byref(nl), C, W, S, past,
         stream_handle())
    return nl.value


def mass_workspace_bytes(S: int) -> int:
    return int(_lib.lib().cia_mass_workspace_bytes(S))


def h2o_workspace_bytes(S: int, C: int) -> int:
    return int(_lib.lib().cia_h2o_workspace_bytes(S, C))


def attention_h2o(q, kf, vf, ks, vs, slot_pos, n_live: int, out, attn_sum, S: int, past: int,
                  scale: float, ws) -> None:
    """engine.cu:337-384 with the deterministic attention-mass rule; ws is a
    uint8 device tensor of at least h2o_workspace_bytes(S, n_live) bytes."""
    call("cia_attention_h2o", _dev(q, "q", _F16, S * NH * D),
         _dev(kf, "kf", (torch.uint8,), n_live * NKV * D), _dev(vf, "vf", (torch.uint8,), n_live * NKV * D),
         _dev(ks, "ks", _F16, n_live * NKV), _dev(vs, "vs", _F16, n_live * NKV),
         _dev(slot_pos, "slot_pos", (torch.int32,), n_live), n_live,
         _dev(out, "out", _F16, S * NH * D), _dev(attn_sum, "attn_sum", (torch.float32,), n_live),
         S, past, float(scale), _dev(ws, "ws", (torch.uint8,), h2o_workspace_bytes(S, n_live)),
         ws.numel(), stream_handle())


# ------------------------------------------------------------ QK producers
def qk_norm_rope(q, k, qw, kw, pos, S: int, eps: float = 1e-5, theta: float = 5.0e6) -> None:
    """engine.cu:799-801 (rmsnorm_head on q and k, then rope) in place, one launch."""
    call("cia_qk_norm_rope", _dev(q, "q", _F16, S * NH * D), _dev(k, "k", _F16, S * NKV * D),
         _dev(qw, "qw", _F16, D), _dev(kw, "kw", _F16, D), _dev(pos, "pos", (torch.int32,), S),
         S, float(eps), float(theta), stream_handle())


# ------------------------------------------------------------ INT4 projections
def _int4(packed, scales, N: int, K: int, name: str):
    return (_dev(packed, name + ".packed", (torch.uint8,), N * K // 2),
            _dev(scales, name + ".scales", _F16, N * K // 128))


def gemv_int4(x, packed, scales, y, N: int, K: int, M: int, add: bool = False) -> None:
    """engine.cu:83-109 / 626-630: y fp32 [M, N] = x [M, K] W^T for INT4
    group-128 W (packed u8 [N, K/2], scales fp16 [N, K/128]); add=True
    accumulates into y (out_proj + residual, engine.cu:858-859)."""
    p, s = _int4(packed, scales, N, K, "w")
    call("cia_gemv_int4_add" if add else "cia_gemv_int4", _dev(x, "x", _F16, M * K), p, s,
         _dev(y, "y", (torch.float32,), M * N), N, K, M, stream_handle())


def qkv_proj_int4(x, wq, wk, wv, q, k, v, M: int, K: int = 2048) -> None:
    """engine.cu:792-797 in one launch: q/k/v fp16 = fp16(x W^T); wq, wk, wv
    are (packed, scales) pairs with N = q.shape[-1] / k.shape[-1] rows."""
    Nq = q.numel() // M
    Nkv = k.numel() // M
    pq, sq = _int4(*wq, Nq, K, "wq")
    pk, sk = _int4(*wk, Nkv, K, "wk")
    pv, sv = _int4(*wv, Nkv, K, "wv")
    call("cia_qkv_proj_int4", _dev(x, "x", _F16, M * K), pq, sq, Nq, pk, sk, pv, sv, Nkv, K, M,
         _dev(q, "q", _F16, M * Nq), _dev(k, "k", _F16, M * Nkv), _dev(v, "v", _F16, M * Nkv),
         stream_handle())


# ------------------------------------------------------------ feed-forward branch
# A decode token's call of these is bound by the host, so a tensor is looked at in one
# condition, and again in detail where it does not hold (moe_up_int4 of one token: 7.5
# us of host time, 8.7 with _dev() for each; the foreign call with its launch is 3.9).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _at(t, name: str, dtypes, numel: int, dev: int):
    """_dev() of a tensor that has to be on device dev."""
    try:
        if t.get_device() == dev and t.is_contiguous() and t.dtype in dtypes and t.numel() >= numel:
            return t.data_ptr()
    except AttributeError:
        pass  # no tensor
    _dev(t, name, dtypes, numel)
    raise ValueError(f"{name}: on {t.device}, and other tensors of the call on cuda:{dev}")


def _stream_on(dev: int) -> int:
    """stream_handle() of device dev, which has to be the current one, where the
    call runs."""
    if _current_device() != dev:
        raise ValueError(f"the tensors are on cuda:{dev}, the current device is cuda:{_current_device()}")
    return stream_handle() if _raw_stream is None else _raw_stream(dev)


_F32, _I32, _U8 = (torch.float32,), (torch.int32,), (torch.uint8,)


def add_rmsnorm(h, w, out, S: int, H: int, eps: float = 1e-5, add=None, hsum=None) -> None:
    """add_f32_inplace (engine.cu:867) and rmsnorm (870): hsum = h + add (fp32 [S, H];
    add and hsum optional, hsum may be h or add), out = fp16(hsum *
    rsqrt(mean(hsum^2) + eps) * w)."""
    hp, dev, n = _dev(h, "h", _F32, S * H), h.get_device(), S * H
    call("cia_add_rmsnorm", hp, None if add is None else _at(add, "add", _F32, n, dev), _at(w, "w", _F16, H, dev),
         eps, None if hsum is None else _at(hsum, "hsum", _F32, n, dev), _at(out, "out", _F16, n, dev), S, H,
         _stream_on(dev))


def moe_gating(E: int, k: int, score: str = "sigmoid", n_group: int = 1, topk_group: int = 1,
               renorm: bool = True, eps: float = 1e-6, scale: float = 1.0):
    """How a router chooses, as moe_route and moe_select take it."""
    if score not in _lib.SCORES:
        raise ValueError(f"score: {score!r} is not one of {sorted(_lib.SCORES)}")
    return _lib.cia_moe_gating(E, k, _lib.SCORES[score], n_group, topk_group, bool(renorm), eps, scale)


def moe_route(x, gate, ids, weights, S: int, H: int, E: int, k: int, bias=None, logits=None,
              **gating) -> None:
    """The router of engine.cu:869-905 on the device: the k experts of each of the S
    rows of x (fp16 [S, H]; gate fp16 [E, H]; bias fp32 [E], for the choice alone)
    into ids int32 [S, k] and weights fp32 [S, k]; logits fp32 [S, E], optional.
    gating: score, n_group, topk_group, renorm, eps, scale, as moe_gating."""
    xp, dev = _dev(x, "x", _F16, S * H), x.get_device()
    call("cia_moe_route", xp, _at(gate, "gate", _F16, E * H, dev),
         None if bias is None else _at(bias, "bias", _F32, E, dev), ctypes.byref(moe_gating(E, k, **gating)),
         _at(ids, "ids", _I32, S * k, dev), _at(weights, "weights", _F32, S * k, dev),
         None if logits is None else _at(logits, "logits", _F32, S * E, dev), S, H, _stream_on(dev))


def moe_select(logits, ids, weights, S: int, E: int, k: int, bias=None, **gating) -> None:
    """moe_route from logits fp32 [S, E] that the caller has."""
    lp, dev = _dev(logits, "logits", _F32, S * E), logits.get_device()
    call("cia_moe_select", lp, None if bias is None else _at(bias, "bias", _F32, E, dev),
         ctypes.byref(moe_gating(E, k, **gating)), _at(ids, "ids", _I32, S * k, dev),
         _at(weights, "weights", _F32, S * k, dev), S, _stream_on(dev))


def q4_experts(w, name: str):
    """(cia_q4_experts, E, rows, cols) of INT4 group-128 experts: w = (packed u8
    [E, rows, cols / 2], scales fp16 [E, rows, cols / 128]) on the device.  Each
    expert is contiguous; the experts may lie apart, at one stride."""
    return _q4(w, name, None)


def _q4(w, name: str, dev):
    """q4_experts of a call whose tensors are on device dev (None: any)."""
    packed, scales = w
    try:
        E, rows, half = packed.shape
        groups = half // 64
        on = packed.get_device() if dev is None else dev
        if (on >= 0 and packed.get_device() == on and scales.get_device() == on and packed.dtype is torch.uint8
                and scales.dtype in _F16 and half == 64 * groups and scales.shape == (E, rows, groups)):
            if packed.is_contiguous() and scales.is_contiguous():
                return (_lib.cia_q4_experts(packed.data_ptr(), scales.data_ptr(), rows * half, rows * groups),
                        E, rows, 2 * half)
            ps, ss = packed.stride(), scales.stride()
            if ps[1:] == (half, 1) and ss[1:] == (groups, 1):
                return _lib.cia_q4_experts(packed.data_ptr(), scales.data_ptr(), ps[0], ss[0]), E, rows, 2 * half
    except (AttributeError, ValueError):
        pass  # no tensors, or not of three dimensions
    if not (isinstance(packed, torch.Tensor) and isinstance(scales, torch.Tensor) and packed.dim() == 3
            and scales.dim() == 3):
        raise ValueError(f"{name}: need two tensors [experts, rows, columns], packed and scales")
    for t, part, dtypes in ((packed, ".packed", _U8), (scales, ".scales", _F16)):
        if not t.is_cuda:
            raise ValueError(f"{name}{part}: must be a device tensor")
        if t.dtype not in dtypes:
            raise TypeError(f"{name}{part}: dtype {t.dtype} not in {dtypes}")
        if t.stride()[1:] != (t.shape[2], 1):
            raise ValueError(f"{name}{part}: an expert must be contiguous")
    if packed.get_device() != scales.get_device() or dev not in (None, packed.get_device()):
        raise ValueError(f"{name}: packed is on {packed.device}, scales on {scales.device}"
                         + ("" if dev is None else f", other tensors of the call on cuda:{dev}"))
    raise ValueError(f"{name}: packed {tuple(packed.shape)} and scales {tuple(scales.shape)} do not fit: "
                     "[E, rows, cols / 2] and [E, rows, cols / 128], cols a multiple of 128")


def moe_workspace_bytes(S: int, k: int, E: int, H: int, F: int) -> int:
    """Workspace bytes of moe_up_int4 and moe_down_int4 for up to S tokens."""
    return int(_lib.lib().cia_moe_workspace_bytes(S, k, E, H, F))


def moe_up_int4(x, ids, w1, w3, act, S: int, k: int, ws) -> None:
    """w1, w3 and swiglu of engine.cu:869-905 for every token and chosen expert:
    act [S, k, F] fp16 = silu(W1[e] x) * (W3[e] x), e = ids[s, j]; x fp16 [S, H],
    ids int32 [S, k] (outside [0, E): the pair's act row is left as it was; None:
    one expert, every row), w1 and w3 as q4_experts takes them, [E, F, H]."""
    q1, E, F, H = _q4(w1, "w1", None)
    dev = w1[0].get_device()
    q3, E3, F3, H3 = _q4(w3, "w3", dev)
    if F3 != F or H3 != H or E3 != E:
        raise ValueError(f"w3: experts {(E3, F3, H3)}, but w1 has {(E, F, H)}")
    call("cia_moe_up_int4", _at(x, "x", _F16, S * H, dev), None if ids is None else _at(ids, "ids", _I32, S * k, dev),
         ctypes.byref(q1), ctypes.byref(q3), _at(act, "act", _F16, S * k * F, dev), S, k, E, H, F,
         _at(ws, "ws", _U8, 0, dev), ws.numel(), _stream_on(dev))


def moe_down_int4(act, ids, weights, w2, res, out, S: int, k: int, ws) -> None:
    """w2 and acc_scaled of engine.cu:869-905 for every token and chosen expert:
    out [S, H] fp32 = res + sum over j of weights[s, j] * (W2[e] act[s, j]); out may
    be res; weights fp32 [S, k] or None (1); ids as moe_up_int4's; w2 [E, H, F]."""
    q2, E, H, F = _q4(w2, "w2", None)
    dev, n = w2[0].get_device(), S * k
    call("cia_moe_down_int4", _at(act, "act", _F16, n * F, dev), None if ids is None else _at(ids, "ids", _I32, n, dev),
         None if weights is None else _at(weights, "weights", _F32, n, dev), ctypes.byref(q2),
         _at(res, "res", _F32, S * H, dev), _at(out, "out", _F32, S * H, dev), S, k, E, H, F,
         _at(ws, "ws", _U8, 0, dev), ws.numel(), _stream_on(dev))


# ------------------------------------------------------------ a batch's decode step
class KvPages:
    """One layer's paged key-value cache for many sequences, as kv_pages_write,
    kv_pages_read and attn_pages take it (cia_kv_pages).

    ``k``, ``v``: [pages, kv heads, page, dim], contiguous, fp16, or u8 (e4m3) with
    ``ks``, ``vs`` fp16 [pages, kv heads, page].  ``table``: int32 [sequences, columns],
    the pages of each sequence in order; rows may lie apart.  Its contents may change
    between calls, as the pages' may; the tensors are kept."""

    def __init__(self, k, v, table, ks=None, vs=None):
        if not isinstance(k, torch.Tensor) or k.dim() != 4 or not k.numel():
            raise ValueError("k: need a tensor [pages, kv heads, page, dim]")
        quant = k.dtype == torch.uint8
        if not quant and k.dtype not in _F16:
            raise TypeError(f"k: dtype {k.dtype}: need fp16, or uint8 for e4m3")
        kp, dev, n = _dev(k, "k"), k.get_device(), k.numel()
        vp = _at(v, "v", (k.dtype,), n, dev)
        rows = n // k.shape[3]
        if quant:
            sp = [_at(t, name, _F16, rows, dev) for t, name in ((ks, "ks"), (vs, "vs"))]
        elif ks is not None or vs is not None:
            raise ValueError("ks, vs: fp16 pages have no scales")
        else:
            sp = [None, None]
        for t, name, like in ((v, "v", k.shape), (ks, "ks", k.shape[:3]), (vs, "vs", k.shape[:3])):
            if t is not None and t.shape != like:
                raise ValueError(f"{name}: shape {tuple(t.shape)}, and k's is {tuple(k.shape)}")
        if (not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.int32
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            raise ValueError("table: need an int32 tensor [sequences, columns], rows contiguous")
        if table.get_device() != dev:
            raise ValueError(f"table: on {table.device}, and the pages on cuda:{dev}")
        n_pages, n_kv, page, dim = k.shape
        stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        self._s = _lib.cia_kv_pages(kp, vp, *sp, 0 if quant else 1, n_pages, page, n_kv, dim, table.shape[0],
                                    table.shape[1], table.data_ptr(), stride)
        self._ref, self._device, self._n_seq = ctypes.byref(self._s), dev, table.shape[0]
        self.k, self.v, self.ks, self.vs, self.table = k, v, ks, vs, table
        self.n_kv, self.head_dim, self.page = n_kv, dim, page


def _rows(t, name: str, heads: int, dim: int, T: int, dev: int):
    """Address and row stride of fp16 rows [T, heads, dim], each contiguous."""
    try:
        if (t.get_device() == dev and t.dtype in _F16 and t.shape == (T, heads, dim)
                and (t.is_contiguous() or (t.stride(2) == 1 and (heads == 1 or t.stride(1) == dim)))):
            return t.data_ptr(), t.stride(0) if T > 1 else heads * dim
    except AttributeError:
        pass  # no tensor
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in _F16:
        raise TypeError(f"{name}: dtype {t.dtype} not in {_F16}")
    raise ValueError(f"{name}: {tuple(t.shape)} on {t.device}: need rows [{T}, {heads}, {dim}], each contiguous, "
                     f"on cuda:{dev}")


def _tokens(pos) -> int:
    if not isinstance(pos, torch.Tensor):
        raise TypeError(f"pos: expected a torch.Tensor, got {type(pos).__name__}")
    return pos.numel()


def _move(fn: str, pages: KvPages, k, v, pos, seq) -> None:
    T, dev = _tokens(pos), pages._device
    kp, ks = _rows(k, "k", pages.n_kv, pages.head_dim, T, dev)
    vp, vs = _rows(v, "v", pages.n_kv, pages.head_dim, T, dev)
    call(fn, pages._ref, kp, ks, vp, vs, None if seq is None else _at(seq, "seq", _I32, T, dev),
         _at(pos, "pos", _I32, T, dev), T, _stream_on(dev))


def kv_pages_write(pages: KvPages, k, v, pos, seq=None) -> None:
    """k and v (fp16 [T, kv heads, dim], rows may lie apart) into the pages at
    positions ``pos`` (int32 [T]) of sequences ``seq`` (int32 [T]; None: token t is
    sequence t's), quantised as kv_quant_write does (engine.cu:317-333) in an e4m3
    cache.  A position of -1, or one without a page, is passed over; two tokens of a
    call must not have one place."""
    _move("cia_kv_pages_write", pages, k, v, pos, seq)


def kv_pages_read(pages: KvPages, k, v, pos, seq=None) -> None:
    """The reverse of kv_pages_write: k and v rows from the pages, fp16; rows of
    tokens without a place are left as they were."""
    _move("cia_kv_pages_read", pages, k, v, pos, seq)


def attn_pages_workspace_bytes(n_q: int, n_kv: int, head_dim: int) -> int:
    """Workspace bytes of attn_pages, for any number of rows."""
    return int(_lib.lib().cia_attn_pages_workspace_bytes(n_q, n_kv, head_dim))


def new_attn_pages_workspace(pages: KvPages, n_q: int) -> torch.Tensor:
    """Workspace of attn_pages over these pages with n_q query heads.  Zeroed here;
    every call leaves its counters at zero."""
    n = attn_pages_workspace_bytes(n_q, pages.n_kv, pages.head_dim)
    if not n:
        raise ValueError(f"{n_q} query heads on {pages.n_kv} kv heads of {pages.head_dim}: beyond what a call takes")
    return torch.zeros(n, dtype=torch.uint8, device=pages.k.device)


def attn_pages(pages: KvPages, q, out, pos, ws, seq=None, scale: float = 0.125, window: int = 0) -> None:
    """Attention of one query token per row over its sequence's pages: q fp16 [T, query
    heads, dim] (rows may lie apart) at positions ``pos`` (int32 [T]) of ``seq`` (int32
    [T]; None: row t is sequence t's), into out fp16 [T, query heads, dim]; all tokens
    up to pos, the last ``window`` of them if window > 0.  Rows with none (pos -1) are
    0.  Calls sharing ws must be ordered on one stream, after what zeroed it."""
    T, dev = _tokens(pos), pages._device
    n_q = q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    qp, qs = _rows(q, "q", n_q, pages.head_dim, T, dev)
    call("cia_attn_pages", pages._ref, qp, qs, None if seq is None else _at(seq, "seq", _I32, T, dev),
         _at(pos, "pos", _I32, T, dev), T, n_q, scale, window,
         _at(out, "out", _F16, T * n_q * pages.head_dim, dev), _at(ws, "ws", _U8, 0, dev), ws.numel(), _stream_on(dev))


_LOGITS = {torch.float32: 0, torch.float16: 1}  # CIA_LOGITS_*


def sample_workspace_bytes(B: int, V: int) -> int:
    """Workspace bytes of sample for up to B rows of V logits."""
    return int(_lib.lib().cia_sample_workspace_bytes(B, V))


def sample(logits, u, ids, ws, temperature=None, top_k=None, top_p=None, min_p=None, p=None) -> None:
    """A token for each row of logits (fp32 or fp16 [B, V], rows may lie apart) from the
    given random numbers u (fp32 [B], in [0, 1)) into ids (int32 [B]), after
    temperature (0: the largest logit), top_k, top_p and min_p in this order (fp32 [B],
    top_k int32 [B]; None: 1, and no filter); p (fp32 [B], optional): the probability it
    was drawn with.  In place of argmax_kernel (engine.cu:562-572)."""
    try:
        B, V = logits.shape
        kind, dev = _LOGITS[logits.dtype], logits.get_device()
    except (AttributeError, KeyError, ValueError):
        raise ValueError("logits: need a device tensor [B, V] of fp32 or fp16") from None
    if dev < 0 or (V > 1 and logits.stride(1) != 1):
        raise ValueError("logits: need a device tensor [B, V], rows contiguous")
    f = [None if t is None else _at(t, name, d, B, dev) for t, name, d in (
        (temperature, "temperature", _F32), (top_k, "top_k", _I32), (top_p, "top_p", _F32), (min_p, "min_p", _F32))]
    call("cia_sample", logits.data_ptr(), kind, logits.stride(0) if B > 1 else V, *f, _at(u, "u", _F32, B, dev),
         _at(ids, "ids", _I32, B, dev), None if p is None else _at(p, "p", _F32, B, dev), B, V,
         _at(ws, "ws", _U8, 0, dev), ws.numel(), _stream_on(dev))
