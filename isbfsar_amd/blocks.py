"""The operators of a cross-attention layer over feature sequences (include/isbfsar.h: isb_xattn_*, isb_ffn_*, isb_norm_*).

They stand beside the tuple attention, the MLPs and the LayerNorm that live inside :class:`isbfsar_amd.engine.ArEngine` and work on
what it hands out: the embeddings of query windows ([B, L, 256], ``infer(want_embed=True)``) and the frames of a support set
(``support_features()``), both f32: :func:`cross_attention` and :func:`gated_ffn` take them as fp16 or bf16 (``.half()``)::

    n = block_norm(x, pre="layer", pre_weight=w, pre_bias=b)                      # norm before the block
    out, lse = cross_attention(q, k, v, kv_len=lengths)                           # windows against the support set's frames
    x, n = block_norm(x, proj(out), scale=s, pre="layer", ...)                    # residual sum + the next block's norm, one pass
    y = gated_ffn(n, w_gate, w_up, w_down)

torch owns the device memory and the stream (the tensors' current stream); every call is asynchronous on it, allocates its results and
its workspace with torch and may be captured into a graph. Backward passes are calls of their own and take what the forward call
returned; nothing is recorded on an autograd tape. A tensor that requires a gradient is therefore refused while gradients are recorded (the
result would not carry it): call under torch.no_grad(), or detach; parameters then take the gradients that the backward calls return. Forward-mode
tangents are refused likewise.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
NORMS = {None: 0, "layer": 1, "rms": 2}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_HALF = (torch.float16, torch.bfloat16)


def _refuse(msg: str):
    raise ValueError(msg)


def _on_tape(name: str):
    _refuse(f"{name} requires a gradient, which no result would carry: call under torch.no_grad() or detach it (gradients: the backward calls)")


def _tangents(*tensors) -> None:
    """called inside forward_ad.dual_level only"""
    for t in tensors:
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            _refuse("a tensor has a forward-mode tangent, which no result would carry")


def _first(name: str, t, types) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.dtype not in types:
        raise TypeError(f"{name} is {t.dtype}, expected one of {sorted(str(x) for x in types)}")
    if t.requires_grad and torch.is_grad_enabled():
        _on_tape(name)


def _tensor(name: str, t, dtype, dev: int, shape) -> None:
    if not (isinstance(t, torch.Tensor) and (t.get_device() == dev or t.is_cuda)):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} lives on {t.device}, the first tensor on cuda:{dev}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected {tuple(shape)}, got {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        _on_tape(name)


_FAR = 1 << 22         # elements between the rows that a kernel steps through, at most (include/isbfsar.h)


def _rows16(t: torch.Tensor, walked: Optional[int] = None):
    """(t, its leading strides), or a contiguous copy where its last dimension is not contiguous, its rows do not lie on 16 bytes or those along
    dimension `walked` lie too far apart"""
    st = t.stride()
    bits = t.data_ptr() & 15
    for s in st[:-1]:
        bits |= s & 7
    if bits == 0 and st[-1] == 1 and (walked is None or st[walked] <= _FAR):
        return t, st[:-1]
    t = _flat16(t)
    st, n = [], 1
    for d in reversed(t.shape):                  # (torch leaves the strides of dimensions of size 1 as they were)
        st.append(n)
        n *= d
    return t, tuple(reversed(st))[:-1]


def _flat16(t: torch.Tensor) -> torch.Tensor:
    """t contiguous on 16 bytes"""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _workspace(fn, what: str, args, *more) -> int:
    n = C.c_size_t()
    rc = fn(C.byref(args), *more, C.byref(n))
    if rc:
        _lib.check(rc, what)
    return n.value


# the current stream's handle: the raw query costs 0.1 us of the 4 us that a launch takes, the stream object 2
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


# ------------------------------------------------------------------------------------------------ cross attention
def _xattn_args(q, k, v, kv_len, key_mask, scale):
    _first("q", q, _HALF)
    t, dev = q.dtype, q.get_device()
    if q.dim() != 4 or not isinstance(k, torch.Tensor) or k.dim() != 4:
        _refuse("expected q [B,Lq,Hq,D] and k, v [Bk,Lk,Hk,D]")
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hk, _ = shape = k.shape
    _tensor("k", k, t, dev, (Bk, Lk, Hk, D))
    _tensor("v", v, t, dev, shape)
    q, qs = _rows16(q)
    k, ks = _rows16(k, 1)
    v, vs = _rows16(v, 1)
    a = _lib.isb_xattn_args(dev, _TYPES[t], B, Bk, Lq, Lk, Hq, Hk, D, D ** -0.5 if scale is None and D else float(scale or 0),
                            q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks, vs)
    keep = [q, k, v]
    if kv_len is not None:
        _tensor("kv_len", kv_len, torch.int32, dev, (Bk,))
        kv_len = kv_len.contiguous()
        keep.append(kv_len)
        a.kv_len = kv_len.data_ptr()
    if key_mask is not None:
        _tensor("key_mask", key_mask, torch.bool, dev, (Bk, Lk))
        if Lk > 1 and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        keep.append(key_mask)
        a.key_mask, a.mask_stride = key_mask.data_ptr(), key_mask.stride(0)
    return a, keep


def _xattn_empty(a) -> bool:
    """there is nothing to attend, or to attend to: no launch. What can be wrong with the arguments all the same is refused."""
    if a.B and a.Bk and a.Lq and a.Lk:
        return False
    if a.B and not a.Bk:
        _refuse(f"{a.B} samples share no set of states")
    one = _lib.isb_xattn_args(a.device, a.dtype, a.B or a.Bk or 1, a.Bk or 1, a.Lq or 1, a.Lk or 1, a.Hq, a.Hk, a.D, a.scale)
    _workspace(_lib.lib().isb_xattn_workspace, "isb_xattn_workspace", one, 0)
    return True


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_len: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """softmax(scale q k^T) v over an encoder's states of another length; (out [B,Lq,Hq,D], lse f32 [B,Hq,Lq]).

    q [B,Lq,Hq,D], k and v [Bk,Lk,Hk,D], fp16 or bf16, any strides (copied where rows do not lie on 16 bytes, or k's and v's
    states too far apart); D a multiple of 8 up to 128. Hq is a multiple of Hk (grouped heads). B is a multiple of Bk: sample b reads the states
    of b // (B // Bk), so Bk = 1 is ONE support set for every window, read once for all of them. State j takes part iff j < kv_len[bk] (int32 [Bk]) and key_mask[bk, j]
    (bool [Bk,Lk]); a row without states (Lk may be 0) gets zeros and lse = -inf. scale defaults to 1 / sqrt(D)."""
    if _forward_ad._current_level >= 0:
        _tangents(q, k, v)
    a, keep = _xattn_args(q, k, v, kv_len, key_mask, scale)
    if not (q.numel() and k.numel()) and _xattn_empty(a):
        return q.new_zeros(q.shape), q.new_full((a.B, a.Hq, a.Lq), -math.inf, dtype=torch.float32)
    B, Lq, Hq, _ = shape = q.shape
    out = q.new_empty(shape)
    lse = q.new_empty((B, Hq, Lq), dtype=torch.float32)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    lib = _lib.lib()
    n = _workspace(lib.isb_xattn_workspace, "isb_xattn_workspace", a, 0)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    rc = lib.isb_xattn_forward(C.byref(a), ws.data_ptr() if n else None, n, _stream(a.device))
    if rc:
        _lib.check(rc, "isb_xattn_forward")
    return out, lse


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                             kv_len: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                             scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) of :func:`cross_attention`, given its arguments and results. Gradients of shared heads and shared states are summed;
    masked states get zeros."""
    if _forward_ad._current_level >= 0:
        _tangents(dout, q, k, v, out, lse)
    a, keep = _xattn_args(q, k, v, kv_len, key_mask, scale)
    dev, t = q.get_device(), q.dtype
    _tensor("dout", dout, t, dev, q.shape)
    _tensor("out", out, t, dev, q.shape)
    _tensor("lse", lse, torch.float32, dev, (q.shape[0], q.shape[2], q.shape[1]))
    if not (q.numel() and k.numel()) and _xattn_empty(a):
        return q.new_zeros(q.shape), k.new_zeros(k.shape), v.new_zeros(v.shape)
    dout, a.dout_stride = _rows16(dout)
    out, lse = _flat16(out), lse.contiguous()
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), k.new_empty(k.shape)
    a.out, a.lse, a.dout = out.data_ptr(), lse.data_ptr(), dout.data_ptr()
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    lib = _lib.lib()
    n = _workspace(lib.isb_xattn_workspace, "isb_xattn_workspace", a, 1)
    ws = q.new_empty(n, dtype=torch.uint8)
    rc = lib.isb_xattn_backward(C.byref(a), ws.data_ptr(), n, _stream(a.device))
    if rc:
        _lib.check(rc, "isb_xattn_backward")
    return dq, dk, dv


# ------------------------------------------------------------------------------------------------ gated feed-forward block
def _ffn_args(x, w_gate, w_up, w_down, activation):
    _first("x", x, _HALF)
    t, dev = x.dtype, x.get_device()
    if not isinstance(w_gate, torch.Tensor) or w_gate.dim() != 2 or x.dim() < 1:
        _refuse("expected x [..,D] and w_gate [F,D]")
    F, D = shape = w_gate.shape
    if x.shape[-1] != D:
        _refuse(f"x: expected [..,{D}], got {tuple(x.shape)}")
    _tensor("w_gate", w_gate, t, dev, shape)
    _tensor("w_up", w_up, t, dev, shape)
    _tensor("w_down", w_down, t, dev, (D, F))
    if activation not in ACTIVATIONS:
        _refuse(f"activation {activation!r} not in {sorted(ACTIVATIONS)}")
    x2, xs = _rows2(x)
    wg, wu, wd = _flat16(w_gate), _flat16(w_up), _flat16(w_down)
    if x2.shape[0] == 0:                                     # no launch; what can be wrong with the arguments all the same is refused
        one = _lib.isb_ffn_args(dev, _TYPES[t], 1, D, F, ACTIVATIONS[activation])
        _workspace(_lib.lib().isb_ffn_workspace, "isb_ffn_workspace", one, 0)
    a = _lib.isb_ffn_args(dev, _TYPES[t], x2.shape[0], D, F, ACTIVATIONS[activation], xs, 0, x2.data_ptr(), wg.data_ptr(), wu.data_ptr(),
                          wd.data_ptr())
    return a, [x2, wg, wu, wd]


def _rows2(x):
    """x [.., D] as (rows [M, D], their stride), the rows on 16 bytes; a copy only where they are not a constant stride apart, overlap, lie too far
    apart or not on 16 bytes"""
    x2, (st,) = _rows16(x if x.dim() == 2 else x.reshape(x.numel() // max(x.shape[-1], 1), x.shape[-1]), 0)
    if x2.shape[0] > 1 and st < x2.shape[1]:
        x2, st = x2.contiguous(), x2.shape[1]
    return x2, st


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
              b_up: Optional[torch.Tensor] = None, b_down: Optional[torch.Tensor] = None, activation: str = "silu", save: bool = False):
    """y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down, fp16 or bf16.

    x [..,D] (rows a constant stride apart), w_gate and w_up [F,D], w_down [D,F] (torch Linear layout), biases or None; D and F multiples
    of 8; activation "silu", "gelu" (exact), "relu" or "sigmoid". Returns y, or (y, saved) with save=True: what
    :func:`gated_ffn_backward` needs (both pre-activations in f32, the hidden rows in x's type; fp16: in a form of the library's own, which the backward
    call may write anew)."""
    if _forward_ad._current_level >= 0:
        _tangents(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    a, keep = _ffn_args(x, w_gate, w_up, w_down, activation)
    dev, t, M, D, F = x.get_device(), x.dtype, a.M, a.D, a.F
    for n, b, size in (("b_gate", b_gate, F), ("b_up", b_up, F), ("b_down", b_down, D)):
        if b is not None:
            _tensor(n, b, t, dev, (size,))
            b = _flat16(b)
            keep.append(b)
            setattr(a, n, b.data_ptr())
    y = x.new_empty(x.shape)
    a.y = y.data_ptr()
    saved = None
    if save:
        saved = (x.new_empty((M, F), dtype=torch.float32), x.new_empty((M, F), dtype=torch.float32), x.new_empty((M, F)))
        a.pre_gate, a.pre_up, a.hidden = (s.data_ptr() for s in saved)
    if M == 0:
        return (y, saved) if save else y
    lib = _lib.lib()
    n = _workspace(lib.isb_ffn_workspace, "isb_ffn_workspace", a, 0)
    ws = x.new_empty(n, dtype=torch.uint8) if n else None
    rc = lib.isb_ffn_forward(C.byref(a), ws.data_ptr() if n else None, n, _stream(a.device))
    if rc:
        _lib.check(rc, "isb_ffn_forward")
    return (y, saved) if save else y


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, saved,
                       bias: bool = False, activation: str = "silu") -> Dict[str, torch.Tensor]:
    """Gradients of :func:`gated_ffn`: {"dx", "dw_gate", "dw_up", "dw_down"} and, with bias=True, {"db_gate", "db_up", "db_down"}. The two
    first weights' gradients are the halves of one [2F,D] tensor."""
    if _forward_ad._current_level >= 0:
        _tangents(dy, x, w_gate, w_up, w_down)
    a, keep = _ffn_args(x, w_gate, w_up, w_down, activation)
    dev, t, M, D, F = x.get_device(), x.dtype, a.M, a.D, a.F
    _tensor("dy", dy, t, dev, x.shape)
    if not (isinstance(saved, tuple) and len(saved) == 3):
        _refuse("saved: expected what gated_ffn(save=True) returned")
    for n, s, st in zip(("pre_gate", "pre_up", "hidden"), saved, (torch.float32, torch.float32, t)):
        _tensor(n, s, st, dev, (M, F))
        if not s.is_contiguous():
            _refuse(f"{n} is not contiguous")
        setattr(a, n, s.data_ptr())
    dy2, a.dy_stride = _rows2(dy)
    a.dy = dy2.data_ptr()
    dx, dw, dwd = x.new_empty(x.shape), x.new_empty((2 * F, D)), x.new_empty((D, F))
    a.dx, a.dw_gate_up, a.dw_down = dx.data_ptr(), dw.data_ptr(), dwd.data_ptr()
    r = {"dx": dx, "dw_gate": dw[:F], "dw_up": dw[F:], "dw_down": dwd}
    if bias:
        db = x.new_empty(2 * F + D)
        r["db_gate"], r["db_up"], r["db_down"] = db[:F], db[F:2 * F], db[2 * F:]
        at = db.data_ptr()
        a.db_gate, a.db_up, a.db_down = at, at + 2 * F, at + 4 * F
    if M == 0:
        for v in r.values():
            v.zero_()
        return r
    lib = _lib.lib()
    n = _workspace(lib.isb_ffn_workspace, "isb_ffn_workspace", a, 1)
    ws = x.new_empty(n, dtype=torch.uint8)
    rc = lib.isb_ffn_backward(C.byref(a), ws.data_ptr(), n, _stream(a.device))
    if rc:
        _lib.check(rc, "isb_ffn_backward")
    return r


# ------------------------------------------------------------------------------------------------ norms around a block
def _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps):
    _first("x", x, _TYPES)
    t, dev = x.dtype, x.get_device()
    if x.dim() != 3:
        _refuse(f"x: expected [B,L,D], got {tuple(x.shape)}")
    if post not in NORMS or pre not in NORMS:
        _refuse(f"norms {post!r}, {pre!r}: None, 'layer' or 'rms'")
    B, L, D = shape = x.shape
    x = x.contiguous()
    keep, p, vec = [x], [x.data_ptr()], (D,)
    for n, v, sh, dt in (("y", y, shape, t), ("gate", gate, (B, D), t), ("scale", scale, vec, torch.float32),
                         ("post_weight", post_weight, vec, torch.float32), ("post_bias", post_bias, vec, torch.float32),
                         ("pre_weight", pre_weight, vec, torch.float32), ("pre_bias", pre_bias, vec, torch.float32)):
        if v is None:
            p.append(None)
        else:
            _tensor(n, v, dt, dev, sh)
            v = v.contiguous()
            keep.append(v)
            p.append(v.data_ptr())
    a = _lib.isb_norm_args(dev, _TYPES[t], B, L, D, NORMS[post], NORMS[pre], eps, *p)
    if B == 0 or L == 0:                                     # no launch; what can be wrong with the arguments all the same is refused
        p = [None if v is None else 16 for v in (x, y, gate, scale, post_weight, post_bias, pre_weight, pre_bias)]      # (never read)
        one = _lib.isb_norm_args(dev, _TYPES[t], 1, 1, D, NORMS[post], NORMS[pre], eps, *p)
        _workspace(_lib.lib().isb_norm_workspace, "isb_norm_workspace", one)
    return a, keep


def block_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
               post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, save: bool = False):
    """r = x + scale * gate * N_post(y) and z = N_pre(r) in one pass; (r, z), or (r, z, stats) with save=True.

    x, y [B,L,D] f32, fp16 or bf16, D up to 8192 (any); gate [B,D] of x's type (B up to 65535), scale, weights and biases f32 [D], or None; post / pre:
    None, "layer" or "rms" (no bias). y None: the norm before the first block, r is x itself. pre None: z is None. z is the norm of r
    before r is rounded; stats f32 [B,L,4] are for :func:`block_norm_backward`."""
    if _forward_ad._current_level >= 0:
        _tangents(x, y, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    a, keep = _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps)
    r, z, stats = x, None, None
    if y is not None:
        r = x.new_empty(x.shape)
        a.r = r.data_ptr()
    if pre is not None:
        z = x.new_empty(x.shape)
        a.z = z.data_ptr()
    if save:
        stats = x.new_empty((*x.shape[:2], 4), dtype=torch.float32)
        a.stats = stats.data_ptr()
    if x.numel() or not x.shape[2]:
        rc = _lib.lib().isb_norm_forward(C.byref(a), _stream(a.device))
        if rc:
            _lib.check(rc, "isb_norm_forward")
    return (r, z, stats) if save else (r, z)


def block_norm_backward(dr: Optional[torch.Tensor], dz: Optional[torch.Tensor], x: torch.Tensor, y: Optional[torch.Tensor], stats: torch.Tensor, *,
                        gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, post: Optional[str] = None,
                        post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, pre: Optional[str] = None,
                        pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
                        eps: float = 1e-5) -> Dict[str, torch.Tensor]:
    """Gradients of :func:`block_norm` (same arguments, its stats): {"dx", "dy"?, "dgate"?, "dscale"?, "dpost_weight"?, "dpost_bias"?,
    "dpre_weight"?, "dpre_bias"?}, one for each tensor given. dr (or None: zeros) and dz are the gradients of r and z."""
    if _forward_ad._current_level >= 0:
        _tangents(dr, dz, x, y, stats, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    a, keep = _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps)
    dev, t = x.get_device(), x.dtype
    if (dz is not None) != (pre is not None):
        _refuse("dz goes with a pre norm")
    if dr is None and dz is None:
        _refuse("neither dr nor dz")
    for n, v in (("dr", dr), ("dz", dz)):
        if v is not None:
            _tensor(n, v, t, dev, x.shape)
            v = v.contiguous()
            keep.append(v)
            setattr(a, n, v.data_ptr())
    _tensor("stats", stats, torch.float32, dev, (*x.shape[:2], 4))
    if not stats.is_contiguous():
        _refuse("stats are not contiguous")
    a.stats = stats.data_ptr()
    g = {"dx": x.new_empty(x.shape)}
    if y is not None:
        g["dy"] = x.new_empty(x.shape)
    if gate is not None:
        g["dgate"] = x.new_empty(gate.shape)
    for n, v in (("dscale", scale), ("dpost_weight", post_weight), ("dpost_bias", post_bias), ("dpre_weight", pre_weight),
                 ("dpre_bias", pre_bias)):
        if v is not None:
            g[n] = v.new_empty(v.shape)
    if x.numel() == 0 and x.shape[2]:
        for v in g.values():
            v.zero_()
        return g
    for n, v in g.items():
        setattr(a, n, v.data_ptr())
    lib = _lib.lib()
    n = _workspace(lib.isb_norm_workspace, "isb_norm_workspace", a)
    ws = x.new_empty(n, dtype=torch.uint8)
    rc = lib.isb_norm_backward(C.byref(a), ws.data_ptr(), n, _stream(a.device))
    if rc:
        _lib.check(rc, "isb_norm_backward")
    return g
