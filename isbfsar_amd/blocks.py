"""The operators of a cross-attention layer over feature sequences (include/isbfsar.h: isb_xattn_*, isb_ffn_*, isb_norm_*).

They stand beside the tuple attention, the MLPs and the LayerNorm that live inside :class:`isbfsar_amd.engine.ArEngine` and work on
what it hands out: the embeddings of query windows ([B, L, 256], ``infer(want_embed=True)``) and the frames of a support set
(``support_features()``)::

    n = block_norm(x, pre="layer", pre_weight=w, pre_bias=b)                      # norm before the block
    out, lse = cross_attention(q, k, v, kv_len=lengths)                           # windows against the support set's frames
    x, n = block_norm(x, proj(out), scale=s, pre="layer", ...)                    # residual sum + the next block's norm, one pass
    y = gated_ffn(n, w_gate, w_up, w_down)

torch owns the device memory and the stream (the tensors' current stream); every call is asynchronous on it, allocates its results and
its workspace with torch and may be captured into a graph. Backward passes are calls of their own and take what the forward call
returned; nothing is recorded on an autograd tape and no result requires a gradient.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
NORMS = {None: 0, "layer": 1, "rms": 2}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check(ok: bool, msg: str, *args) -> None:
    if not ok:
        raise ValueError(msg.format(*args))


def _on_gpu(name: str, t, dtype, device) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    _check(t.device == device, "{} lives on {}, the first tensor on {}", name, t.device, device)
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")


def _first(name: str, t, types) -> None:
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if t.dtype not in types:
        raise TypeError(f"{name} is {t.dtype}, expected one of {sorted(str(x) for x in types)}")


_HALF = (torch.float16, torch.bfloat16)


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its last dimension is not contiguous or its rows do not lie on 16 bytes"""
    if t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1]):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _flat16(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t contiguous on 16 bytes"""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(fn, what: str, args, *more) -> Tuple[Optional[torch.Tensor], int]:
    n = C.c_size_t()
    _lib.check(fn(C.byref(args), *more, C.byref(n)), what)
    return n.value


def _stream(device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# ------------------------------------------------------------------------------------------------ cross attention
def _xattn_args(q, k, v, kv_len, key_mask, scale):
    _first("q", q, _HALF)
    dev, t = q.device, q.dtype
    _on_gpu("k", k, t, dev)
    _on_gpu("v", v, t, dev)
    _check(q.dim() == 4 and k.dim() == 4 and k.shape == v.shape, "expected q [B,Lq,Hq,D] and k, v [Bk,Lk,Hk,D], got {} {} {}",
           tuple(q.shape), tuple(k.shape), tuple(v.shape))
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hk, Dk = k.shape
    _check(D == Dk, "head sizes {} and {} differ", D, Dk)
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    a = _lib.isb_xattn_args(dev.index, _TYPES[t], B, Bk, Lq, Lk, Hq, Hk, D, 1.0 / math.sqrt(max(D, 1)) if scale is None else float(scale),
                            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride()[:3], k.stride()[:3], v.stride()[:3])
    keep = [q, k, v]
    if kv_len is not None:
        _on_gpu("kv_len", kv_len, torch.int32, dev)
        _check(tuple(kv_len.shape) == (Bk,), "kv_len: expected [{}], got {}", Bk, tuple(kv_len.shape))
        kv_len = kv_len.contiguous()
        keep.append(kv_len)
        a.kv_len = kv_len.data_ptr()
    if key_mask is not None:
        _on_gpu("key_mask", key_mask, torch.bool, dev)
        _check(tuple(key_mask.shape) == (Bk, Lk), "key_mask: expected [{},{}], got {}", Bk, Lk, tuple(key_mask.shape))
        if key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        keep.append(key_mask)
        a.key_mask, a.mask_stride = key_mask.data_ptr(), key_mask.stride(0)
    return a, keep


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_len: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """softmax(scale q k^T) v over an encoder's states of another length; (out [B,Lq,Hq,D], lse f32 [B,Hq,Lq]).

    q [B,Lq,Hq,D], k and v [Bk,Lk,Hk,D], fp16 or bf16, any strides (copied where rows do not lie on 16 bytes); D a multiple of 8 up to
    128. Hq is a multiple of Hk (grouped heads). B is a multiple of Bk: sample b reads the states of b // (B // Bk), so Bk = 1 is ONE
    support set for every window, read once for all of them. State j takes part iff j < kv_len[bk] (int32 [Bk]) and key_mask[bk, j]
    (bool [Bk,Lk]); a row without states gets zeros and lse = -inf. scale defaults to 1 / sqrt(D)."""
    a, keep = _xattn_args(q, k, v, kv_len, key_mask, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    lib = _lib.lib()
    n = _workspace(lib.isb_xattn_workspace, "isb_xattn_workspace", a, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _lib.check(lib.isb_xattn_forward(C.byref(a), _ptr(ws), n, _stream(q.device)), "isb_xattn_forward")
    return out, lse


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                             kv_len: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None,
                             scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) of :func:`cross_attention`, given its arguments and results. Gradients of shared heads and shared states are summed;
    masked states get zeros."""
    a, keep = _xattn_args(q, k, v, kv_len, key_mask, scale)
    dev, t = q.device, q.dtype
    _on_gpu("dout", dout, t, dev)
    _on_gpu("out", out, t, dev)
    _on_gpu("lse", lse, torch.float32, dev)
    _check(dout.shape == q.shape and out.shape == q.shape, "dout, out: expected {}, got {} {}", tuple(q.shape), tuple(dout.shape), tuple(out.shape))
    _check(tuple(lse.shape) == (q.shape[0], q.shape[2], q.shape[1]), "lse: expected [B,Hq,Lq], got {}", tuple(lse.shape))
    dout, out, lse = _rows16(dout), _flat16(out), lse.contiguous()
    dq = torch.empty(q.shape, dtype=t, device=dev)
    dk = torch.empty(k.shape, dtype=t, device=dev)
    dv = torch.empty(k.shape, dtype=t, device=dev)
    a.out, a.lse, a.dout, a.dout_stride = out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dout.stride()[:3]
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    lib = _lib.lib()
    n = _workspace(lib.isb_xattn_workspace, "isb_xattn_workspace", a, 1)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.isb_xattn_backward(C.byref(a), ws.data_ptr(), n, _stream(dev)), "isb_xattn_backward")
    return dq, dk, dv


# ------------------------------------------------------------------------------------------------ gated feed-forward block
def _ffn_args(x, w_gate, w_up, w_down, activation):
    _first("x", x, _HALF)
    dev, t = x.device, x.dtype
    for n, w in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        _on_gpu(n, w, t, dev)
    _check(x.dim() >= 1 and w_gate.dim() == 2, "expected x [..,D] and w_gate [F,D], got {} {}", tuple(x.shape), tuple(w_gate.shape))
    F, D = w_gate.shape
    _check(x.shape[-1] == D and tuple(w_up.shape) == (F, D) and tuple(w_down.shape) == (D, F),
           "expected x [..,{}], w_up [{},{}], w_down [{},{}], got {} {} {}", D, F, D, D, F, tuple(x.shape), tuple(w_up.shape), tuple(w_down.shape))
    _check(activation in ACTIVATIONS, "activation {!r} not in {}", activation, sorted(ACTIVATIONS))
    x2 = _rows2(x)
    w = [_flat16(w_gate), _flat16(w_up), _flat16(w_down)]
    a = _lib.isb_ffn_args(dev.index, _TYPES[t], x2.shape[0], D, F, ACTIVATIONS[activation], x2.stride(0), 0, x2.data_ptr(),
                          w[0].data_ptr(), w[1].data_ptr(), w[2].data_ptr())
    return a, [x2, *w]


def _rows2(x):
    """x [.., D] as rows [M, D] whose starts lie on 16 bytes, a copy only where they do not; rows may be a constant stride apart, not
    overlap"""
    x2 = _rows16(x.reshape(-1, x.shape[-1]))
    return x2 if x2.shape[0] == 1 or x2.stride(0) >= x2.shape[1] else x2.contiguous()


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
              b_up: Optional[torch.Tensor] = None, b_down: Optional[torch.Tensor] = None, activation: str = "silu", save: bool = False):
    """y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down, fp16 or bf16.

    x [..,D] (rows a constant stride apart), w_gate and w_up [F,D], w_down [D,F] (torch Linear layout), biases or None; D and F multiples
    of 8; activation "silu", "gelu" (exact), "relu" or "sigmoid". Returns y, or (y, saved) with save=True: what
    :func:`gated_ffn_backward` needs (both pre-activations in f32, the hidden rows in x's type)."""
    a, keep = _ffn_args(x, w_gate, w_up, w_down, activation)
    dev, t, M, D, F = x.device, x.dtype, a.M, a.D, a.F
    for n, b, s in (("b_gate", b_gate, F), ("b_up", b_up, F), ("b_down", b_down, D)):
        if b is not None:
            _on_gpu(n, b, t, dev)
            _check(tuple(b.shape) == (s,), "{}: expected [{}], got {}", n, s, tuple(b.shape))
            b = _flat16(b)
            keep.append(b)
            setattr(a, n, b.data_ptr())
    y = torch.empty(x.shape, dtype=t, device=dev)
    if M == 0:
        _check(False, "x has no rows")
    a.y = y.data_ptr()
    saved = None
    if save:
        saved = (torch.empty((M, F), dtype=torch.float32, device=dev), torch.empty((M, F), dtype=torch.float32, device=dev),
                 torch.empty((M, F), dtype=t, device=dev))
        a.pre_gate, a.pre_up, a.hidden = (s.data_ptr() for s in saved)
    lib = _lib.lib()
    n = _workspace(lib.isb_ffn_workspace, "isb_ffn_workspace", a, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _lib.check(lib.isb_ffn_forward(C.byref(a), _ptr(ws), n, _stream(dev)), "isb_ffn_forward")
    return (y, saved) if save else y


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, saved,
                       bias: bool = False, activation: str = "silu") -> Dict[str, torch.Tensor]:
    """Gradients of :func:`gated_ffn`: {"dx", "dw_gate", "dw_up", "dw_down"} and, with bias=True, {"db_gate", "db_up", "db_down"}. The two
    first weights' gradients are the halves of one [2F,D] tensor."""
    a, keep = _ffn_args(x, w_gate, w_up, w_down, activation)
    dev, t, M, D, F = x.device, x.dtype, a.M, a.D, a.F
    _on_gpu("dy", dy, t, dev)
    _check(dy.shape == x.shape, "dy: expected {}, got {}", tuple(x.shape), tuple(dy.shape))
    _check(isinstance(saved, tuple) and len(saved) == 3, "saved: expected what gated_ffn(save=True) returned")
    for n, s, st in zip(("pre_gate", "pre_up", "hidden"), saved, (torch.float32, torch.float32, t)):
        _on_gpu(n, s, st, dev)
        _check(tuple(s.shape) == (M, F) and s.is_contiguous(), "{}: expected [{},{}], got {}", n, M, F, tuple(s.shape))
        setattr(a, n, s.data_ptr())
    dy2 = _rows2(dy)
    a.dy, a.dy_stride = dy2.data_ptr(), dy2.stride(0)
    dx = torch.empty(x.shape, dtype=t, device=dev)
    dw = torch.empty((2 * F, D), dtype=t, device=dev)
    dwd = torch.empty((D, F), dtype=t, device=dev)
    a.dx, a.dw_gate_up, a.dw_down = dx.data_ptr(), dw.data_ptr(), dwd.data_ptr()
    r = {"dx": dx, "dw_gate": dw[:F], "dw_up": dw[F:], "dw_down": dwd}
    if bias:
        db = torch.empty(2 * F + D, dtype=t, device=dev)
        r["db_gate"], r["db_up"], r["db_down"] = db[:F], db[F:2 * F], db[2 * F:]
        a.db_gate, a.db_up, a.db_down = (r[n].data_ptr() for n in ("db_gate", "db_up", "db_down"))
    lib = _lib.lib()
    n = _workspace(lib.isb_ffn_workspace, "isb_ffn_workspace", a, 1)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.isb_ffn_backward(C.byref(a), ws.data_ptr(), n, _stream(dev)), "isb_ffn_backward")
    return r


# ------------------------------------------------------------------------------------------------ norms around a block
def _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps):
    _first("x", x, tuple(_TYPES))
    dev, t = x.device, x.dtype
    _check(x.dim() == 3, "expected x [B,L,D], got {}", tuple(x.shape))
    B, L, D = x.shape
    _check(post in NORMS and pre in NORMS, "norms {!r}, {!r}: None, 'layer' or 'rms'", post, pre)
    x = x.contiguous()
    keep = {"x": x}
    for n, v, shape, dt in (("y", y, (B, L, D), t), ("gate", gate, (B, D), t), ("scale", scale, (D,), torch.float32),
                            ("post_weight", post_weight, (D,), torch.float32), ("post_bias", post_bias, (D,), torch.float32),
                            ("pre_weight", pre_weight, (D,), torch.float32), ("pre_bias", pre_bias, (D,), torch.float32)):
        if v is not None:
            _on_gpu(n, v, dt, dev)
            _check(tuple(v.shape) == shape, "{}: expected {}, got {}", n, shape, tuple(v.shape))
            keep[n] = v.contiguous()
    p = [_ptr(keep.get(n)) for n in ("x", "y", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")]
    return _lib.isb_norm_args(dev.index, _TYPES[t], B, L, D, NORMS[post], NORMS[pre], float(eps), *p), keep


def block_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
               post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, save: bool = False):
    """r = x + scale * gate * N_post(y) and z = N_pre(r) in one pass; (r, z), or (r, z, stats) with save=True.

    x, y [B,L,D] f32, fp16 or bf16, D up to 8192 (any); gate [B,D] of x's type, scale, weights and biases f32 [D], or None; post / pre:
    None, "layer" or "rms" (no bias). y None: the norm before the first block, r is x itself. pre None: z is None. z is the norm of r
    before r is rounded; stats f32 [B,L,4] are for :func:`block_norm_backward`."""
    a, keep = _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps)
    r = x if y is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    z = None if pre is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((*x.shape[:2], 4), dtype=torch.float32, device=x.device) if save else None
    a.r, a.z, a.stats = None if y is None else r.data_ptr(), _ptr(z), _ptr(stats)
    _lib.check(_lib.lib().isb_norm_forward(C.byref(a), _stream(x.device)), "isb_norm_forward")
    return (r, z, stats) if save else (r, z)


def block_norm_backward(dr: Optional[torch.Tensor], dz: Optional[torch.Tensor], x: torch.Tensor, y: Optional[torch.Tensor], stats: torch.Tensor, *,
                        gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, post: Optional[str] = None,
                        post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, pre: Optional[str] = None,
                        pre_weight: Optional[torch.Tensor] = None, pre_bias: Optional[torch.Tensor] = None,
                        eps: float = 1e-5) -> Dict[str, torch.Tensor]:
    """Gradients of :func:`block_norm` (same arguments, its stats): {"dx", "dy"?, "dgate"?, "dscale"?, "dpost_weight"?, "dpost_bias"?,
    "dpre_weight"?, "dpre_bias"?}, one for each tensor given. dr (or None: zeros) and dz are the gradients of r and z."""
    a, keep = _norm_args(x, y, gate, scale, post, post_weight, post_bias, pre, pre_weight, pre_bias, eps)
    dev, t = x.device, x.dtype
    _check((dz is not None) == (pre is not None), "dz goes with a pre norm")
    _check(dr is not None or dz is not None, "neither dr nor dz")
    for n, v in (("dr", dr), ("dz", dz)):
        if v is not None:
            _on_gpu(n, v, t, dev)
            _check(v.shape == x.shape, "{}: expected {}, got {}", n, tuple(x.shape), tuple(v.shape))
            keep[n] = v.contiguous()
            setattr(a, n, keep[n].data_ptr())
    _on_gpu("stats", stats, torch.float32, dev)
    _check(tuple(stats.shape) == (*x.shape[:2], 4) and stats.is_contiguous(), "stats: expected [B,L,4], got {}", tuple(stats.shape))
    a.stats = stats.data_ptr()
    g = {"dx": torch.empty(x.shape, dtype=t, device=dev)}
    if y is not None:
        g["dy"] = torch.empty(x.shape, dtype=t, device=dev)
    if gate is not None:
        g["dgate"] = torch.empty(gate.shape, dtype=t, device=dev)
    for n, v in (("dscale", scale), ("dpost_weight", post_weight), ("dpost_bias", post_bias), ("dpre_weight", pre_weight),
                 ("dpre_bias", pre_bias)):
        if v is not None:
            g[n] = torch.empty(v.shape, dtype=torch.float32, device=dev)
    for n, v in g.items():
        setattr(a, n, v.data_ptr())
    lib = _lib.lib()
    n = _workspace(lib.isb_norm_workspace, "isb_norm_workspace", a)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _lib.check(lib.isb_norm_backward(C.byref(a), ws.data_ptr(), n, _stream(dev)), "isb_norm_backward")
    return g
