"""GPU tests of the layer operators' calls (isbfsar_amd/blocks.py): layouts that need a copy, empty tensors, tensors on autograd's tape."""
import math

import pytest
import torch

import blocks_ref as ref
from test_blocks_gpu import BF16, F32, FP16, blocks, ffn_inputs, gen, held, norm_inputs, normal, xattn_inputs

pytestmark = pytest.mark.gpu
FAR = (1 << 22) + 8                                           # elements between rows, more than a launch takes


def far(t):
    """t [n, ...] with its rows FAR elements apart"""
    w = t[0].numel()
    base = torch.zeros(t.shape[0], FAR, dtype=t.dtype, device="cuda")
    base[:, :w] = t.reshape(t.shape[0], w)
    return base[:, :w].unflatten(1, t.shape[1:])


@pytest.mark.parametrize("Lk", [40, 1])
def test_xattn_states_far_apart(Lk):
    """any strides: states further apart than a launch takes are copied"""
    q, k, v, dout, _ = xattn_inputs((2, 1, 33, Lk, 4, 2, 64, ""), BF16)
    fk, fv = far(k[0])[None], far(v[0])[None]
    if Lk == 1:
        fk, fv = (x.as_strided(x.shape, (8, FAR, 64, 1)) for x in (fk, fv))
    assert fk.stride(1) == FAR and torch.equal(fk, k) and torch.equal(fv, v)
    want = blocks().cross_attention(q, k, v)
    out, lse = blocks().cross_attention(q, fk, fv)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    for a, b in zip(blocks().cross_attention_backward(dout, q, fk, fv, out, lse), blocks().cross_attention_backward(dout, q, k, v, *want)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("M", [2, 40])
def test_ffn_rows_far_apart(M):
    a, b, dy = ffn_inputs(M, 64, 136, BF16, True)
    w = [a["wg"], a["wu"], a["wd"]]
    want, saved = blocks().gated_ffn(a["x"], *w, *b, save=True)
    y, saved = blocks().gated_ffn(far(a["x"]), *w, *b, save=True)
    assert torch.equal(y, want)
    grads = blocks().gated_ffn_backward(dy, a["x"], *w, saved)
    for n, g in blocks().gated_ffn_backward(far(dy), far(a["x"]), *w, saved).items():
        assert torch.equal(g, grads[n]), n


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("B,Bk,Lq,Lk", [(2, 1, 3, 0), (0, 1, 3, 5), (2, 2, 0, 5), (0, 0, 3, 5), (0, 2, 0, 0)])
def test_xattn_of_nothing(t, B, Bk, Lq, Lk):
    """no states: zeros, lse -inf, no gradient; no rows: empty results, the states' gradients zero"""
    q, dout = (torch.ones(B, Lq, 4, 64, dtype=t, device="cuda") for _ in range(2))
    k, v = (torch.ones(Bk, Lk, 2, 64, dtype=t, device="cuda") for _ in range(2))
    m = {"kv_len": torch.full((Bk,), Lk, dtype=torch.int32, device="cuda"), "key_mask": torch.ones(Bk, Lk, dtype=torch.bool, device="cuda")}
    for mask in ({}, m):
        out, lse = blocks().cross_attention(q, k, v, **mask)
        assert out.shape == q.shape and out.dtype == t and not out.any()
        assert lse.shape == (B, 4, Lq) and lse.dtype == F32 and bool((lse == -math.inf).all())
        for g, like in zip(blocks().cross_attention_backward(dout, q, k, v, out, lse, **mask), (q, k, v)):
            assert g.shape == like.shape and g.dtype == t and not g.any()


def test_xattn_of_nothing_is_checked_all_the_same():
    q, k = torch.ones(0, 3, 4, 64, dtype=BF16, device="cuda"), torch.ones(1, 5, 2, 64, dtype=BF16, device="cuda")
    for bad in ((q, k, k[:, :, :, :32]), (q, k, k.half()), (q[..., :60], k[..., :60], k[..., :60]), (q[:, :, :3], k, k), (q[:, :, :0], k, k),
                (torch.ones(2, 3, 4, 64, dtype=BF16, device="cuda"), k[:0], k[:0])):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            blocks().cross_attention(*bad)
    with pytest.raises((ValueError, RuntimeError)):
        blocks().cross_attention(q, k, k, scale=-1.0)


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64)])
def test_ffn_of_nothing(shape):
    a, b, _ = ffn_inputs(1, 64, 136, FP16, True)
    w = [a["wg"], a["wu"], a["wd"]]
    x = torch.ones(*shape, dtype=FP16, device="cuda")
    assert blocks().gated_ffn(x, *w, *b).shape == shape
    y, saved = blocks().gated_ffn(x, *w, *b, save=True)
    assert y.shape == shape and y.dtype == FP16
    d = blocks().gated_ffn_backward(y, x, *w, saved, bias=True)
    for n, like in zip(("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), (x, *w, *b)):
        assert d[n].shape == like.shape and d[n].dtype == FP16 and not d[n].any(), n
    for bad in ((x, w[0], w[1][:, :32], w[2]), (x[..., :60], *(v[:, :60] for v in w[:2]), w[2][:60])):
        with pytest.raises((ValueError, RuntimeError)):
            blocks().gated_ffn(*bad)


@pytest.mark.parametrize("B,L", [(0, 3), (2, 0)])
def test_norm_of_nothing(B, L):
    x, y, dr, dz, a = norm_inputs(1, 1, 72, BF16, ("layer", "rms"), True)
    x, y, dr, dz = (v[:, :0].expand(B, 0, 72) if L == 0 else v[:0].expand(0, L, 72) for v in (x, y, dr, dz))
    a["gate"] = a["gate"].expand(B, 72) if B else a["gate"][:0]
    r, z, stats = blocks().block_norm(x, y, save=True, **a)
    assert r.shape == z.shape == (B, L, 72) and stats.shape == (B, L, 4)
    d = blocks().block_norm_backward(dr, dz, x, y, stats, **a)
    for n, like in {"dx": x, "dy": y, "dgate": a["gate"], "dscale": a["scale"], "dpost_weight": a["post_weight"], "dpost_bias": a["post_bias"],
                    "dpre_weight": a["pre_weight"]}.items():
        assert d[n].shape == like.shape and d[n].dtype == like.dtype and not d[n].any(), n
    r, z = blocks().block_norm(x, pre="layer")
    assert r is x and z.shape == x.shape
    with pytest.raises((ValueError, RuntimeError)):
        blocks().block_norm(x, y, pre="rms", pre_bias=a["scale"])
    with pytest.raises((ValueError, RuntimeError)):
        blocks().block_norm(torch.ones(2, 3, 0, device="cuda"), pre="layer")


# ------------------------------------------------------------------------------------------------ autograd
def calls():
    q, k, v, dout, _ = xattn_inputs((2, 1, 3, 40, 2, 2, 64, ""), BF16)
    out, lse = blocks().cross_attention(q, k, v)
    a, b, dy = ffn_inputs(6, 64, 136, BF16, True)
    f = [a["x"], a["wg"], a["wu"], a["wd"]]
    y, saved = blocks().gated_ffn(*f, *b, save=True)
    nx, ny, dr, dz, na = norm_inputs(2, 3, 64, BF16, ("layer", "rms"), True)
    _, _, st = blocks().block_norm(nx, ny, save=True, **na)
    names = [n for n, t in na.items() if torch.is_tensor(t)]

    def norm(x, y, *p):
        return blocks().block_norm(x, y, **{**na, **dict(zip(names, p))})

    def norm_backward(dr, dz, x, y, *p):
        return list(blocks().block_norm_backward(dr, dz, x, y, st, **{**na, **dict(zip(names, p))}).values())
    return {"xattn": (blocks().cross_attention, [q, k, v]), "xattn backward": (blocks().cross_attention_backward, [dout, q, k, v, out]),
            "ffn": (lambda *t: [blocks().gated_ffn(*t)], [*f, *b]), "ffn backward": (lambda *t: list(blocks().gated_ffn_backward(*t, saved).values()), [dy, *f]),
            "norm": (norm, [nx, ny, *(na[n] for n in names)]), "norm backward": (norm_backward, [dr, dz, nx, ny, *(na[n] for n in names)])}, lse


@pytest.mark.parametrize("name", ["xattn", "xattn backward", "ffn", "ffn backward", "norm", "norm backward"])
def test_tensors_on_the_tape_are_refused(name):
    """no result would carry their gradient: an error, not silence. Under no_grad they are tensors like others."""
    (f, args), lse = calls()[0][name], calls()[1]
    more = [lse] if name == "xattn backward" else []
    want = f(*args, *more)
    for i in range(len(args)):
        on = list(args)
        on[i] = args[i].clone().requires_grad_(True)
        with pytest.raises(ValueError, match="no_grad"):
            f(*on, *more)
        with torch.no_grad():
            got = f(*on, *more)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_tangents_and_transforms_are_refused():
    import torch.autograd.forward_ad as fw
    q, k, v, _, _ = xattn_inputs((2, 1, 3, 40, 2, 2, 64, ""), BF16)
    with fw.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            blocks().cross_attention(fw.make_dual(q, torch.ones_like(q)), k, v)
        blocks().cross_attention(q, k, v)
        for f, args in (c for n, c in calls()[0].items() if n != "xattn backward"):
            for i in range(len(args)):
                with pytest.raises(ValueError, match="tangent"):
                    f(*args[:i], fw.make_dual(args[i], torch.ones_like(args[i])), *args[i + 1:])
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        torch.func.grad(lambda x: blocks().cross_attention(x, k, v)[0].float().sum())(q)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        torch.func.vmap(lambda x: blocks().cross_attention(x[None], k, v)[0])(q)
