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
