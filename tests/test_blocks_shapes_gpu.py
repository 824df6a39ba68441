"""GPU tests of the layer operators (isbfsar_amd/blocks.py) at shapes and layouts beside those of test_blocks_gpu.py, with its inputs and the
64-bit forms and bounds of blocks_ref."""
import pytest
import torch

import blocks_ref as ref
from test_blocks_gpu import BF16, F32, FP16, blocks, held, norm_inputs, xattn_inputs

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ cross attention
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("case", [
    # B, Bk, Lq, Lk, Hq, Hk, D, masks: tiles of 32 rows in one round of the CUs and in two, around the lengths where the form changes
    (16, 16, 512, 100, 1, 1, 128, "len holes"), (17, 17, 512, 100, 1, 1, 128, "len holes"), (20, 5, 128, 192, 16, 4, 64, "holes"),
    (20, 5, 128, 193, 16, 4, 64, "holes"), (32, 32, 511, 65, 1, 1, 72, "len empty"), (33, 33, 512, 250, 1, 1, 128, "len"),
])
def test_xattn_short_states_many_tiles(case, t):
    q, k, v, dout, m = xattn_inputs(case, t)
    out, lse = blocks().cross_attention(q, k, v, **m)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse, **m)
    want = ref.xattn(q, k, v, dout=dout, **m)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *d)):
        held(got, *want[name], name)


# ------------------------------------------------------------------------------------------------ norms around a block
@pytest.mark.parametrize("t", [BF16, FP16, F32])
@pytest.mark.parametrize("kinds", [("layer", "rms"), ("rms", "layer"), (None, "layer"), ("layer", None)])
@pytest.mark.parametrize("shape", [(7000, 1, 64), (12400, 3, 72), (6145, 2, 65), (2100, 1, 1280), (600, 1, 8192), (513, 2, 4100), (600, 3, 2056), (30000, 1, 8)])
def test_norm_more_samples_than_workgroups(shape, kinds, t):
    x, y, dr, dz, a = norm_inputs(*shape, t, kinds, True)
    if kinds[1] is None:
        dz = None
    r, z, stats = blocks().block_norm(x, y, save=True, **a)
    d = blocks().block_norm_backward(dr, dz, x, y, stats, **a)
    want = ref.norm(x, y, dr=dr, dz=dz, **a)
    for n, got in {"r": r, **({} if z is None else {"z": z}), **d}.items():
        held(got, *want[n], n)
    again = blocks().block_norm_backward(dr, dz, x, y, stats, **a)
    assert all(torch.equal(again[n], d[n]) for n in d)
