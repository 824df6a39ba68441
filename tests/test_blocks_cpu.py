"""What the layer operators refuse, without a GPU: every check of include/isbfsar.h's layer operators is made on the host before any HIP
call, so a refused call launches nothing and touches nothing."""
import ctypes as C
import math

import pytest

from isbfsar_amd import _lib

OK16 = 4096          # a plausible 16-byte aligned address; never dereferenced by a refused call


@pytest.fixture(scope="module")
def lib():
    from isbfsar_amd.build import build
    build(verbose=False)
    return _lib.lib()


def xattn(**k):
    s = k.pop("strides", (1024, 128, 64))
    f = {"device": 0, "dtype": 1, "B": 4, "Bk": 2, "Lq": 3, "Lk": 5, "Hq": 4, "Hk": 2, "D": 64, "scale": 0.125, "q": OK16, "k": OK16, "v": OK16,
         "out": OK16, "lse": OK16, "dout": OK16, "dq": OK16, "dk": OK16, "dv": OK16, **k}
    a = _lib.isb_xattn_args(**f)
    for n in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        if n not in k:
            setattr(a, n, s)
    return a


I3 = C.c_int64 * 3
BAD_SHAPE = [dict(dtype=0), dict(dtype=7), dict(B=0), dict(Bk=0), dict(Lq=0), dict(Lk=0), dict(Hq=0), dict(Hk=0), dict(D=0), dict(D=60), dict(D=136),
             dict(B=3), dict(Hq=3), dict(Lk=(1 << 30) + 1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
             dict(B=1 << 20, Bk=1, Lq=1 << 20)]
BAD_ARGS = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lse=None), dict(q=OK16 + 2), dict(k=OK16 + 8), dict(out=OK16 + 4),
            dict(strides=(1024, 127, 64)), dict(strides=(-8, 128, 64)), dict(k_stride=I3(0, (1 << 22) + 8, 64)),
            dict(key_mask=OK16, mask_stride=-1)]


@pytest.mark.parametrize("bad", BAD_SHAPE)
def test_xattn_shapes(lib, bad):
    n = C.c_size_t()
    a = xattn(**bad)
    assert lib.isb_xattn_workspace(C.byref(a), 0, C.byref(n)) == -1 and lib.isb_last_error()
    assert lib.isb_xattn_forward(C.byref(a), OK16, 1 << 40, None) == -1
    assert lib.isb_xattn_backward(C.byref(a), OK16, 1 << 40, None) == -1


@pytest.mark.parametrize("bad", BAD_ARGS)
def test_xattn_pointers_and_strides(lib, bad):
    a = xattn(**bad)
    assert lib.isb_xattn_forward(C.byref(a), OK16, 1 << 40, None) == -1 and lib.isb_last_error()
    assert lib.isb_xattn_backward(C.byref(a), OK16, 1 << 40, None) == -1


@pytest.mark.parametrize("bad", [dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(dq=OK16 + 8), dict(dout_stride=I3(8, 4, 8))])
def test_xattn_backward_arguments(lib, bad):
    assert lib.isb_xattn_backward(C.byref(xattn(**bad)), OK16, 1 << 40, None) == -1


def test_xattn_more_workgroups_than_a_launch_holds(lib):
    n = C.c_size_t()
    for big in (dict(B=1 << 21, Bk=1 << 21, Lq=1, Hq=4, Hk=4), dict(B=1, Bk=1, Lq=1 << 27, Hq=8, Hk=8), dict(B=1, Bk=1, Hq=8, Hk=8, Lk=1 << 27)):
        assert lib.isb_xattn_workspace(C.byref(xattn(**big)), 0, C.byref(n)) == -1, big
        assert lib.isb_xattn_backward(C.byref(xattn(**big)), OK16, 1 << 50, None) == -1
        for f in ("Bk", "Lq", "Lk"):
            if big.get(f, 0) >= 1 << 21:
                less = {**big, f: big[f] // 2, **({"B": big["B"] // 2} if f == "Bk" else {})}
                assert lib.isb_xattn_workspace(C.byref(xattn(**less)), 1, C.byref(n)) == 0, less


def test_null_and_workspace(lib):
    n = C.c_size_t()
    assert lib.isb_xattn_forward(None, None, 0, None) == -1 and lib.isb_ffn_forward(None, None, 0, None) == -1
    assert lib.isb_norm_forward(None, None) == -1 and lib.isb_xattn_workspace(C.byref(xattn()), 0, None) == -1
    a = xattn(Lk=4096)
    assert lib.isb_xattn_workspace(C.byref(a), 0, C.byref(n)) == 0 and n.value > 0
    assert lib.isb_xattn_forward(C.byref(a), OK16, n.value - 1, None) == -1
    assert lib.isb_xattn_forward(C.byref(a), None, n.value, None) == -1
    assert lib.isb_xattn_forward(C.byref(a), OK16 + 8, n.value, None) == -1
    assert lib.isb_xattn_workspace(C.byref(a), 1, C.byref(n)) == 0 and n.value > 0
    assert lib.isb_xattn_backward(C.byref(a), OK16, n.value - 1, None) == -1


def ffn(**k):
    f = {"device": 0, "dtype": 2, "M": 3, "D": 64, "F": 128, "act": 0, "x_stride": 64, "dy_stride": 64}
    f.update({n: OK16 for n in ("x", "w_gate", "w_up", "w_down", "y", "dy", "pre_gate", "pre_up", "hidden", "dx", "dw_gate_up", "dw_down")})
    return _lib.isb_ffn_args(**{**f, **k})


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(M=0), dict(M=(1 << 22) + 1), dict(D=0), dict(D=60), dict(F=4), dict(F=132), dict(D=1 << 21), dict(act=-1),
                                 dict(act=4), dict(x=None), dict(x=OK16 + 2), dict(x_stride=56), dict(x_stride=68), dict(w_gate=None), dict(w_up=OK16 + 8),
                                 dict(w_down=None)])
def test_ffn(lib, bad):
    a = ffn(**bad)
    assert lib.isb_ffn_forward(C.byref(a), OK16, 1 << 40, None) == -1 and lib.isb_last_error()
    assert lib.isb_ffn_backward(C.byref(a), OK16, 1 << 40, None) == -1


@pytest.mark.parametrize("bad", [dict(y=None), dict(pre_up=None), dict(pre_gate=None), dict(hidden=None), dict(b_gate=OK16 + 2), dict(hidden=OK16 + 2)])
def test_ffn_forward(lib, bad):
    assert lib.isb_ffn_forward(C.byref(ffn(**bad)), OK16, 1 << 40, None) == -1


@pytest.mark.parametrize("bad", [dict(dy=None), dict(dy_stride=8), dict(pre_gate=None), dict(pre_up=None), dict(hidden=None), dict(dx=None),
                                 dict(dw_gate_up=None), dict(dw_down=None), dict(db_gate=OK16), dict(db_up=OK16), dict(db_down=OK16 + 2)])
def test_ffn_backward(lib, bad):
    assert lib.isb_ffn_backward(C.byref(ffn(**bad)), OK16, 1 << 40, None) == -1


def test_ffn_workspace(lib):
    n = C.c_size_t()
    a = ffn()
    assert lib.isb_ffn_workspace(C.byref(a), 1, C.byref(n)) == 0 and n.value >= 3 * 2 * 128 * 2
    assert lib.isb_ffn_backward(C.byref(a), OK16, n.value - 1, None) == -1
    a = ffn(hidden=None, pre_gate=None, pre_up=None)
    assert lib.isb_ffn_workspace(C.byref(a), 0, C.byref(n)) == 0 and n.value >= 3 * 128 * 2
    assert lib.isb_ffn_forward(C.byref(a), OK16, n.value - 1, None) == -1


def norm(**k):
    f = {"device": 0, "dtype": 2, "B": 2, "L": 3, "D": 64, "post": 1, "pre": 1, "eps": 1e-5}
    f.update({n: OK16 for n in ("x", "y", "r", "z", "stats", "dr", "dz", "dx", "dy")})
    return _lib.isb_norm_args(**{**f, **k})


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(B=0), dict(L=0), dict(D=0), dict(D=8200), dict(post=3), dict(pre=-1), dict(eps=-1.0), dict(eps=math.nan),
                                 dict(x=None), dict(x=OK16 + 1), dict(y=None), dict(y=None, post=0, pre=0), dict(y=None, post=0, gate=OK16),
                                 dict(y=None, post=0, scale=OK16), dict(post=0, post_weight=OK16), dict(post=2, post_bias=OK16), dict(pre=0, pre_weight=OK16),
                                 dict(pre=2, pre_bias=OK16), dict(stats=OK16 + 4), dict(B=70000, gate=OK16)])
def test_norm(lib, bad):
    a = norm(**bad)
    assert lib.isb_norm_forward(C.byref(a), None) == -1 and lib.isb_last_error()
    assert lib.isb_norm_backward(C.byref(a), OK16, 1 << 40, None) == -1


@pytest.mark.parametrize("bad", [dict(stats=None), dict(dx=None), dict(dy=None), dict(dz=None), dict(pre=0, dr=None), dict(dgate=OK16)])
def test_norm_backward(lib, bad):
    assert lib.isb_norm_backward(C.byref(norm(**bad)), OK16, 1 << 40, None) == -1
    n = C.c_size_t()
    assert lib.isb_norm_workspace(C.byref(norm()), C.byref(n)) == 0
    assert lib.isb_norm_backward(C.byref(norm()), OK16, n.value - 1, None) == -1


def test_norm_forward_outputs(lib):
    assert lib.isb_norm_forward(C.byref(norm(r=None)), None) == -1
    assert lib.isb_norm_forward(C.byref(norm(z=None)), None) == -1


def test_python_refuses_host_tensors_and_wrong_types():
    import torch
    from isbfsar_amd import blocks as b
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    with pytest.raises(TypeError, match="CUDA tensor"):
        b.cross_attention(q, q, q)
    with pytest.raises(TypeError, match="CUDA tensor"):
        b.gated_ffn(q, q, q, q)
    with pytest.raises(TypeError, match="CUDA tensor"):
        b.block_norm(q, pre="layer")


def test_fast_division_is_exact():
    """the multiplier of csrc/blk_common.h's FastDiv, for every divisor class and the numbers around its multiples"""
    for d in [*range(1, 300), 511, 512, 513, 1000, 65535, 65536, 65537, (1 << 20) - 1, 1 << 24, (1 << 30) - 1, 1 << 30]:
        ln = (d - 1).bit_length()
        m = ((1 << 32) * ((1 << ln) - d)) // d + 1
        assert m < 1 << 32
        ns = {0, 1, d - 1, d, d + 1, 2 * d - 1, (1 << 31) - 1}
        for q in (1, 3, 7, 1000, 12345):
            ns |= {q * d - 1, q * d, q * d + 1}
        top = ((1 << 31) - 1) // d * d
        ns |= {top - 1, top, top + 1}
        for n in ns:
            if 0 <= n < 1 << 31:
                hi = (n * m) >> 32
                assert hi + n < 1 << 32 and (hi + n) >> ln == n // d, (n, d)
