"""GPU tests of the stand-alone layer operators (isbfsar_amd/blocks.py) against plain 64-bit implementations (tests/blocks_ref.py, where
the bounds are derived): types, head layouts, lengths, masks, strides, gradients, graphs, streams, and the layer as a whole."""
import math

import pytest
import torch

import blocks_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = [BF16, FP16]


def blocks():
    from isbfsar_amd import blocks as b
    return b


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, type=F32, std=1.0):
    return torch.empty(shape, device="cuda", dtype=F32).normal_(0, std, generator=g).to(type)


def held(got, want, bound, name):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    g = got.double()
    same = (g == want) | (g.isnan() & want.isnan())            # (infinities: -inf of an empty row's lse)
    off = torch.where(same, 0.0, (g - want).abs() - bound)
    assert not off.isnan().any() and bool((off <= 0).all()), (name, float(off.nan_to_num(math.inf).max()), float((g - want).abs().nan_to_num(0).max()))


# ------------------------------------------------------------------------------------------------ cross attention
XATTN = [
    # B, Bk, Lq, Lk, Hq, Hk, D, masks
    (1, 1, 1, 1, 1, 1, 8, ""),                  # one token, one state, the smallest head
    (1, 1, 1, 1800, 4, 4, 64, ""),              # a streaming tick
    (3, 3, 1, 515, 8, 2, 128, "len"),           # single tokens, grouped heads, ragged lengths, splits
    (16, 16, 1, 2050, 8, 1, 128, "len holes"),
    (6, 2, 5, 77, 4, 2, 64, "holes"),           # two sets of states, three samples each
    (2, 2, 31, 63, 2, 2, 32, ""),
    (2, 2, 33, 65, 3, 3, 40, "len"),            # just past a tile, a head size that ends inside one
    (2, 1, 130, 129, 4, 2, 72, "holes"),        # shared states, D between the two tile widths
    (9, 1, 30, 90, 2, 2, 128, "len holes"),     # windows against one support set
    (1, 1, 257, 1000, 2, 1, 128, ""),
    (4, 4, 100, 300, 2, 2, 64, "empty"),        # a sample without states
    (3, 3, 64, 64, 2, 2, 128, "len holes empty"),
    (1, 1, 33, 4100, 1, 1, 64, "holes"),        # few rows, a long axis: splits
    (2, 1, 50, 140, 6, 2, 64, "len"),           # three heads to a state head
    (1, 1, 2, 300, 40, 1, 128, "holes"),        # forty heads to a state head: more rows than a token's, two positions
    (4, 1, 64, 200, 4, 1, 32, ""),              # samples that end with a tile of rows
    (5, 1, 67, 129, 2, 1, 128, "len"),          # samples that end inside one
    (40, 2, 3, 1500, 8, 2, 72, "len holes"),    # short samples, many of them on one set of states
]


def xattn_inputs(case, t, seed=0, std=1.0):
    B, Bk, Lq, Lk, Hq, Hk, D, masks = case
    g = gen(seed + 7)
    q, k, v, dout = normal(g, B, Lq, Hq, D, type=t), normal(g, Bk, Lk, Hk, D, type=t), normal(g, Bk, Lk, Hk, D, type=t), normal(g, B, Lq, Hq, D, type=t, std=std)
    kv_len = key_mask = None
    if "len" in masks:
        kv_len = torch.randint(1, Lk + 1, (Bk,), generator=g, device="cuda").to(torch.int32)
    if "holes" in masks:
        key_mask = torch.rand(Bk, Lk, generator=g, device="cuda") < 0.7
    if "empty" in masks:
        if kv_len is None:
            kv_len = torch.full((Bk,), Lk, dtype=torch.int32, device="cuda")
        kv_len[1] = 0
        if key_mask is not None:
            key_mask[2] = False
    ok = ref.valid_states(Bk, Lk, kv_len, key_mask, "cuda")
    # what masked states hold must not matter: NaN, infinities, the lowest value
    for x in (k, v):
        junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(t).min], device="cuda", dtype=t)
        x[~ok] = junk[torch.arange(int((~ok).sum()), device="cuda") % 4][:, None, None]
    return q, k, v, dout, {"kv_len": kv_len, "key_mask": key_mask}


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("case", XATTN)
def test_xattn_forward_and_gradients(case, t):
    q, k, v, dout, m = xattn_inputs(case, t)
    out, lse = blocks().cross_attention(q, k, v, **m)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse, **m)
    want = ref.xattn(q, k, v, dout=dout, **m)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *d)):
        held(got, *want[name], name)
    ok = ref.valid_states(k.shape[0], k.shape[1], m["kv_len"], m["key_mask"], "cuda")
    assert not d[1][~ok].any() and not d[2][~ok].any()              # masked states: zeros
    none = ~ok.any(1).repeat_interleave(q.shape[0] // k.shape[0])
    assert not out[none].any() and bool((lse[none] == -math.inf).all()) and not d[0][none].any()


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("case", [
    (1, 1, 257, 2100, 2, 1, 128, "holes"),         # a long axis in splits of 128-row tiles
    (3, 3, 70, 2055, 2, 2, 72, "len holes empty"),
    (600, 600, 33, 65, 1, 1, 40, "len holes empty"),       # more tiles than one round of the chip
    (140, 70, 67, 70, 4, 2, 64, "len"),
    (260, 2, 30, 333, 4, 2, 128, "holes"),
    (2, 2, 100, 64, 2, 2, 128, "holes"),           # two blocks of states
    (32, 32, 32, 2048, 2, 2, 64, "len"),           # tiles of 32 rows at their most states
    (1, 1, 33, 2048, 2, 1, 128, ""),
    (16, 1, 31, 1800, 1, 1, 128, "holes"),
    (8, 8, 100, 300, 4, 4, 64, "len holes empty"), # tiles of 32 rows backward too
    (16, 16, 70, 130, 2, 2, 72, "len holes"),
    (6, 3, 60, 1000, 16, 2, 128, "holes"),
    (100, 100, 3, 66, 1, 1, 8, "len"),
])
def test_xattn_forms(case, t):
    """the forms that test_xattn_forward_and_gradients' sizes do not reach"""
    q, k, v, dout, m = xattn_inputs(case, t)
    out, lse = blocks().cross_attention(q, k, v, **m)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse, **m)
    want = ref.xattn(q, k, v, dout=dout, **m)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *d)):
        held(got, *want[name], name)


@pytest.mark.parametrize("t", HALF)
def test_xattn_small_gradients_keep_their_digits(t):
    """dout of 2^-12: dS lies far below fp16's normal range and must not lose digits there"""
    case = (2, 1, 40, 700, 2, 2, 64, "")
    q, k, v, dout, m = xattn_inputs(case, t, std=2.0 ** -12)
    out, lse = blocks().cross_attention(q, k, v)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse)
    want = ref.xattn(q, k, v, dout=dout)
    for name, got in zip(("dq", "dk", "dv"), d):
        held(got, *want[name], name)


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("Lq", [1, 40])
def test_xattn_scores_that_grow_along_the_states(t, Lq):
    """the running maximum moves in every tile, by more and by less than the step that rescales"""
    g = gen(3)
    q, k, v = normal(g, 1, Lq, 2, 64, type=t), normal(g, 1, 900, 2, 64, type=t), normal(g, 1, 900, 2, 64, type=t)
    k = (k * torch.linspace(0.1, 6, 900, device="cuda")[None, :, None, None]).to(t)
    dout = normal(g, 1, Lq, 2, 64, type=t)
    out, lse = blocks().cross_attention(q, k, v)
    want = ref.xattn(q, k, v, dout=dout)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *d)):
        held(got, *want[name], name)


def test_xattn_scale_and_lengths_outside_the_range():
    q, k, v, _, _ = xattn_inputs((2, 2, 3, 50, 2, 2, 64, ""), BF16)
    n = torch.tensor([-4, 1000], dtype=torch.int32, device="cuda")
    out, lse = blocks().cross_attention(q, k, v, kv_len=n, scale=0.5)
    want = ref.xattn(q, k, v, kv_len=n.clamp(0, 50), scale=0.5)
    held(out, *want["out"], "out")
    held(lse, *want["lse"], "lse")


@pytest.mark.parametrize("Lq", [1, 70])
def test_xattn_strides(Lq):
    """heads first, a packed k / v projection, an expanded query, rows that do not lie on 16 bytes"""
    g = gen(5)
    q = normal(g, 2, 4, Lq, 64, type=BF16).transpose(1, 2)                         # [B, Lq, Hq, D] with the heads outside
    kv = normal(g, 2, 99, 2, 2, 64, type=BF16)
    k, v = kv[:, :, 0], kv[:, :, 1]
    dout = normal(g, 2, 4, Lq, 64, type=BF16).transpose(1, 2)
    want = ref.xattn(q, k, v, dout=dout)
    out, lse = blocks().cross_attention(q, k, v)
    held(out, *want["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), blocks().cross_attention_backward(dout, q, k, v, out, lse)):
        held(got, *want[name], name)
    q1 = normal(g, 1, Lq, 4, 64, type=BF16).expand(2, -1, -1, -1)                  # stride 0
    o = blocks().cross_attention(q1, k, v)[0]
    held(o, *ref.xattn(q1.contiguous(), k, v)["out"], "expanded")
    odd = normal(g, 2, 99, 2, 65, type=BF16)[..., 1:]                              # neither aligned nor in strides of 8
    o = blocks().cross_attention(q, odd, odd)[0]
    held(o, *ref.xattn(q, odd.contiguous(), odd.contiguous())["out"], "odd rows")


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("Lq", [2, 70])
def test_xattn_a_nan_stays_where_it_belongs(Lq, t):
    """a NaN in a query row makes that row NaN, one in a valid state every row of its sample and state head; nothing else"""
    q, k, v, dout, _ = xattn_inputs((3, 3, Lq, 90, 4, 2, 64, ""), t)
    q[0, 1, 3, 7] = math.nan
    k[1, 44, 1, 5] = math.nan
    v[2, 80, 0, 9] = math.nan
    out, lse = blocks().cross_attention(q, k, v)
    want = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    want[0, 1, 3] = True
    want[1, :, 2:] = True
    want[2, :, :2, 9] = True
    assert torch.equal(out.isnan(), want)
    assert bool(lse[0, 3, 1].isnan()) and bool(lse[1, 2:].isnan().all()) and int(lse.isnan().sum()) == 1 + 2 * Lq
    dq, dk, dv = blocks().cross_attention_backward(dout, q, k, v, out, lse)
    assert bool(dq[0, 1, 3].isnan().all()) and not dq[0, :, :2].isnan().any() and not dq[1, :, :2].isnan().any()
    assert bool(dk[0, :, 1].isnan().all()) and not dk[0, :, 0].isnan().any() and bool(dv[1, :, 1].isnan().all()) and not dv[1, :, 0].isnan().any()


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("Lq", [64, 1200])
def test_xattn_an_infinite_gradient_stays_in_its_row(t, Lq):
    """dout holds an infinity (a loss scaled too far): dq of the other rows, dk and dv of the other head are what they are without it"""
    q, k, v, dout, _ = xattn_inputs((1, 1, Lq, 300, 2, 2, 64, ""), t, std=8.0)
    out, lse = blocks().cross_attention(q, k, v)
    without, bad = dout.clone(), dout.clone()
    without[0, 3, 0], bad[0, 3, 0, 7] = 0, math.inf
    want = ref.xattn(q, k, v, dout=without)
    dq, dk, dv = blocks().cross_attention_backward(bad, q, k, v, out, lse)
    assert not dq[0, 3, 0].isfinite().any()
    dq[0, 3, 0] = 0
    held(dq, *want["dq"], "dq")
    for name, got in (("dk", dk), ("dv", dv)):
        held(got[:, :, 1], want[name][0][:, :, 1], want[name][1][:, :, 1], name)


def test_xattn_results_past_the_type_s_range():
    """fp16 results saturate: dv sums 300 rows of 6e4 into one state"""
    q = torch.zeros(1, 300, 1, 64, dtype=FP16, device="cuda")
    k, v = torch.zeros(1, 1, 1, 64, dtype=FP16, device="cuda"), torch.ones(1, 1, 1, 64, dtype=FP16, device="cuda")
    dout = torch.full_like(q, 60000.0)
    out, lse = blocks().cross_attention(q, k, v)
    dq, dk, dv = blocks().cross_attention_backward(dout, q, k, v, out, lse)
    assert bool((out == 1).all()) and bool((dv == 65504).all()) and not dq.any() and not dk.any()


def test_xattn_offsets_past_32_bits():
    """k and v of more than 2^31 elements (4.3 GB each): the last states are the ones attended to"""
    Lk, Hk, D = 131200, 128, 128
    k = torch.zeros(1, Lk, Hk, D, dtype=FP16, device="cuda")
    v = torch.zeros(1, Lk, Hk, D, dtype=FP16, device="cuda")
    g = gen(11)
    k[:, -300:], v[:, -300:] = normal(g, 1, 300, Hk, D, type=FP16), normal(g, 1, 300, Hk, D, type=FP16)
    mask = torch.zeros(1, Lk, dtype=torch.bool, device="cuda")
    mask[:, -300:] = True
    for Lq in (1, 40):
        q = normal(g, 1, Lq, Hk, D, type=FP16)
        out, lse = blocks().cross_attention(q, k, v, key_mask=mask)
        want = ref.xattn(q, k[:, -300:], v[:, -300:])
        held(out, *want["out"], "out")
        held(lse, *want["lse"], "lse")


def test_xattn_gradients_against_differences():
    """<gradient, direction> against central differences of the 64-bit loss <out, dout>; the kernel may be off by its bound along the
    direction, the differences by 1e-6 of their size"""
    case = (4, 2, 9, 70, 4, 2, 32, "len holes")
    q, k, v, dout, m = xattn_inputs(case, FP16)
    k, v = k.nan_to_num(0, 0, 0).clamp(-4, 4), v.nan_to_num(0, 0, 0).clamp(-4, 4)
    out, lse = blocks().cross_attention(q, k, v, **m)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse, **m)
    want = ref.xattn(q, k, v, dout=dout, **m)
    loss = lambda a, b, c: float((ref.xattn(a, b, c, **m)["out"][0] * dout.double()).sum())     # noqa: E731
    x = [q.double(), k.double(), v.double()]
    for i, name in enumerate(("dq", "dk", "dv")):
        g = gen(20 + i)
        e = torch.empty_like(x[i]).normal_(0, 1, generator=g)
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + 1e-5 * e, x[i] - 1e-5 * e
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        along = float((d[i].double() * e).sum())
        assert abs(along - diff) <= float((want[name][1] * e.abs()).sum()) + 1e-6 * (1 + abs(diff)), (name, along, diff)


# ------------------------------------------------------------------------------------------------ gated feed-forward block
FFN = [
    # M, D, F
    (1, 8, 8), (1, 256, 1024), (2, 72, 136), (4, 1280, 2056), (5, 64, 128), (30, 256, 1024), (33, 136, 520), (64, 640, 1288), (65, 128, 256),
    (129, 384, 776), (300, 72, 1032), (1030, 264, 520),
]


def ffn_inputs(M, D, F, t, bias, seed=0):
    g = gen(seed + 13)
    a = {"x": normal(g, M, D, type=t), "wg": normal(g, F, D, type=t, std=D ** -0.5), "wu": normal(g, F, D, type=t, std=D ** -0.5),
         "wd": normal(g, D, F, type=t, std=F ** -0.5)}
    b = [normal(g, n, type=t, std=0.3) for n in (F, F, D)] if bias else [None] * 3
    return a, b, normal(g, M, D, type=t)


@pytest.mark.parametrize("t", HALF)
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True), ("relu", False), ("sigmoid", True)])
@pytest.mark.parametrize("shape", FFN)
def test_ffn_forward_and_gradients(shape, act, bias, t):
    a, b, dy = ffn_inputs(*shape, t, bias)
    w = [a["wg"], a["wu"], a["wd"]]
    y, saved = blocks().gated_ffn(a["x"], *w, *b, activation=act, save=True)
    d = blocks().gated_ffn_backward(dy, a["x"], *w, saved, bias=bias, activation=act)
    want = ref.ffn(a["x"], *w, *b, activation=act, dy=dy)
    held(y, *want["y"], "y")
    assert set(d) == {n for n in want if n != "y" and (bias or not n.startswith("db"))}
    for n, got in d.items():
        held(got, *want[n], n)
    assert torch.equal(y, blocks().gated_ffn(a["x"], *w, *b, activation=act))      # the same bits without saving


@pytest.mark.parametrize("shape", [(4000, 1280, 5120), (2100, 2048, 4104), (7001, 1280, 2056)])
def test_ffn_large_tiles(shape):
    """enough rows and features for the largest tiles, with ragged edges; the last: more tiles than places, a tail of them in parts"""
    a, b, dy = ffn_inputs(*shape, BF16, True)
    w = [a["wg"], a["wu"], a["wd"]]
    y, saved = blocks().gated_ffn(a["x"], *w, *b, save=True)
    d = blocks().gated_ffn_backward(dy, a["x"], *w, saved, bias=True)
    want = ref.ffn(a["x"], *w, *b, dy=dy)
    held(y, *want["y"], "y")
    for n, got in d.items():
        held(got, *want[n], n)


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_ffn_tall_tiles(act):
    """rows and features that leave the largest tiles a nearly empty round, both with ragged edges"""
    a, b, dy = ffn_inputs(2101, 264, 4104, FP16, True)
    w = [a["wg"], a["wu"], a["wd"]]
    y, saved = blocks().gated_ffn(a["x"], *w, *b, activation=act, save=True)
    d = blocks().gated_ffn_backward(dy, a["x"], *w, saved, bias=True, activation=act)
    want = ref.ffn(a["x"], *w, *b, activation=act, dy=dy)
    held(y, *want["y"], "y")
    for n, got in d.items():
        held(got, *want[n], n)


def test_ffn_strides_and_leading_dimensions():
    a, b, dy = ffn_inputs(60, 128, 264, BF16, True)
    w = [a["wg"], a["wu"], a["wd"]]
    wide = torch.zeros(60, 200, dtype=BF16, device="cuda")
    wide[:, 8:136] = a["x"]
    y = blocks().gated_ffn(wide[:, 8:136], *w, *b)
    assert torch.equal(y, blocks().gated_ffn(a["x"], *w, *b))
    y3 = blocks().gated_ffn(a["x"].view(2, 30, 128), *w, *b)
    assert y3.shape == (2, 30, 128) and torch.equal(y3.view(60, 128), y)
    one = a["x"][:1].expand(60, -1)                                                 # stride 0: rows that overlap are copied
    assert torch.equal(blocks().gated_ffn(one, *w, *b), blocks().gated_ffn(one.contiguous(), *w, *b))
    odd = torch.zeros(60, 129, dtype=BF16, device="cuda")
    odd[:, 1:] = a["x"]
    assert torch.equal(blocks().gated_ffn(odd[:, 1:], *w, *b), y)


def test_ffn_offsets_past_32_bits():
    """pre-activations of more than 2^31 elements: rows of zeros (which leave no trace in any gradient), the last ones filled"""
    M, D, F, n = (1 << 20) + 37, 64, 2056, 77
    a, _, dy = ffn_inputs(n, D, F, BF16, False)
    w = [a["wg"], a["wu"], a["wd"]]
    x, d = torch.zeros(M, D, dtype=BF16, device="cuda"), torch.zeros(M, D, dtype=BF16, device="cuda")
    x[-n:], d[-n:] = a["x"], dy
    y, saved = blocks().gated_ffn(x, *w, save=True)
    g = blocks().gated_ffn_backward(d, x, *w, saved)
    want = ref.ffn(a["x"], *w, dy=dy)
    for name, got in (("y", y), ("dx", g["dx"])):
        held(got[-n:], *want[name], name)
        assert not got[:-n].any(), name
    for name in ("dw_gate", "dw_up", "dw_down"):
        held(g[name], *want[name], name)


def test_ffn_gradients_against_differences():
    a, b, dy = ffn_inputs(7, 24, 40, FP16, True)
    x = [a["x"], a["wg"], a["wu"], a["wd"], *b]
    y, saved = blocks().gated_ffn(*x, activation="gelu", save=True)
    d = blocks().gated_ffn_backward(dy, *x[:4], saved, bias=True, activation="gelu")
    want = ref.ffn(*x, activation="gelu", dy=dy)
    x64 = [v.double() for v in x]
    loss = lambda v: float((ref.ffn(*v, activation="gelu")["y"][0] * dy.double()).sum())     # noqa: E731
    for i, name in enumerate(("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")):
        e = torch.empty_like(x64[i]).normal_(0, 1, generator=gen(40 + i))
        hi, lo = list(x64), list(x64)
        hi[i], lo[i] = x64[i] + 1e-5 * e, x64[i] - 1e-5 * e
        diff = (loss(hi) - loss(lo)) / 2e-5
        along = float((d[name].double() * e).sum())
        assert abs(along - diff) <= float((want[name][1] * e.abs()).sum()) + 1e-6 * (1 + abs(diff)), (name, along, diff)


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_ffn_results_past_the_type_s_range(M):
    """fp16 results past 65504 are stored as 65504; a NaN stays one, in its row alone"""
    t = FP16
    x = torch.full((M, 64), 8.0, dtype=t, device="cuda")
    w = torch.full((64, 64), 4.0, dtype=t, device="cuda")
    y = blocks().gated_ffn(x, w, w, w, activation="relu")            # 2048 x 2048 x ...: far past the range
    assert bool((y == 65504).all())
    x[M // 2, 5] = math.nan
    y = blocks().gated_ffn(x, w, w, w, activation="relu")
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[M // 2] = True
    assert bool(y[bad].isnan().all()) and not y[~bad].isnan().any()


# ------------------------------------------------------------------------------------------------ norms around a block
NORM = [(1, 1, 1), (1, 1, 256), (3, 5, 7), (2, 30, 256), (4, 33, 513), (2, 17, 1280), (1, 9, 4096), (2, 3, 8192), (5, 70, 129), (600, 2, 64)]


def norm_inputs(B, L, D, t, kinds, gate, seed=0):
    post, pre = kinds
    g = gen(seed + 29)
    x, y, dr, dz = normal(g, B, L, D, type=t, std=2.0), normal(g, B, L, D, type=t) + 0.25, normal(g, B, L, D, type=t), normal(g, B, L, D, type=t)
    a = {"gate": normal(g, B, D, type=t) if gate else None, "scale": normal(g, D, std=0.5), "post": post, "pre": pre}
    for n, kind in (("post", post), ("pre", pre)):
        a[n + "_weight"] = 1 + normal(g, D, std=0.2) if kind else None
        a[n + "_bias"] = normal(g, D, std=0.2) if kind == "layer" else None
    return x, y, dr, dz, a


@pytest.mark.parametrize("t", [BF16, FP16, F32])
@pytest.mark.parametrize("kinds", [("layer", "layer"), ("rms", "rms"), (None, "layer"), ("rms", None)])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("shape", NORM)
def test_norm_forward_and_gradients(shape, gate, kinds, t):
    x, y, dr, dz, a = norm_inputs(*shape, t, kinds, gate)
    if kinds[1] is None:
        dz = None
    r, z, stats = blocks().block_norm(x, y, save=True, **a)
    d = blocks().block_norm_backward(dr, dz, x, y, stats, **a)
    want = ref.norm(x, y, dr=dr, dz=dz, **a)
    held(r, *want["r"], "r")
    if z is not None:
        held(z, *want["z"], "z")
    assert set(d) == set(want) - {"r", "z"}
    for n, got in d.items():
        held(got, *want[n], n)
    again = blocks().block_norm(x, y, **a)
    assert torch.equal(again[0], r) and (z is None or torch.equal(again[1], z))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_before_the_first_block(kind, t):
    x, _, _, dz, a = norm_inputs(2, 30, 264, t, (None, kind), False)
    a = {k: v for k, v in a.items() if k.startswith("pre")}
    r, z, stats = blocks().block_norm(x, save=True, **a)
    assert r is x
    want = ref.norm(x, dz=dz, **a)
    held(z, *want["z"], "z")
    d = blocks().block_norm_backward(None, dz, x, None, stats, **a)
    assert set(d) == set(want) - {"z"}
    for n, got in d.items():
        held(got, *want[n], n)


def test_norm_rows_far_from_zero():
    """LayerNorm of rows whose mean is 1000 times their spread (f32): the deviations are summed, not the squares"""
    g = gen(31)
    x = 1000 + normal(g, 2, 9, 640)
    z = blocks().block_norm(x, pre="layer")[1]
    held(z, *ref.norm(x, pre="layer")["z"], "z")


def test_norm_unaligned_tensors():
    x, y, dr, dz, a = norm_inputs(2, 5, 256, BF16, ("layer", "layer"), True)
    base = torch.zeros(x.numel() + 1, dtype=BF16, device="cuda")
    base[1:] = x.reshape(-1)
    odd = base[1:].view(x.shape)
    r, z = blocks().block_norm(odd, y, **a)
    r0, z0 = blocks().block_norm(x, y, **a)
    assert torch.equal(r, r0) and torch.equal(z, z0)


def test_norm_offsets_past_32_bits():
    """more than 2^31 elements: rows of zeros, the last ones filled"""
    L, D, n = (1 << 20) + 11, 2056, 60
    x, y, dr, dz, a = norm_inputs(1, n, D, BF16, ("rms", "rms"), False)
    big = []
    for v in (x, y, dr, dz):
        big.append(torch.zeros(1, L, D, dtype=BF16, device="cuda"))
        big[-1][:, -n:] = v
    r, z, stats = blocks().block_norm(big[0], big[1], save=True, **a)
    d = blocks().block_norm_backward(big[2], big[3], big[0], big[1], stats, **a)
    want = ref.norm(x, y, dr=dr, dz=dz, **a)
    for name, got in (("r", r), ("z", z), ("dx", d["dx"]), ("dy", d["dy"])):
        held(got[:, -n:], *want[name], name)
        assert not got[:, :-n].any(), name
    for name in ("dscale", "dpost_weight", "dpre_weight"):
        held(d[name], *want[name], name)


def test_norm_gradients_against_differences():
    x, y, dr, dz, a = norm_inputs(3, 4, 40, F32, ("layer", "rms"), True)
    r, z, stats = blocks().block_norm(x, y, save=True, **a)
    d = blocks().block_norm_backward(dr, dz, x, y, stats, **a)
    want = ref.norm(x, y, dr=dr, dz=dz, **a)
    names = {"dx": "x", "dy": "y", "dgate": "gate", "dscale": "scale", "dpost_weight": "post_weight", "dpost_bias": "post_bias", "dpre_weight": "pre_weight"}
    args = {"x": x, "y": y, **a}
    args = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in args.items()}

    def loss(v):
        w = ref.norm(**v)
        return float((w["r"][0] * dr.double()).sum() + (w["z"][0] * dz.double()).sum())
    for i, (name, of) in enumerate(names.items()):
        e = torch.empty_like(args[of]).normal_(0, 1, generator=gen(60 + i))
        diff = (loss({**args, of: args[of] + 1e-5 * e}) - loss({**args, of: args[of] - 1e-5 * e})) / 2e-5
        along = float((d[name].double() * e).sum())
        assert abs(along - diff) <= float((want[name][1] * e.abs()).sum()) + 1e-6 * (1 + abs(diff)), (name, along, diff)


# ------------------------------------------------------------------------------------------------ the layer, graphs, streams
class Layer:
    """norm -> cross attention -> residual + norm -> gated block -> residual, with its backward pass: the operators as they are used"""

    def __init__(self, D=256, H=4, F=520, t=BF16, seed=0):
        g = gen(seed + 71)
        s = D ** -0.5
        self.H, self.D = H, D
        self.wq, self.wo, self.wk, self.wv = (normal(g, D, D, type=t, std=s) for _ in range(4))
        self.ffn = [normal(g, F, D, type=t, std=s), normal(g, F, D, type=t, std=s), normal(g, D, F, type=t, std=F ** -0.5)]
        self.n1 = {"pre": "layer", "pre_weight": 1 + normal(g, D, std=0.1), "pre_bias": normal(g, D, std=0.1)}
        self.n2 = {"post": "rms", "post_weight": 1 + normal(g, D, std=0.1), "scale": normal(g, D, std=0.3), "pre": "layer",
                   "pre_weight": 1 + normal(g, D, std=0.1), "pre_bias": normal(g, D, std=0.1)}
        self.n3 = {"scale": normal(g, D, std=0.3)}

    def states(self, ctx):
        return (ctx @ self.wk.T).unflatten(-1, (self.H, -1)), (ctx @ self.wv.T).unflatten(-1, (self.H, -1))

    def forward(self, x, ctx, gate, kv_len, save=False):
        b = blocks()
        k, v = self.states(ctx)
        _, n, st1 = b.block_norm(x, save=True, **self.n1)
        q = (n @ self.wq.T).unflatten(-1, (self.H, -1))
        out, lse = b.cross_attention(q, k, v, kv_len=kv_len)
        a = out.flatten(-2) @ self.wo.T
        r, n2, st2 = b.block_norm(x, a, gate=gate, save=True, **self.n2)
        y, saved = b.gated_ffn(n2, *self.ffn, save=True)
        r3, _, st3 = b.block_norm(r, y, save=True, **self.n3)
        if not save:
            return r3
        return r3, (x, n, st1, q, k, v, out, lse, a, r, n2, st2, y, saved, st3, gate, kv_len)

    def backward(self, d, kept):
        b = blocks()
        x, n, st1, q, k, v, out, lse, a, r, n2, st2, y, saved, st3, gate, kv_len = kept
        g3 = b.block_norm_backward(d, None, r, y, st3, **self.n3)
        gf = b.gated_ffn_backward(g3["dy"], n2, *self.ffn, saved)
        g2 = b.block_norm_backward(g3["dx"], gf["dx"], x, a, st2, gate=gate, **self.n2)
        do = (g2["dy"] @ self.wo).unflatten(-1, (self.H, -1))
        dq, dk, dv = b.cross_attention_backward(do, q, k, v, out, lse, kv_len=kv_len)
        g1 = b.block_norm_backward(g2["dx"], dq.flatten(-2) @ self.wq, x, None, st1, **self.n1)
        return {"x": g1["dx"], "gate": g2["dgate"], "ctx": dk.flatten(-2) @ self.wk + dv.flatten(-2) @ self.wv, "w_down": gf["dw_down"],
                "w_gate": gf["dw_gate"], "post_weight": g2["dpost_weight"], "scale": g3["dscale"]}

    def plain(self, x, ctx, gate, kv_len):
        """the same in whatever type the arguments have, for autograd"""
        c = lambda w: w.to(x.dtype)     # noqa: E731

        def ln(v, a, kind):
            if kind == "layer":
                v = v - v.mean(-1, keepdim=True)
            return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * a
        self.p = {"w_down": c(self.ffn[2]).requires_grad_(True), "w_gate": c(self.ffn[0]).requires_grad_(True),
                  "post_weight": c(self.n2["post_weight"]).requires_grad_(True), "scale": c(self.n3["scale"]).requires_grad_(True)}
        n = ln(x, c(self.n1["pre_weight"]), "layer") + c(self.n1["pre_bias"])
        q = (n @ c(self.wq).T).unflatten(-1, (self.H, -1)).transpose(1, 2)
        k, v = ((ctx @ c(w).T).unflatten(-1, (self.H, -1)).transpose(1, 2) for w in (self.wk, self.wv))
        s = q @ k.transpose(-1, -2) / math.sqrt(self.D // self.H)
        s = s.masked_fill(torch.arange(ctx.shape[1], device=x.device)[None, None, None, :] >= kv_len[:, None, None, None], -math.inf)
        a = (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(-2) @ c(self.wo).T
        r = x + c(self.n2["scale"]) * gate[:, None, :] * ln(a, self.p["post_weight"], "rms")
        n2 = ln(r, c(self.n2["pre_weight"]), "layer") + c(self.n2["pre_bias"])
        g = n2 @ self.p["w_gate"].T
        y = (g * torch.sigmoid(g) * (n2 @ c(self.ffn[1]).T)) @ self.p["w_down"].T
        return r + self.p["scale"] * y


def layer_inputs(t=BF16, B=3, L=30, Lk=90, D=256):
    g = gen(81)
    return (normal(g, B, L, D, type=t), normal(g, B, Lk, D, type=t), normal(g, B, D, type=t),
            torch.tensor([Lk, 17, 1][:B], dtype=torch.int32, device="cuda"), normal(g, B, L, D, type=t))


@pytest.mark.parametrize("t", HALF)
def test_a_layer_runs_and_its_gradients_are_those_of_the_formula(t):
    """16-bit tensors between the operators: at most 12 roundings lie between an input and a gradient, each at most half a step of values
    of the gradient's size, so the difference's 2-norm stays within 12 half steps of the gradient's"""
    layer, (x, ctx, gate, n, d) = Layer(t=t), layer_inputs(t)
    y, kept = layer.forward(x, ctx, gate, n, save=True)
    got = layer.backward(d, kept)
    xs = [v.double().requires_grad_(True) for v in (x, ctx, gate)]
    want = layer.plain(*xs, n)
    grads = dict(zip(("x", "ctx", "gate", *layer.p), torch.autograd.grad(want, xs + list(layer.p.values()), d.double())))
    tol = 12 * ref.half_step(t)
    want = want.detach()
    assert float((y.double() - want).norm()) <= tol * float(want.norm())
    for name, g in got.items():
        assert float((g.double() - grads[name]).norm()) <= tol * float(grads[name].norm()), name


def test_the_layer_in_a_graph_replays_with_new_inputs():
    """forward and backward captured; every replay equals the eager run on the same inputs, with eager work and new lengths in between"""
    layer, (x, ctx, gate, n, d) = Layer(), layer_inputs()

    def step():
        y, kept = layer.forward(x, ctx, gate, n, save=True)
        return [y, *layer.backward(d, kept).values()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for i in range(4):
        x.copy_(normal(gen(90 + i), *x.shape, type=BF16))
        n.copy_(torch.tensor([90 - 7 * i, 20 * i, i], dtype=torch.int32, device="cuda"))
        want = [v.clone() for v in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(res, want):
            assert torch.equal(a, b)


def test_two_graphs_in_flight_do_not_share_a_workspace():
    cases = [xattn_inputs((2, 2, 1, 3000, 4, 2, 64, "len"), BF16, seed=s) for s in (1, 2)]
    graphs, outs, want = [], [], []
    for q, k, v, _, m in cases:
        want.append(blocks().cross_attention(q, k, v, **m))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = blocks().cross_attention(q, k, v, **m)
        graphs.append(g)
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_calls_on_another_stream_and_the_same_bits_every_time():
    q, k, v, dout, m = xattn_inputs((4, 1, 30, 500, 2, 2, 128, "holes"), BF16)
    out, lse = blocks().cross_attention(q, k, v, **m)
    d = blocks().cross_attention_backward(dout, q, k, v, out, lse, **m)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            o2, l2 = blocks().cross_attention(q, k, v, **m)
            d2 = blocks().cross_attention_backward(dout, q, k, v, o2, l2, **m)
    side.synchronize()
    assert torch.equal(o2, out) and torch.equal(l2, lse) and all(torch.equal(a, b) for a, b in zip(d, d2))


def test_two_streams_at_once():
    """every operator on two streams that run side by side, each with its own inputs: the bits of one after the other"""
    a = [ffn_inputs(300, 256, 1032, BF16, True, seed=s) for s in (1, 2)]
    c = [xattn_inputs((3, 1, 40, 2500, 4, 2, 64, "holes"), BF16, seed=s) for s in (1, 2)]
    n = [norm_inputs(4, 50, 640, BF16, ("rms", "layer"), True, seed=s) for s in (1, 2)]

    def work(i):
        (f, b, dy), (q, k, v, do, m), (x, y, dr, dz, na) = a[i], c[i], n[i]
        w = [f["wg"], f["wu"], f["wd"]]
        yy, saved = blocks().gated_ffn(f["x"], *w, *b, save=True)
        o, lse = blocks().cross_attention(q, k, v, **m)
        r, z, st = blocks().block_norm(x, y, save=True, **na)
        return [yy, *blocks().gated_ffn_backward(dy, f["x"], *w, saved, bias=True).values(), o, lse,
                *blocks().cross_attention_backward(do, q, k, v, o, lse, **m), r, z, *blocks().block_norm_backward(dr, dz, x, y, st, **na).values()]
    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = work(i)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert len(g) == len(w) and all(torch.equal(x, y) for x, y in zip(g, w))


def test_threads_that_call_at_once():
    """four host threads, a stream each, the same calls: the bits of a call alone"""
    import threading

    q, k, v, dout, m = xattn_inputs((2, 1, 40, 300, 4, 2, 72, "holes"), FP16)
    a, b, dy = ffn_inputs(70, 136, 264, FP16, True)
    w = [a["wg"], a["wu"], a["wd"]]

    def work():
        o, lse = blocks().cross_attention(q, k, v, **m)
        y, saved = blocks().gated_ffn(a["x"], *w, *b, save=True)
        return [o, lse, *blocks().cross_attention_backward(dout, q, k, v, o, lse, **m), y,
                *blocks().gated_ffn_backward(dy, a["x"], *w, saved, bias=True).values()]
    want = work()
    torch.cuda.synchronize()
    got = [None] * 4

    def run(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(5):
                got[i] = work()
        st.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g in got:
        assert g is not None and all(torch.equal(x, y) for x, y in zip(g, want))


def test_nothing_is_written_past_the_results():
    """results inside larger buffers through the C ABI: what lies around them stays"""
    import ctypes as C

    from isbfsar_amd import _lib
    lib = _lib.lib()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for Lq, D in ((3, 72), (50, 40)):
        q, k, v, _, _ = xattn_inputs((1, 1, Lq, 70, 2, 2, D, ""), BF16)
        buf = torch.full((q.numel() + 1024,), 7.0, dtype=BF16, device="cuda")
        lse = torch.full((2 * Lq + 512,), 7.0, device="cuda")
        a = _lib.isb_xattn_args(0, 2, 1, 1, Lq, 70, 2, 2, D, 0.1, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride()[:3], k.stride()[:3], v.stride()[:3])
        a.out, a.lse = buf.data_ptr() + 1024, lse.data_ptr() + 1024
        n = C.c_size_t()
        _lib.check(lib.isb_xattn_workspace(C.byref(a), 0, C.byref(n)), "workspace")
        ws = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
        _lib.check(lib.isb_xattn_forward(C.byref(a), ws.data_ptr(), n.value, st), "forward")
        assert bool((buf[:512] == 7).all()) and bool((buf[512 + q.numel():] == 7).all())
        assert bool((lse[:256] == 7).all()) and bool((lse[256 + 2 * Lq:] == 7).all())
        held(buf[512:512 + q.numel()].view(q.shape), *ref.xattn(q, k, v, scale=0.1)["out"], "out")


@pytest.mark.parametrize("M,D,F", [(1, 72, 136), (3, 72, 136), (70, 72, 136), (300, 136, 264)])
def test_ffn_and_norm_write_nothing_past_their_results(M, D, F):
    import ctypes as C

    from isbfsar_amd import _lib
    lib = _lib.lib()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def around(n, t=BF16):
        b = torch.full((n + 1024,), 7.0, dtype=t, device="cuda")
        return b, b.data_ptr() + 512 * b.element_size(), n

    def kept(b, _, n):
        return bool((b[:512] == 7).all()) and bool((b[512 + n:] == 7).all())
    a, b, dy = ffn_inputs(M, D, F, BF16, True)
    o = {"y": around(M * D), "pre_gate": around(M * F, F32), "pre_up": around(M * F, F32), "hidden": around(M * F), "dx": around(M * D),
         "dw_gate_up": around(2 * F * D), "dw_down": around(D * F), "db_gate": around(F), "db_up": around(F), "db_down": around(D)}
    args = _lib.isb_ffn_args(0, 2, M, D, F, 0, D, D, a["x"].data_ptr(), a["wg"].data_ptr(), a["wu"].data_ptr(), a["wd"].data_ptr(),
                             b[0].data_ptr(), b[1].data_ptr(), b[2].data_ptr())
    args.dy = dy.data_ptr()
    for name, v in o.items():
        setattr(args, name, v[1])
    for back, call in ((0, lib.isb_ffn_forward), (1, lib.isb_ffn_backward)):
        n = C.c_size_t()
        _lib.check(lib.isb_ffn_workspace(C.byref(args), back, C.byref(n)), "workspace")
        ws = torch.full((n.value + 4096,), 9, dtype=torch.uint8, device="cuda")
        _lib.check(call(C.byref(args), ws.data_ptr(), n.value, st), "call")
        assert bool((ws[n.value:] == 9).all())
    for name, v in o.items():
        assert kept(*v), name
    x, y, dr, dz, na = norm_inputs(2, M, D, BF16, ("layer", "layer"), True)
    rows = 2 * M * D
    o = {"r": around(rows), "z": around(rows), "stats": around(8 * M, F32), "dx": around(rows), "dy": around(rows), "dgate": around(2 * D),
         "dscale": around(D, F32), "dpre_bias": around(D, F32)}
    args = _lib.isb_norm_args(0, 2, 2, M, D, 1, 1, 1e-5, x.data_ptr(), y.data_ptr(), na["gate"].data_ptr(), na["scale"].data_ptr())
    args.dr, args.dz = dr.data_ptr(), dz.data_ptr()
    for name, v in o.items():
        setattr(args, name, v[1])
    n = C.c_size_t()
    _lib.check(lib.isb_norm_workspace(C.byref(args), C.byref(n)), "workspace")
    ws = torch.full((n.value + 4096,), 9, dtype=torch.uint8, device="cuda")
    _lib.check(lib.isb_norm_forward(C.byref(args), st), "forward")
    _lib.check(lib.isb_norm_backward(C.byref(args), ws.data_ptr(), n.value, st), "backward")
    assert bool((ws[n.value:] == 9).all())
    for name, v in o.items():
        assert kept(*v), name


def test_a_device_that_is_not_there():
    """the call fails with the library's error, and neither the thread's device nor the next launch notices"""
    import ctypes as C

    from isbfsar_amd import _lib
    x, _, _, _, a = norm_inputs(1, 3, 64, F32, (None, "layer"), False)
    z = blocks().block_norm(x, pre="layer")[1]
    got = torch.zeros_like(x)
    args = _lib.isb_norm_args(63, 0, 1, 3, 64, 0, 1, 1e-5, x.data_ptr())
    args.z = got.data_ptr()
    assert _lib.lib().isb_norm_forward(C.byref(args), None) == -3 and b"device 63" in _lib.lib().isb_last_error()
    assert torch.cuda.current_device() == 0 and torch.equal(blocks().block_norm(x, pre="layer")[1], z) and not got.any()


def test_the_engine_s_embeddings_go_in():
    """embeddings of query windows against the frames of the installed support set (ArEngine), shared by all windows"""
    from isbfsar_amd import synth, weights
    from isbfsar_amd.engine import ArEngine
    L, J, way, B = 16, 30, 5, 6
    eng = ArEngine(L, J, way)
    eng.load_weights(weights.make_ar_state(L, J, seed=0))
    eng.set_support(poses=synth.skeleton_windows(way, L, J, seed=100))
    _, _, emb = eng.infer(torch.from_numpy(synth.skeleton_windows(B, L, J, seed=200)).cuda(), want_embed=True)
    frames = torch.from_numpy(eng.support_features()).cuda().reshape(1, way * L, 2, 128).half()
    q = emb.half().view(B, L, 2, 128)
    out, lse = blocks().cross_attention(q, frames, frames)
    want = ref.xattn(q, frames, frames)
    held(out, *want["out"], "out")
    held(lse, *want["lse"], "lse")
    eng.close()
