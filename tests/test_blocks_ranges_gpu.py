"""GPU tests of the layer operators (isbfsar_amd/blocks.py) where a value's size is what matters: intermediates past fp16's range or below
its normal numbers while the results lie inside, activations far out on their tails, weights far below a row's largest.

Bounds, beside those of blocks_ref: u is half a step of the type, e = 2^-24. What the feed-forward block keeps in fp16 between its products (h,
dG, dU) carries a power of two per group of 8 rows x 32 features, chosen from the group's largest magnitude m: none while 2^-10 <= m <= 65504, up
by 2^16, 2^32, ... below, down by just enough above. A value is then off by u of itself or by half an fp16 step of 2^-24 times the power, and a
product brings the groups that it adds up to the largest of their powers. With m the largest magnitude of what is added up that half step is at
most 2^-25 (m in between), 2^-25 2^10 m (below) or 2^-25 2^-14 m (above); it is counted twice, for the store and for the common power."""
import math

import pytest
import torch

import blocks_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def blocks():
    from isbfsar_amd import blocks as b
    return b


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, type=F32, std=1.0):
    return torch.empty(shape, device="cuda", dtype=F32).normal_(0, std, generator=g).to(type)


def held(got, want, bound, name):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.double() - want).abs() - bound
    assert not off.isnan().any() and bool((off <= 0).all()), (name, float(off.nan_to_num(math.inf).max()), float((got.double() - want).abs().max()),
                                                              float(((got.double() - want).abs() / bound).max()))


# ------------------------------------------------------------------------------------------------ gated feed-forward block, fp16
def step16(m):
    """twice half a step of fp16 values whose power of two follows the magnitude m (see above)"""
    return 2 * torch.where(m < 2.0 ** -10, 2.0 ** -15 * m, torch.where(m <= 65504, 2.0 ** -25, 2.0 ** -39 * m))


def groups(x, rows, cols):
    """the largest magnitude of each group of `rows` x `cols` (0: all of them), for every element"""
    M, N = x.shape
    r, c = rows or M, cols or N
    pad = torch.nn.functional.pad(x.abs(), (0, -N % c, 0, -M % r))
    m = pad.view(pad.shape[0] // r, r, pad.shape[1] // c, c).amax((1, 3))
    return m.repeat_interleave(r, 0).repeat_interleave(c, 1)[:M, :N]


def ffn16(x, wg, wu, wd, act, dy=None):
    """{name: (value, bound)} in fp16 with f32 sums: blocks_ref.ffn with the half steps of step16"""
    u = 2.0 ** -11
    M, D = x.shape
    F = wg.shape[0]
    X, G, U, W = (a.double() for a in (x, wg, wu, wd))
    g, v = X @ G.T, X @ U.T
    eg, ev = ((X.abs() @ w.abs().T) * (D + 4) * E for w in (G, U))
    a, da = ref.act(act, g)
    ea, eda = 1.2 * eg + 16 * E * (1 + g.abs()), eg + 16 * E * (1 + g.abs())
    if act == "relu":
        eda = torch.where(g.abs() <= eg, 1.0, 0.0)
    h = a * v
    eh = h.abs() * (u + 2 * E) + (ea * v.abs() + (a.abs() + ea) * ev) * (1 + u)
    e_row = eh + (step16(groups(h, 8, 0)) if M > 4 else 0)                        # one to four rows keep h in f32
    y = h @ W.T
    out = lambda val, err: (val, u * val.abs() + err * (1 + u) + 2.0 ** -25)      # noqa: E731
    r = {"y": out(y, e_row @ W.abs().T + (F + 8) * E * (h.abs() @ W.abs().T))}
    if dy is None:
        return r
    Y = dy.double()
    dh, edh = Y @ W, (Y.abs() @ W.abs()) * (D + 4) * E
    dg, dv = dh * v * da, dh * a
    edg = dg.abs() * (u + 4 * E) + (edh * v.abs() * da.abs() + dh.abs() * (ev * da.abs() + (v.abs() + ev) * eda)) * (1 + u)
    edv = dv.abs() * (u + 4 * E) + (edh * a.abs() + (dh.abs() + edh) * ea) * (1 + u)
    both = step16(torch.maximum(groups(dg, 8, 0), groups(dv, 8, 0)))
    n = M + 8
    r["dx"] = out(dg @ G + dv @ U, (edg + both) @ G.abs() + (edv + both) @ U.abs() + (2 * F + 8) * E * (dg.abs() @ G.abs() + dv.abs() @ U.abs()))
    for name, d, ed in (("dw_gate", dg, edg), ("dw_up", dv, edv)):
        r[name] = out(d.T @ X, (ed + step16(groups(d, 0, 32))).T @ X.abs() + n * E * (d.abs().T @ X.abs()))
    r["dw_down"] = out(Y.T @ h, Y.abs().T @ (eh + step16(groups(h, 0, 32))) + n * E * (Y.abs().T @ h.abs()))
    return r


def check_ffn16(x, wg, wu, wd, act, dy, names=("y", "dx", "dw_gate", "dw_up", "dw_down")):
    y, saved = blocks().gated_ffn(x, wg, wu, wd, activation=act, save=True)
    d = {"y": y, **blocks().gated_ffn_backward(dy, x, wg, wu, wd, saved, activation=act)}
    want = ffn16(x, wg, wu, wd, act, dy)
    for name in names:
        assert bool((want[name][0].abs() < 65504).all()), name
        held(d[name], *want[name], name)


@pytest.mark.parametrize("M", [1, 4, 5, 40, 300])
def test_ffn_hidden_values_past_the_type_s_range(M):
    """h = 320 x 320 = 102400 does not fit fp16, y = 64 h / 256 = 25600 and dw_down = M h / 1024 = 100 M do, exactly"""
    x = torch.full((M, 64), 8.0, dtype=FP16, device="cuda")
    w = torch.full((64, 64), 0.625, dtype=FP16, device="cuda")
    wd = torch.full((64, 64), 2.0 ** -8, dtype=FP16, device="cuda")
    y, saved = blocks().gated_ffn(x, w, w, wd, activation="relu", save=True)
    assert bool((y == 25600).all())
    d = blocks().gated_ffn_backward(torch.full_like(x, 2.0 ** -10), x, w, w, wd, saved, activation="relu")
    assert bool((d["dw_down"] == 100 * M).all())
    assert bool((blocks().gated_ffn(x, w, w, wd, activation="relu") == 25600).all())


@pytest.mark.parametrize("M,D,F", [(5, 64, 136), (37, 128, 520), (300, 136, 1032), (1500, 264, 2056)])
@pytest.mark.parametrize("act", ["relu", "silu", "sigmoid"])
def test_ffn_rows_of_very_different_size(M, D, F, act):
    """rows of x from 2^-8 to 2^8: h spans more than fp16, and a row of large hidden values leaves the digits of the rows behind its group alone"""
    g = gen(M + F)
    x = (normal(g, M, D) * 2.0 ** torch.randint(-8, 9, ((M + 15) // 16, 1), generator=g, device="cuda").repeat_interleave(16, 0)[:M]).to(FP16)
    w = [normal(g, F, D, type=FP16, std=4 * D ** -0.5) for _ in range(2)]
    wd = normal(g, D, F, type=FP16, std=2.0 ** -8 * F ** -0.5)
    check_ffn16(x, *w, wd, act, normal(g, M, D, type=FP16, std=2.0 ** -10), ("y", "dw_down"))


@pytest.mark.parametrize("std", [2.0 ** -8, 2.0 ** -12, 2.0 ** -18, 2.0 ** -22])
@pytest.mark.parametrize("M,D,F", [(3, 64, 136), (33, 136, 520), (300, 72, 1032), (2101, 264, 1160)])
def test_ffn_small_gradients_keep_their_digits(M, D, F, std):
    """dy far below fp16's normal numbers' middle: dG and dU must not lose what dx and the weights' gradients can hold"""
    g = gen(M)
    x, dy = normal(g, M, D, type=FP16), normal(g, M, D, std=std).to(FP16)
    w = [normal(g, F, D, type=FP16, std=D ** -0.5) for _ in range(2)]
    check_ffn16(x, *w, normal(g, D, F, type=FP16, std=F ** -0.5), "silu", dy)


@pytest.mark.parametrize("M,D,F", [(12, 64, 136), (300, 72, 1032), (1030, 264, 520), (2101, 264, 2056)])
def test_ffn_gradients_of_very_different_size(M, D, F):
    """rows of dy from 2^-20 to 2^6 in blocks that end inside tiles, features of the up projection from 2^-12 to 2^2: every group of dG and dU has
    its own power of two"""
    g = gen(M + 1)
    x = normal(g, M, D, type=FP16)
    dy = (normal(g, M, D) * 2.0 ** torch.randint(-20, 7, ((M + 11) // 12, 1), generator=g, device="cuda").repeat_interleave(12, 0)[:M]).to(FP16)
    dy[:3] = 0
    wu = normal(g, F, D) * 2.0 ** torch.randint(-12, 3, ((F + 39) // 40, 1), generator=g, device="cuda").repeat_interleave(40, 0)[:F]
    check_ffn16(x, normal(g, F, D, type=FP16, std=D ** -0.5), (wu * D ** -0.5).to(FP16), normal(g, D, F, type=FP16, std=F ** -0.5), "gelu", dy)


@pytest.mark.parametrize("M,D,F", [(3, 64, 136), (40, 64, 264), (300, 136, 520)])
def test_ffn_gradients_past_the_type_s_range(M, D, F):
    """dG past 65504, the weights' gradients inside"""
    g = gen(M + 2)
    x = normal(g, M, D, type=FP16, std=2.0 ** -9)
    dy = normal(g, M, D, type=FP16, std=2.0 ** 8)
    wg, wu = normal(g, F, D, type=FP16, std=2.0 ** -10), normal(g, F, D, type=FP16, std=2.0 ** 8)
    wd = normal(g, D, F, type=FP16, std=2.0 ** 6)
    v, dh = x.double() @ wu.double().T, dy.double() @ wd.double()
    assert float((dh * v / 4).abs().max()) > 65504
    check_ffn16(x, wg, wu, wd, "sigmoid", dy, ("dw_gate", "dw_up"))


@pytest.mark.parametrize("M", [12, 300])
def test_ffn_an_infinite_gradient_row_leaves_the_others_alone(M):
    """a row of dy with an infinity: dx of the other rows is what it is without it, within its bound"""
    g = gen(M + 3)
    x, dy = normal(g, M, 64, type=FP16), normal(g, M, 64, std=2.0 ** -14).to(FP16)
    w = [normal(g, 136, 64, type=FP16, std=0.125) for _ in range(2)] + [normal(g, 64, 136, type=FP16, std=0.1)]
    y, saved = blocks().gated_ffn(x, *w, save=True)
    want = ffn16(x, *w, "silu", dy)["dx"]
    bad = dy.clone()
    bad[5, 7] = math.inf
    d = blocks().gated_ffn_backward(bad, x, *w, saved)["dx"]
    assert not d[5].isfinite().any()
    d[5] = want[0][5].to(FP16)
    held(d, *want, "dx")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("M", [3, 5, 260])
def test_ffn_an_infinite_weight_reaches_the_bias_gradients_as_it_is(M, t):
    """dh = inf in one feature of every row: db_up there is inf -- the rows that fill a tile up behind the last one must not make a NaN of it"""
    a = [torch.ones(M, 64, dtype=t, device="cuda"), *(torch.full((136, 64), 2.0 ** -6, dtype=t, device="cuda") for _ in range(2))]
    wd = torch.full((64, 136), 2.0 ** -6, dtype=t, device="cuda")
    wd[5, 77] = math.inf
    y, saved = blocks().gated_ffn(*a, wd, activation="sigmoid", save=True)
    d = blocks().gated_ffn_backward(torch.ones_like(a[0]), *a, wd, saved, bias=True, activation="sigmoid")
    for n in ("db_gate", "db_up"):
        assert float(d[n][77]) == math.inf and bool(d[n][:77].isfinite().all()) and bool(d[n][78:].isfinite().all()), n


@pytest.mark.parametrize("M", [1, 4, 5])
def test_ffn_weights_below_the_normal_numbers(M):
    """weights of 2^-20 (fp16 holds them as subnormal numbers): g = 64 x 2^-20 = 2^-14, u = 1, y = 64 x 2^-14 x 4096 = 16, exactly"""
    x = torch.ones(M, 64, dtype=FP16, device="cuda")
    wg, wu, wd = (torch.full((64, 64), v, dtype=FP16, device="cuda") for v in (2.0 ** -20, 2.0 ** -6, 4096.0))
    assert bool((blocks().gated_ffn(x, wg, wu, wd, activation="relu") == 16).all())
    assert bool((blocks().gated_ffn(x * 2.0 ** -18, wg * 2.0 ** 20, wu * 2.0 ** 18, wd, activation="relu") == 64 * 2.0 ** -12 * 4096 * 1).all())


# ------------------------------------------------------------------------------------------------ activations' tails
def tail(act, M):
    """a feed-forward block that hands its activation through: g = the bias, u = 1, w_down = 1 -> y = act(g), db_gate = M act'(g)"""
    n = 64
    bg = torch.linspace(-20, 20, n, device="cuda").to(BF16)
    one, nul = torch.ones(n, dtype=BF16, device="cuda"), torch.zeros(n, n, dtype=BF16, device="cuda")
    x, eye = torch.zeros(M, n, dtype=BF16, device="cuda"), torch.eye(n, device="cuda").to(BF16)
    y, saved = blocks().gated_ffn(x, nul, nul, eye, bg, one, torch.zeros_like(one), activation=act, save=True)
    d = blocks().gated_ffn_backward(torch.ones_like(x), x, nul, nul, eye, saved, bias=True, activation=act)
    g = bg.double()
    if act == "gelu":
        phi = 0.5 * torch.erfc(-g / math.sqrt(2))
        return y, d["db_gate"], g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s, c = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    return (y, d["db_gate"], s, s * c) if act == "sigmoid" else (y, d["db_gate"], g * s, s * (1 + g * c))


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("M", [1, 5])
def test_ffn_activations_keep_their_digits_on_the_tails(act, M):
    """values relative to themselves: h and y are rounded once each (half a step of bf16, 2^-8), the functions are good to 2^-14 of what they
    return: e^-x to x 2^-23 relative (x <= 20; 200 for GELU's e^-xx/2), a handful of f32 steps. The slopes of SiLU and GELU pass through
    zero: to 2^-14 of their two terms' magnitudes. db_gate is rounded once. bf16 and f32 end at 2^-126 alike: what lies below (GELU from -13 on) may
    come out as anything up to that."""
    y, db, want, slope = tail(act, M)
    half = 2.0 ** -8
    held(y, want.expand(M, -1), (want.abs() * (2 * half + half * half + 2.0 ** -14) + 2.0 ** -126).expand(M, -1), "y")
    terms = slope.abs()
    if act == "silu":
        g = torch.linspace(-20, 20, 64, device="cuda").to(BF16).double()
        terms = 1 / (1 + torch.exp(-g)) * (1 + g.abs() / (1 + torch.exp(g)))
    if act == "gelu":
        g = torch.linspace(-20, 20, 64, device="cuda").to(BF16).double()
        terms = 0.5 * torch.erfc(-g / math.sqrt(2)) + g.abs() * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    held(db, M * slope, M * (slope.abs() * half + terms * 2.0 ** -14 * (1 + half)) + M * 2.0 ** -126, "db_gate")


# ------------------------------------------------------------------------------------------------ cross attention, fp16
@pytest.mark.parametrize("Lq,Lk", [(1, 2000), (1, 20000), (40, 2000), (40, 20000), (700, 2000)])
def test_xattn_weights_far_below_a_row_s_largest(Lq, Lk):
    """one state of weight 1 and value 0, all others of weight e^-17 = 2^-24.5 and value 1: together they make the result, and their weights must
    not be rounded to steps of 2^-24. A weight is rounded to half a step u = 2^-11 (normal numbers), the result once more; f32's part is Lk e at most"""
    q = torch.zeros(1, Lq, 1, 64, dtype=FP16, device="cuda")
    k, v = torch.zeros(1, Lk, 1, 64, dtype=FP16, device="cuda"), torch.ones(1, Lk, 1, 64, dtype=FP16, device="cuda")
    q[..., 0] = 1
    k[:, 1:, :, 0] = -17
    v[:, 0] = 0
    out, lse = blocks().cross_attention(q, k, v, scale=1.0)
    w = (Lk - 1) * math.exp(-17)
    want = torch.full(out.shape, w / (1 + w), dtype=torch.float64, device="cuda")
    held(out, want, want * (2 * 2.0 ** -11 + 2 ** -22 + (Lk + 64) * E) + 2.0 ** -25, "out")
    held(lse, torch.full(lse.shape, math.log1p(w), dtype=torch.float64, device="cuda"), torch.full(lse.shape, (Lk + 64) * E * 2, dtype=torch.float64, device="cuda"), "lse")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("B,Bk,Lq,Lk,Hq,Hk,D,lens", [
    (1, 1, 1, 2, 1, 1, 64, None), (4, 4, 1, 5, 4, 4, 96, None), (11, 1, 4, 5, 4, 1, 64, None), (2, 2, 1, 54, 1, 1, 128, [54, 27]), (3, 3, 3, 32, 2, 2, 72, [32, 1, 9]),
    (2, 2, 40, 64, 2, 2, 128, [64, 33]), (3, 3, 200, 30, 2, 1, 64, [30, 2, 4]), (4, 4, 1, 300, 2, 2, 64, [2, 3, 60, 31]), (2, 2, 70, 2500, 1, 1, 128, [4, 40]),
    (3, 3, 130, 700, 1, 1, 128, [5, 33, 64])])
def test_xattn_few_states_or_rows(B, Bk, Lq, Lk, Hq, Hk, D, lens, t):
    """up to 64 states enter P and dS whole (two operands: u^2 of a rounding is left, and fp16's steps of 2^-24 behind 2^12 P and a dS of 2^10), up to
    64 rows the same for dk and dv; up to 32 states delta is sum P dP in f32 (before, out's rounding stood in it). What is left: one rounding u
    of each result and f32's part -- ep as in blocks_ref, D + 16 terms in dP, Lk + 16 in delta."""
    g = gen(D + Lk)
    q, dout = normal(g, B, Lq, Hq, D, type=t), normal(g, B, Lq, Hq, D, type=t)
    k, v = normal(g, Bk, Lk, Hk, D, type=t), normal(g, Bk, Lk, Hk, D, type=t)
    kv_len = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = blocks().cross_attention(q, k, v, kv_len=kv_len)
    dq, dk, dv = blocks().cross_attention_backward(dout, q, k, v, out, lse, kv_len=kv_len)
    u, G, nb, scale = ref.half_step(t), Hq // Hk, B // Bk, 1 / math.sqrt(D)
    rest = u * u + 2 * E
    for b in range(Bk):
        n = Lk if lens is None else lens[b]
        for h in range(Hk):
            bs, hs = slice(b * nb, (b + 1) * nb), slice(h * G, (h + 1) * G)
            Q, dO = (x[bs, :, hs].double().reshape(-1, D) for x in (q, dout))
            K, V = k[b, :n, h].double(), v[b, :n, h].double()
            s = Q @ K.T * scale
            P = torch.softmax(s, -1)
            es = ((Q.abs() @ K.abs().T) * scale * (D + 4) * E + s.abs() * 4 * E).amax(-1, keepdim=True)
            ep = 2 * es + 8 * E + (n + 64) * E
            o = P @ V
            held(out[bs, :, hs].reshape(-1, D), o, u * o.abs() + (P @ V.abs()) * (ep + rest) * (1 + u) + 2.0 ** -25 + (2.0 ** -36 if t == FP16 else 0) * V.abs().sum(0), "out")
            dP = dO @ V.T
            abs_dP = dO.abs() @ V.abs().T
            delta = (P * dP).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            edelta = (P * abs_dP).sum(-1, keepdim=True) * (ep + (D + n + 32) * E)
            if n > 32:                                                      # rowsum(dout o out) with out as it was rounded
                edelta = edelta + (dO.abs() * (u * o.abs() + 2.0 ** -25)).sum(-1, keepdim=True)
            edS = dS.abs() * (ep + rest) + P * (edelta + (D + 16) * E * abs_dP) * (1 + u)
            tiny = 2.0 ** -34 if t == FP16 else 0.0
            want = dS @ K * scale
            held(dq[bs, :, hs].reshape(-1, D), want, u * want.abs() + scale * ((edS + tiny * dS.abs().amax(-1, keepdim=True)) @ K.abs()) * (1 + u) + 2.0 ** -25, "dq")
            M = Q.shape[0]
            if M > 64:
                continue
            want = dS.T @ Q * scale
            held(dk[b, :n, h], want, u * want.abs() + scale * ((edS + tiny * dS.abs().amax(0)).T @ Q.abs() + (M + 16) * E * (dS.abs().T @ Q.abs())) * (1 + u) + 2.0 ** -25, "dk")
            want = P.T @ dO
            held(dv[b, :n, h], want, u * want.abs() + ((P * (ep + rest)).T @ dO.abs() + (M + 16) * E * (P.T @ dO.abs())) * (1 + u) + 2.0 ** -25
                 + (2.0 ** -36 if t == FP16 else 0) * dO.abs().sum(0), "dv")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hk,D", [(1, 1, 70, 1, 1, 64), (2, 1, 300, 4, 2, 128), (5, 3, 150, 8, 2, 72), (70, 4, 200, 4, 1, 64), (1, 32, 400, 1, 1, 64)])
def test_xattn_few_rows_of_dq(B, Lq, Lk, Hq, Hk, D, t):
    """up to 32 rows of a group: dS enters whole (two operands), whatever the states. delta is rowsum(dout o out) of the out that is handed in: with
    that one in the formula, what is left is one rounding u of the result and f32's part (ep as in blocks_ref)"""
    g = gen(Lk)
    q, dout = normal(g, B, Lq, Hq, D, type=t), normal(g, B, Lq, Hq, D, type=t)
    k, v = normal(g, B, Lk, Hk, D, type=t), normal(g, B, Lk, Hk, D, type=t)
    out, lse = blocks().cross_attention(q, k, v)
    dq = blocks().cross_attention_backward(dout, q, k, v, out, lse)[0]
    u, G, scale = ref.half_step(t), Hq // Hk, 1 / math.sqrt(D)
    rows = lambda x: x.double().unflatten(2, (Hk, G)).permute(0, 2, 1, 3, 4).reshape(B, Hk, Lq * G, D)     # noqa: E731
    Q, dO, o, got = (rows(x) for x in (q, dout, out, dq))
    K, V = (x.double().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    T = lambda x: x.transpose(-1, -2).contiguous()     # noqa: E731
    s = Q @ T(K) * scale
    P = torch.softmax(s, -1)
    es = ((Q.abs() @ T(K.abs())) * scale * (D + 4) * E + s.abs() * 4 * E).amax(-1, keepdim=True)
    ep = 2 * es + 8 * E + (Lk + 64) * E
    abs_dP = dO.abs() @ T(V.abs())
    dS = P * (dO @ T(V) - (dO * o).sum(-1, keepdim=True))
    edS = dS.abs() * (ep + u * u + 2 * E) + P * ((D + 16) * E * (abs_dP + (dO * o).abs().sum(-1, keepdim=True))) * (1 + u)
    if t == FP16:
        edS = edS + 2.0 ** -34 * dS.abs().amax(-1, keepdim=True)
    want = dS @ K * scale
    held(got, want, u * want.abs() + scale * (edS @ K.abs() + (Lk + 64) * E * (dS.abs() @ K.abs())) * (1 + u) + 2.0 ** -25, "dq")


@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("Lq,Lk", [(1, 5), (3, 40), (40, 60), (130, 20), (70, 300)])
def test_xattn_an_infinity_stays_one(Lq, Lk, t):
    """an infinite value of a valid state makes that column of every row's result infinite (not NaN), an infinite gradient that column of dv"""
    q, k, v, dout = (normal(gen(9 + i), 1, n, 1, 64, type=t) for i, n in enumerate((Lq, Lk, Lk, Lq)))
    inf = v.clone()
    inf[0, Lk // 2, 0, 3], inf[0, Lk - 1, 0, 9] = math.inf, -math.inf
    out, _ = blocks().cross_attention(q, k, inf)
    assert bool((out[..., 3] == math.inf).all()) and bool((out[..., 9] == -math.inf).all()) and int((~out.isfinite()).sum()) == 2 * Lq
    out, lse = blocks().cross_attention(q, k, v)
    dout[0, Lq // 2, 0, 7] = math.inf
    dv = blocks().cross_attention_backward(dout, q, k, v, out, lse)[2]
    assert bool((dv[..., 7] == math.inf).all()) and int((~dv.isfinite()).sum()) == Lk


# ------------------------------------------------------------------------------------------------ the powers of two in use
def odd_ffn(M, D, F, seed=0):
    """a block whose h, dG and dU need powers of two of every kind"""
    g = gen(seed + M)
    x = (normal(g, M, D) * 2.0 ** torch.randint(-9, 9, ((M + 8) // 9, 1), generator=g, device="cuda").repeat_interleave(9, 0)[:M]).to(FP16)
    dy = (normal(g, M, D) * 2.0 ** torch.randint(-20, 0, ((M + 8) // 9, 1), generator=g, device="cuda").repeat_interleave(9, 0)[:M]).to(FP16)
    w = [normal(g, F, D, type=FP16, std=4 * D ** -0.5) for _ in range(2)] + [normal(g, D, F, type=FP16, std=2.0 ** -8 * F ** -0.5)]
    return x, w, dy


@pytest.mark.parametrize("M,D,F", [(3, 64, 136), (45, 72, 264), (700, 136, 520)])
def test_ffn_backward_again_in_a_graph_and_on_two_streams(M, D, F):
    """the backward call may write the saved hidden values anew: a second call on them, replays and two calls at once give the same bits"""
    x, w, dy = odd_ffn(M, D, F)

    def forward():
        return blocks().gated_ffn(x, *w, activation="gelu", save=True)

    def backward(saved):
        return list(blocks().gated_ffn_backward(dy, x, *w, saved, bias=True, activation="gelu").values())
    y, saved = forward()
    want = backward(saved)
    assert all(torch.equal(a, b) for a, b in zip(backward(saved), want))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = backward(saved)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y2, s2 = forward()
        res = backward(s2)
    for i in range(3):
        x2, _, dy2 = odd_ffn(M, D, F, seed=i)
        x.copy_(x2)
        dy.copy_(dy2)
        graph.replay()
        torch.cuda.synchronize()
        y, saved = forward()
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(res, backward(saved)))


@pytest.mark.parametrize("M,D,F", [(3, 72, 136), (45, 72, 136), (300, 136, 264)])
def test_ffn_with_powers_writes_nothing_past_its_results(M, D, F):
    import ctypes as C

    from isbfsar_amd import _lib
    lib = _lib.lib()
    x, w, dy = odd_ffn(M, D, F)

    def around(n, t=FP16):
        b = torch.full((n + 1024,), 7.0, dtype=t, device="cuda")
        return b, b.data_ptr() + 512 * b.element_size(), n
    o = {"y": around(M * D), "pre_gate": around(M * F, F32), "pre_up": around(M * F, F32), "hidden": around(M * F), "dx": around(M * D),
         "dw_gate_up": around(2 * F * D), "dw_down": around(D * F), "db_gate": around(F), "db_up": around(F), "db_down": around(D)}
    args = _lib.isb_ffn_args(0, 1, M, D, F, 0, D, D, x.data_ptr(), *(v.data_ptr() for v in w))
    args.dy = dy.data_ptr()
    for name, v in o.items():
        setattr(args, name, v[1])
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for back, call in ((0, lib.isb_ffn_forward), (1, lib.isb_ffn_backward)):
        n = C.c_size_t()
        _lib.check(lib.isb_ffn_workspace(C.byref(args), back, C.byref(n)), "workspace")
        ws = torch.full((n.value + 4096,), 0x55, dtype=torch.uint8, device="cuda")      # (also what the tables hold before they are written)
        _lib.check(call(C.byref(args), ws.data_ptr(), n.value, st), "call")
        assert bool((ws[n.value:] == 0x55).all())
    for name, (b, _, n) in o.items():
        assert bool((b[:512] == 7).all()) and bool((b[512 + n:] == 7).all()), name
    y, saved = blocks().gated_ffn(x, *w, save=True)
    d = blocks().gated_ffn_backward(dy, x, *w, saved, bias=True)
    assert torch.equal(o["y"][0][512:512 + M * D].view(M, D), y)
    for name, got in (("dx", d["dx"]), ("dw_down", d["dw_down"]), ("db_gate", d["db_gate"])):
        assert torch.equal(o[name][0][512:512 + got.numel()].view(got.shape), got), name
