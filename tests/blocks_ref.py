"""Plain 64-bit implementations of the layer operators (isbfsar_amd/blocks.py) with the bounds on the kernels' rounding that the GPU tests
hold them to. Every function returns {name: (value, bound)}.

Bounds. u = half a step of the 16-bit type, relative to the value (bf16 2^-8, fp16 2^-11): one per rounding. e = 2^-24, f32's. A sum of n
f32 terms in any order is off by at most n e times the sum of their magnitudes; what enters it off carries over. v_exp_f32, v_log_f32 and
v_rcp_f32 are good to one step (2 e)."""
import math

import torch

E = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def valid_states(Bk, Lk, kv_len, key_mask, device):
    v = torch.ones(Bk, Lk, dtype=torch.bool, device=device)
    if kv_len is not None:
        v &= torch.arange(Lk, device=device)[None, :] < kv_len[:, None]
    if key_mask is not None:
        v &= key_mask
    return v


def xattn(q, k, v, kv_len=None, key_mask=None, scale=None, dout=None):
    """out, lse (and dq, dk, dv with dout). The kernels round P (to the type of v) and dS once each, results once more."""
    t, dev = q.dtype, q.device
    B, Lq, Hq, D = q.shape
    Bk, Lk, Hk, _ = k.shape
    nb, G = B // Bk, Hq // Hk
    u = half_step(t)
    tiny = 2.0 ** -24 if t == torch.float16 else 0.0            # fp16 weights below 2^-14 are rounded to steps of 2^-24
    scale = 1 / math.sqrt(D) if scale is None else scale
    ok = valid_states(Bk, Lk, kv_len, key_mask, dev)

    def rows(x):
        return x.double().view(Bk, nb, Lq, Hk, G, D).permute(0, 3, 1, 2, 4, 5).reshape(Bk, Hk, nb * Lq * G, D)

    def back(x):
        return x.reshape(Bk, Hk, nb, Lq, G, -1).permute(0, 2, 3, 1, 4, 5).reshape(B, Lq, Hq, -1)

    def states(x):
        return torch.where(ok[:, None, :, None], x.double().permute(0, 2, 1, 3), 0.0)

    T = lambda x: x.transpose(-1, -2)   # noqa: E731
    Q, K, V = rows(q), states(k), states(v)
    s = (Q @ T(K)) * scale
    s = s.masked_fill(~ok[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    P = torch.where(ok[:, None, None, :], torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)), 0.0)
    out = P @ V
    # scores: D products in f32 and their scaling; twice that (numerator and sum) moves a weight, exp2's argument and value 8 e more
    es = ((Q.abs() @ T(K.abs())) * scale * (D + 4) * E + torch.where(s == -math.inf, 0.0, s).abs() * 4 * E).amax(-1, keepdim=True)
    ep = 2 * es + 8 * E + (Lk + 64) * E
    A = P @ V.abs()
    eo = u * out.abs() + A * (u + ep) * (1 + u) + tiny * V.abs().sum(-2, keepdim=True)
    el = es + (Lk + 64) * E + 4 * E * (lse.abs().clamp(max=1e30) + 8)
    r = {"out": (back(out), back(eo)), "lse": (back(lse).squeeze(-1).transpose(1, 2), back(el).squeeze(-1).transpose(1, 2))}
    def stored(r):                   # fp16 results below 2^-14 are rounded to steps of 2^-24: half of one, 2^-25, besides u
        return {n: (x, y + 2.0 ** -25) if t == torch.float16 and n != "lse" else (x, y) for n, (x, y) in r.items()}
    if dout is None:
        return stored(r)
    dO = rows(dout)
    dV = T(P) @ dO
    n = nb * Lq * G
    edv = u * dV.abs() + (T(P * (u + ep)) @ dO.abs()) + T(P) @ dO.abs() * (n + 64) * E + tiny * dO.abs().sum(-2, keepdim=True) * 2.0 ** -12
    dP = dO @ T(V)
    delta = (dO * out).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    edelta = (dO.abs() * eo).sum(-1, keepdim=True) + D * E * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    edS = dS.abs() * (u + ep + 4 * E) + P * (edelta + (D + 4) * E * (dO.abs() @ T(V.abs()))) * (1 + u)
    if t == torch.float16:          # dS is scaled so that its largest value is at least 2^10: steps of 2^-24 below 2^-14
        edS = edS + torch.where(ok[:, None, None, :], dS.abs().amax((-1, -2), keepdim=True) * 2.0 ** -34, 0.0)
    dQ, dK = (dS @ K) * scale, (T(dS) @ Q) * scale
    edq = u * dQ.abs() + scale * (edS @ K.abs() + (Lk + 64) * E * (dS.abs() @ K.abs()))
    edk = u * dK.abs() + scale * (T(edS) @ Q.abs() + (n + 64) * E * (T(dS.abs()) @ Q.abs()))
    r["dq"] = (back(dQ), back(edq))
    r["dk"], r["dv"] = ((x.permute(0, 2, 1, 3), y.permute(0, 2, 1, 3)) for x, y in ((dK, edk), (dV, edv)))
    return stored(r)


def act(name, g):
    """act(g), act'(g); both and the slope of both are bounded by 1.2 (max(1, |g|) times that for the first)"""
    if name == "relu":
        return g.clamp(min=0), (g > 0).double()
    if name == "gelu":
        phi = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-g))
    return (s, s * (1 - s)) if name == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def ffn(x, wg, wu, wd, bg=None, bu=None, bd=None, activation="silu", dy=None):
    """y (and gradients with dy): h, dG and dU are rounded once where they enter a product, results once more"""
    t, u = x.dtype, half_step(x.dtype)
    M, D = x.shape
    F = wg.shape[0]
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0            # fp16 below 2^-14: steps of 2^-24
    X, G, U, W = (a.double() for a in (x, wg, wu, wd))
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    bg, bu, bd = (zero if b is None else b.double() for b in (bg, bu, bd))
    g, v = X @ G.T + bg, X @ U.T + bu
    eg, ev = ((X.abs() @ w.abs().T + b.abs()) * (D + 4) * E for w, b in ((G, bg), (U, bu)))
    a, da = act(activation, g)
    ea = 1.2 * eg + 16 * E * (1 + g.abs())                       # the slope's bound and the functions' own error
    eda = eg + 16 * E * (1 + g.abs())
    if activation == "relu":                                     # a step at 0
        eda = torch.where(g.abs() <= eg, 1.0, 0.0)
    h = a * v
    eh = h.abs() * (u + 2 * E) + (ea * v.abs() + (a.abs() + ea) * ev) * (1 + u) + tiny
    y = h @ W.T + bd
    r = {"y": (y, u * y.abs() + (eh @ W.abs().T + (F + 8) * E * (h.abs() @ W.abs().T + bd.abs())) * (1 + u) + tiny)}
    if dy is None:
        return r
    Y = dy.double()
    dh = Y @ W
    edh = (Y.abs() @ W.abs()) * (D + 4) * E
    dg, dv = dh * v * da, dh * a
    edg = dg.abs() * (u + 4 * E) + (edh * v.abs() * da.abs() + dh.abs() * (ev * da.abs() + (v.abs() + ev) * eda)) * (1 + u) + tiny
    edv = dv.abs() * (u + 4 * E) + (edh * a.abs() + (dh.abs() + edh) * ea) * (1 + u) + tiny

    def result(val, err):
        return val, u * val.abs() + err * (1 + u) + tiny

    r["dx"] = result(dg @ G + dv @ U, edg @ G.abs() + edv @ U.abs() + (2 * F + 8) * E * (dg.abs() @ G.abs() + dv.abs() @ U.abs()))
    n = M + 8
    r["dw_gate"] = result(dg.T @ X, edg.T @ X.abs() + n * E * (dg.abs().T @ X.abs()))
    r["dw_up"] = result(dv.T @ X, edv.T @ X.abs() + n * E * (dv.abs().T @ X.abs()))
    r["dw_down"] = result(Y.T @ h, Y.abs().T @ eh + n * E * (Y.abs().T @ h.abs()))
    for name, d, ed in (("db_gate", dg, edg), ("db_up", dv, edv), ("db_down", Y, torch.zeros_like(Y))):
        r[name] = result(d.sum(0), ed.sum(0) + n * E * d.abs().sum(0))
    return r


def norm(x, y=None, gate=None, scale=None, post=None, post_weight=None, post_bias=None, pre=None, pre_weight=None, pre_bias=None, eps=1e-5,
         dr=None, dz=None):
    """r, z (and gradients with dr / dz). A row's sums: at most 8 terms per lane, 6 steps over the lanes, 16 waves: S = 32 e relative to
    the sum of magnitudes."""
    t = x.dtype
    u = E if t == torch.float32 else half_step(t)
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    S = 32 * E
    B, L, D = x.shape
    one = torch.ones(D, dtype=torch.float64, device=x.device)
    nul = torch.zeros(D, dtype=torch.float64, device=x.device)
    W = lambda w, d: d if w is None else w.double()      # noqa: E731
    qw, qb, pw, pb, sc = W(post_weight, one), W(post_bias, nul), W(pre_weight, one), W(pre_bias, nul), W(scale, one)
    f = sc if gate is None else sc * gate.double()[:, None, :]
    mean = lambda v: v.mean(-1, keepdim=True)            # noqa: E731

    def norm_of(kind, v, ev):
        """normalised rows, 1 / sd, and the bound on the normalised rows, given the rows' own bound"""
        if kind is None:
            return v, one.new_ones(()), ev
        c, ec = v, ev + 2 * E * v.abs()
        if kind == "layer":
            c = v - mean(v)
            ec = ec + mean(ev) + S * mean(v.abs())
        var = mean(c * c)
        inv = 1 / torch.sqrt(var + eps)
        rel = (mean(2 * c.abs() * ec) + S * var) / (var + eps) / 2 + 4 * E           # of inv
        return c * inv, inv, (ec + c.abs() * rel + 2 * E * c.abs()) * inv

    X = x.double()
    got, r, er = {}, X, torch.zeros_like(X)
    if y is not None:
        Y = y.double()
        yh, iy, eyh = norm_of(post, Y, torch.zeros_like(Y))
        n = yh * qw + qb
        en = eyh * qw.abs() + 2 * E * (yh.abs() * qw.abs() + qb.abs())
        r = X + f * n
        er = f.abs() * en + 3 * E * (X.abs() + 2 * (f * n).abs())
        got["r"] = (r, er * (1 + u) + u * r.abs() + tiny)
    rh, ir, erh = norm_of(pre, r, er)
    if pre is not None:
        z = rh * pw + pb
        got["z"] = (z, (erh * pw.abs() + 2 * E * (rh.abs() * pw.abs() + pb.abs())) * (1 + u) + u * z.abs() + tiny)
    if dr is None and dz is None:
        return got

    def back(kind, d, ed, h, eh, inv):
        """through the normalisation: value and bound"""
        if kind is None:
            return d, ed
        rel = 64 * E + 2 * mean(h.abs() * eh)                                         # of inv (above, with the row's own bound)
        m1 = mean(d * h)
        em1 = mean(ed * h.abs() + d.abs() * eh) + S * mean((d * h).abs())
        g, eg = d - h * m1, ed + eh * m1.abs() + h.abs() * em1
        if kind == "layer":
            g, eg = g - mean(d), eg + mean(ed) + S * mean(d.abs())
        return g * inv, (eg + 4 * E * (d.abs() + (h * m1).abs() + mean(d.abs())) + g.abs() * rel) * inv

    dR, edR = (torch.zeros_like(X) if dr is None else dr.double()), torch.zeros_like(X)
    rows = B * L + 64
    if pre is not None:
        dZ = dz.double()
        a = dZ * pw
        v, ev = back(pre, a, 2 * E * a.abs(), rh, erh, ir)
        dR, edR = dR + v, ev + 2 * E * (dR.abs() + v.abs())
        col = lambda v, ev: (v.sum((0, 1)), ev.sum((0, 1)) + rows * E * v.abs().sum((0, 1)))     # noqa: E731
        if pre_weight is not None:
            got["dpre_weight"] = col(dZ * rh, dZ.abs() * erh)
        if pre_bias is not None:
            got["dpre_bias"] = col(dZ, torch.zeros_like(dZ))
    got["dx"] = (dR, edR * (1 + u) + u * dR.abs() + tiny)
    if y is None:
        return got
    dN, edN = dR * f, edR * f.abs() + 2 * E * (dR * f).abs()
    b, eb = dN * qw, (edN + 2 * E * dN.abs()) * qw.abs()
    v, ev = back(post, b, eb, yh, eyh, iy)
    got["dy"] = (v, ev * (1 + u) + u * v.abs() + tiny)
    # column sums: rows in f32, then chunks and samples
    by = dR * n
    eby = edR * n.abs() + dR.abs() * en + 4 * E * (dR.abs() * (yh.abs() * qw.abs() + qb.abs()))
    add = rows * E

    def summed(v, ev, dims):
        return v.sum(dims), ev.sum(dims) + add * (v.abs() + (dR.abs() * (yh.abs() * qw.abs() + qb.abs()) if v is by else 0)).sum(dims)

    if gate is not None:
        s, es = summed(by, eby, 1)
        s, es = s * sc, es * sc.abs()
        got["dgate"] = (s, es * (1 + u) + u * s.abs() + tiny)
    gd = 1.0 if gate is None else gate.double()[:, None, :]
    if scale is not None:
        es = (eby * abs(gd)).sum((0, 1)) + 2 * add * (dR.abs() * (yh.abs() * qw.abs() + qb.abs()) * abs(gd)).sum((0, 1))
        got["dscale"] = ((by * gd).sum((0, 1)), es)
    if post_weight is not None:
        got["dpost_weight"] = summed(dN * yh, edN * yh.abs() + dN.abs() * eyh, (0, 1))
    if post_bias is not None:
        got["dpost_bias"] = summed(dN, edN, (0, 1))
    return got
