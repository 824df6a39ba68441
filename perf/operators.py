"""The cross-attention layer's operators as a user's program calls them, and their plain forms.

Three operators, each forward and as a training pass (forward and backward):

* ``xattn``: attention of query windows to an encoder's states (the frames of a support set) of another length;
* ``ffn``: the gated feed-forward block, both projections, activation, product and the projection back;
* ``norm``: the norms behind and before a block with its gate, residual scale and the residual sum.

``own`` False: elementary torch operations in 32 bits, rounded once at the end. ``own`` True: the calls of isbfsar_amd.blocks.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
LAYER_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def listed():
    def xattn(name, **c):
        return {"name": name, "op": "xattn", **c}

    def ffn(name, **c):
        return {"name": name, "op": "ffn", **c}

    def norm(name, **c):
        return {"name": name, "op": "norm", **c}

    return [
        # a streaming tick: the newest frame of one camera against the frames of a 60-class support set (60 windows of 30 frames)
        xattn("xattn tick", train=False, type="fp16", B=1, Bk=1, Lq=1, Lk=1800, Hq=4, Hk=4, D=64, mask="none"),
        # a serving step: 16 streams, one token each, against their own long states of ragged length; grouped heads
        xattn("xattn token long", train=False, type="bf16", B=16, Bk=16, Lq=1, Lk=16384, Hq=32, Hk=8, D=128, mask="len"),
        # a batch of 30-frame windows against ONE support set that all of them share
        xattn("xattn windows shared", train=False, type="fp16", B=256, Bk=1, Lq=30, Lk=1800, Hq=2, Hk=2, D=128, mask="holes"),
        # long sequences against a longer encoder output with holes in its padding mask
        xattn("xattn long", train=False, type="bf16", B=4, Bk=4, Lq=2048, Lk=4099, Hq=16, Hk=4, D=128, mask="holes"),
        # a fine-tuning step: gradients of the support set's states are summed over the windows that share it
        xattn("xattn train shared", train=True, type="bf16", B=64, Bk=1, Lq=30, Lk=1800, Hq=2, Hk=2, D=128, mask="len"),
        # an ordinary training step, ragged encoder lengths
        xattn("xattn train", train=True, type="fp16", B=8, Bk=8, Lq=777, Lk=1031, Hq=8, Hk=4, D=64, mask="len"),
        # a streaming tick through the block: one token, bound by the weights
        ffn("ffn token", train=False, type="bf16", M=1, D=1280, F=5120, act="silu", bias=False),
        # one 30-frame window at the embedding's width
        ffn("ffn window", train=False, type="fp16", M=30, D=256, F=1024, act="gelu", bias=True),
        # a batch of 256 windows
        ffn("ffn batch", train=False, type="bf16", M=7680, D=1280, F=5120, act="silu", bias=False),
        # a training step with ragged token counts
        ffn("ffn train", train=True, type="bf16", M=4111, D=640, F=2560, act="silu", bias=True),
        # a streaming tick: one row
        norm("norm tick", train=False, type="fp16", B=1, L=1, D=256, kind="layer", gate=True),
        # a training step at the trunk's width
        norm("norm train", train=True, type="bf16", B=64, L=511, D=1280, kind="rms", gate=True),
    ]


def _spread(rng, lo, hi, step=1):
    """a whole number in [lo, hi], spread over its logarithm; a multiple of step"""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(["xattn", "xattn", "ffn", "ffn", "norm"])
    train = rng.random() < 0.4
    kind = rng.choice(["bf16", "fp16"])
    if op == "xattn":
        while True:
            Bk = _spread(rng, 1, 16)
            nb = rng.choice([1, 1, 1, _spread(rng, 2, 64)])
            Hk = rng.choice([1, 2, 4, 8])
            c = {"op": op, "train": train, "type": kind, "B": Bk * nb, "Bk": Bk, "Lq": rng.choice([1, _spread(rng, 1, 2048)]),
                 "Lk": _spread(rng, 1, 4096 if train else 16384), "Hq": Hk * rng.choice([1, 1, 2, 4, 8]), "Hk": Hk,
                 "D": rng.choice([32, 64, 64, 72, 96, 128, 128]), "mask": rng.choice(["none", "len", "holes"])}
            w = work(c)
            if w["flops"] < 2.5e11 and w["bytes"] < 1.0e9 and c["B"] * c["Lq"] * c["Hq"] * c["Lk"] < 5.0e8:
                return c
    if op == "ffn":
        while True:
            c = {"op": op, "train": train, "type": kind, "M": _spread(rng, 1, 8192), "D": _spread(rng, 64, 2048, 8),
                 "F": _spread(rng, 128, 8192, 8), "act": rng.choice(["silu", "gelu", "relu", "sigmoid"]), "bias": rng.random() < 0.5}
            if work(c)["flops"] < 3.0e11:
                return c
    while True:
        c = {"op": op, "train": train, "type": rng.choice([kind, "f32"]), "B": _spread(rng, 1, 64), "L": _spread(rng, 1, 4096),
             "D": _spread(rng, 64, 8192), "kind": rng.choice(["layer", "rms"]), "gate": rng.random() < 0.6}
        if work(c)["bytes"] < 5.0e8:
            return c


def work(case):
    """bytes with each input read and each output written once, and the operations of one pass"""
    e = 4 if case["type"] == "f32" else 2
    train = case["train"]
    if case["op"] == "xattn":
        rows = case["B"] * case["Lq"] * case["Hq"]
        q, kv = rows * case["D"] * e, 2 * case["Bk"] * case["Lk"] * case["Hk"] * case["D"] * e
        share = {"none": 1.0, "len": 0.75, "holes": 0.75}[case["mask"]]         # of the states that a row attends to, on average
        flops = (14 if train else 4) * rows * case["Lk"] * case["D"] * share
        # forward: q, k, v -> out, lse; training: and dout -> dq, dk, dv
        return {"bytes": 2 * q + 4 * rows + kv * share + (2 * q + kv if train else 0), "flops": flops}
    if case["op"] == "ffn":
        m, d, f = case["M"], case["D"], case["F"]
        b = (2 * f + d) if case["bias"] else 0
        return {"bytes": e * ((4 if train else 2) * m * d + (2 if train else 1) * (3 * d * f + b)), "flops": (18 if train else 6) * m * d * f}
    n = case["B"] * case["L"] * case["D"]
    g = case["B"] * case["D"] * e if case["gate"] else 0
    # forward: x, y -> r, z; training: and dr, dz -> dx, dy
    return {"bytes": (8 if train else 4) * n * e + (2 if train else 1) * (g + 20 * case["D"]), "flops": (60 if train else 20) * n}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, type=t):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, std, generator=g).to(type)

    s = {"case": dict(case)}
    if case["op"] == "xattn":
        B, Bk, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Bk", "Lq", "Lk", "Hq", "Hk", "D"))
        s["q"] = normal(B, Lq, Hq, D)
        s["k"] = normal(Bk, Lk, Hk, D)
        s["v"] = normal(Bk, Lk, Hk, D)
        if case["mask"] in ("len", "holes"):
            # ragged lengths, the longest one full
            share = 0.5 + 0.5 * torch.rand(Bk, generator=g, device="cuda")
            lens = (share * Lk).to(torch.int32).clamp(0, Lk)
            if Bk > 1:
                lens[0] = Lk
            s["kv_len"] = lens
        if case["mask"] == "holes":
            s["key_mask"] = torch.rand(Bk, Lk, generator=g, device="cuda") < 0.9
        if case["train"]:
            s["dout"] = normal(B, Lq, Hq, D)
    elif case["op"] == "ffn":
        M, D, F = case["M"], case["D"], case["F"]
        s["x"] = normal(M, D)
        s["w_gate"] = normal(F, D, std=1 / math.sqrt(D))
        s["w_up"] = normal(F, D, std=1 / math.sqrt(D))
        s["w_down"] = normal(D, F, std=1 / math.sqrt(F))
        if case["bias"]:
            s["b_gate"], s["b_up"], s["b_down"] = normal(F, std=0.1), normal(F, std=0.1), normal(D, std=0.1)
        if case["train"]:
            s["dy"] = normal(M, D)
    else:
        B, L, D = case["B"], case["L"], case["D"]
        s["x"] = normal(B, L, D, std=2.0)
        s["y"] = normal(B, L, D)
        if case["gate"]:
            s["gate"] = normal(B, D, std=0.5)
        s["scale"] = 0.3 + normal(D, std=0.1, type=torch.float32)
        for n in ("post", "pre"):
            s[n + "_weight"] = 1.0 + normal(D, std=0.1, type=torch.float32)
            s[n + "_bias"] = normal(D, std=0.1, type=torch.float32) if case["kind"] == "layer" else None
        if case["train"]:
            s["dr"], s["dz"] = normal(B, L, D), normal(B, L, D)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "xattn":
        return _own_xattn(state) if own else _plain_xattn(state)
    if op == "ffn":
        return _own_ffn(state) if own else _plain_ffn(state)
    return _own_norm(state) if own else _plain_norm(state)


def _own_xattn(s):
    from isbfsar_amd.blocks import cross_attention, cross_attention_backward
    mask = {"kv_len": s.get("kv_len"), "key_mask": s.get("key_mask")}
    out, lse = cross_attention(s["q"], s["k"], s["v"], **mask)
    if not s["case"]["train"]:
        return {"out": out, "lse": lse}
    dq, dk, dv = cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **mask)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_ffn(s):
    from isbfsar_amd.blocks import gated_ffn, gated_ffn_backward
    w = [s["w_gate"], s["w_up"], s["w_down"]]
    b = [s.get("b_gate"), s.get("b_up"), s.get("b_down")]
    act = s["case"]["act"]
    if not s["case"]["train"]:
        return {"y": gated_ffn(s["x"], *w, *b, activation=act)}
    y, saved = gated_ffn(s["x"], *w, *b, activation=act, save=True)
    d = gated_ffn_backward(s["dy"], s["x"], *w, saved, bias=b[0] is not None, activation=act)
    return {"y": y, **d}


def _own_norm(s):
    from isbfsar_amd.blocks import block_norm, block_norm_backward
    kind = s["case"]["kind"]
    a = {"gate": s.get("gate"), "scale": s["scale"], "post": kind, "post_weight": s["post_weight"], "post_bias": s["post_bias"],
         "pre": kind, "pre_weight": s["pre_weight"], "pre_bias": s["pre_bias"], "eps": LAYER_EPS}
    if not s["case"]["train"]:
        r, z = block_norm(s["x"], s["y"], **a)
        return {"r": r, "z": z}
    r, z, stats = block_norm(s["x"], s["y"], save=True, **a)
    return {"r": r, "z": z, **block_norm_backward(s["dr"], s["dz"], s["x"], s["y"], stats, **a)}


def _valid(s):
    """[Bk, Lk] truth values: the states that rows attend to, or None for all of them"""
    v = None
    if s.get("kv_len") is not None:
        v = torch.arange(s["case"]["Lk"], device="cuda")[None, :] < s["kv_len"][:, None]
    if s.get("key_mask") is not None:
        v = s["key_mask"] if v is None else v & s["key_mask"]
    return v


def _plain_xattn(s):
    B, Bk, Lq, Lk, Hq, Hk, D = (s["case"][k] for k in ("B", "Bk", "Lq", "Lk", "Hq", "Hk", "D"))
    nb, G, scale, t = B // Bk, Hq // Hk, 1.0 / math.sqrt(D), s["q"].dtype

    def rows(x):        # [B, Lq, Hq, D] -> [Bk, Hk, nb Lq G, D]: every row that reads the same states
        return x.float().view(Bk, nb, Lq, Hk, G, -1).permute(0, 3, 1, 2, 4, 5).reshape(Bk, Hk, nb * Lq * G, -1)

    def back(x):
        return x.view(Bk, Hk, nb, Lq, G, -1).permute(0, 2, 3, 1, 4, 5).reshape(B, Lq, Hq, -1)

    def states(x, valid):
        x = x.float().permute(0, 2, 1, 3).contiguous()
        return x if valid is None else torch.where(valid[:, None, :, None], x, 0.0)

    valid = _valid(s)
    q, k, v = rows(s["q"]), states(s["k"], valid), states(s["v"], valid)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if valid is not None:
        p.masked_fill_(~valid[:, None, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    at = torch.where(top == -math.inf, 0.0, top)
    p.sub_(at).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p, v)
    r = {"out": back(out).to(t), "lse": back(at + torch.log(total)).squeeze(-1).transpose(1, 2).contiguous()}
    if s["case"]["train"]:
        do = rows(s["dout"])
        dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
        ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        r["dq"] = back(torch.matmul(ds, k)).to(t)
        r["dk"] = torch.matmul(ds.transpose(-1, -2).contiguous(), q).permute(0, 2, 1, 3).to(t).contiguous()
        r["dv"] = dv.permute(0, 2, 1, 3).to(t).contiguous()
    return r


def _plain_act(name, g):
    """act(g) and its derivative"""
    if name == "relu":
        return g.clamp(min=0.0), (g > 0).float()
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = torch.sigmoid(g)
    if name == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _plain_ffn(s):
    t = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    if s["case"]["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    a, da = _plain_act(s["case"]["act"], g)
    h = a * u
    y = torch.matmul(h, wd.t())
    if s["case"]["bias"]:
        y = y + s["b_down"].float()
    r = {"y": y.to(t)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        dh = torch.matmul(dy, wd)
        dg, du = dh * u * da, dh * a
        r["dx"] = (torch.matmul(dg, wg) + torch.matmul(du, wu)).to(t)
        r["dw_gate"], r["dw_up"] = torch.matmul(dg.t(), x).to(t), torch.matmul(du.t(), x).to(t)
        r["dw_down"] = torch.matmul(dy.t(), h).to(t)
        if s["case"]["bias"]:
            r["db_gate"], r["db_up"], r["db_down"] = dg.sum(0).to(t), du.sum(0).to(t), dy.sum(0).to(t)
    return r


def _plain_stats(kind, x):
    """(x - mean) / sqrt(var + eps) and 1 / sqrt(var + eps); rms: no mean"""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + LAYER_EPS)
    return x * inv, inv


def _plain_back(kind, d, xh, inv):
    """the gradient through the normalisation"""
    c = d - xh * (d * xh).mean(-1, keepdim=True)
    if kind == "layer":
        c = c - d.mean(-1, keepdim=True)
    return c * inv


def _plain_norm(s):
    kind, t = s["case"]["kind"], s["x"].dtype
    x, y = s["x"].float(), s["y"].float()
    factor = s["scale"] if s.get("gate") is None else s["scale"] * s["gate"].float()[:, None, :]
    yh, yi = _plain_stats(kind, y)
    n = yh * s["post_weight"]
    if kind == "layer":
        n = n + s["post_bias"]
    r = x + factor * n
    rh, ri = _plain_stats(kind, r)
    z = rh * s["pre_weight"]
    if kind == "layer":
        z = z + s["pre_bias"]
    got = {"r": r.to(t), "z": z.to(t)}
    if s["case"]["train"]:
        dz = s["dz"].float()
        d = s["dr"].float() + _plain_back(kind, dz * s["pre_weight"], rh, ri)
        dn = d * factor
        got["dx"] = d.to(t)
        got["dy"] = _plain_back(kind, dn * s["post_weight"], yh, yi).to(t)
        got["dpost_weight"], got["dpre_weight"] = (dn * yh).sum((0, 1)), (dz * rh).sum((0, 1))
        if kind == "layer":
            got["dpost_bias"], got["dpre_bias"] = dn.sum((0, 1)), dz.sum((0, 1))
        by = d * n
        if s.get("gate") is not None:
            got["dgate"] = (by.sum(1) * s["scale"]).to(t)
            by = by * s["gate"].float()[:, None, :]
        got["dscale"] = by.sum((0, 1))
    return got


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """the definitions in 64 bits; gradients by differentiating them"""
    s = prepare(case, seed)
    x = {k: v.double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    grad = case["train"]
    with torch.set_grad_enabled(grad):
        if case["op"] == "xattn":
            return _exact_xattn(case, s, x)
        for k in x:
            x[k].requires_grad_(grad)
        if case["op"] == "ffn":
            lin = torch.nn.functional.linear
            g, u = lin(x["x"], x["w_gate"], x.get("b_gate")), lin(x["x"], x["w_up"], x.get("b_up"))
            a = {"silu": lambda v: v / (1 + torch.exp(-v)), "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2)),
                 "relu": torch.relu, "sigmoid": lambda v: 1 / (1 + torch.exp(-v))}[case["act"]](g)
            y = lin(a * u, x["w_down"], x.get("b_down"))
            r = {"y": y}
            if grad:
                names = [n for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down") if n in x]
                r.update(zip(["d" + n for n in names], torch.autograd.grad(y, [x[n] for n in names], x["dy"])))
            return r

        def norm(v, w, b):
            if case["kind"] == "layer":
                return (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + LAYER_EPS) * w + b
            return v / torch.sqrt(v.square().mean(-1, keepdim=True) + LAYER_EPS) * w

        n = norm(x["y"], x["post_weight"], x.get("post_bias")) * x["scale"]
        r = x["x"] + (n * x["gate"].unsqueeze(1) if "gate" in x else n)
        z = norm(r, x["pre_weight"], x.get("pre_bias"))
        got = {"r": r, "z": z}
        if grad:
            names = [n for n in ("x", "y", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias") if n in x]
            d = torch.autograd.grad([r, z], [x[n] for n in names], [x["dr"], x["dz"]])
            got.update(zip(["d" + n for n in names], d))
        return got


def _exact_xattn(case, s, x):
    B, Bk, Hk, D = case["B"], case["Bk"], case["Hk"], case["D"]
    nb, G = B // Bk, case["Hq"] // Hk
    valid = _valid(s)
    got = {k: torch.zeros_like(x[k[1:]]) for k in ("dq", "dk", "dv")} if case["train"] else {}
    got["out"] = torch.zeros_like(x["q"])
    got["lse"] = torch.full((B, case["Hq"], case["Lq"]), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(Bk):
        at = torch.arange(case["Lk"], device="cuda") if valid is None else valid[b].nonzero().squeeze(1)
        if at.numel() == 0:
            continue
        for h in range(Hk):
            bs, hs = slice(b * nb, (b + 1) * nb), slice(h * G, (h + 1) * G)
            q = x["q"][bs, :, hs].detach().reshape(-1, D).requires_grad_(case["train"])
            k, v = (x[n][b, :, h][at].detach().requires_grad_(case["train"]) for n in ("k", "v"))
            logits = q @ k.T / math.sqrt(D)
            lse = torch.logsumexp(logits, -1)
            out = torch.exp(logits - lse[:, None]) @ v
            shape = x["q"][bs, :, hs].shape
            got["out"][bs, :, hs] = out.detach().view(shape)
            got["lse"][bs, hs] = lse.detach().view(shape[:3]).transpose(1, 2)
            if case["train"]:
                d = torch.autograd.grad(out, [q, k, v], x["dout"][bs, :, hs].reshape(-1, D))
                got["dq"][bs, :, hs] = d[0].view(shape)
                got["dk"][b, at, h], got["dv"][b, at, h] = d[1], d[2]
    return got
