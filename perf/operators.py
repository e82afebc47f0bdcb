"""The operators of a transformer block, in plain form and as the framework's kernels: attention (with grouped heads, causal masks and
key lengths), the residual add with the norms before and after it, and the linear layer with bias, activation and residual.

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, through ``coin_amd.layers``."""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the prompt-learning step of the text encoder: 9 classes x 77 tokens, 8 heads of 64
        dict(name="attention text step", op="attention", type="bf16", b=9, lq=77, lk=77, hq=8, hkv=8, d=64, causal=True, ragged=False, grad=True),
        # the 81 prompt templates of one class in the fp32 parity mode
        dict(name="attention templates fp32", op="attention", type="f32", b=81, lq=77, lk=77, hq=8, hkv=8, d=64, causal=True, ragged=True, grad=True),
        # training on long sequences of an odd length, four query heads to a key head
        dict(name="attention long training", op="attention", type="bf16", b=2, lq=4001, lk=4001, hq=16, hkv=4, d=128, causal=True, ragged=False, grad=True),
        # one new token for each of 16 sequences over ragged caches
        dict(name="attention single token", op="attention", type="bf16", b=16, lq=1, lk=32768, hq=32, hkv=8, d=128, causal=True, ragged=True, grad=False),
        # between two halves of a text encoder block: add and LayerNorm of 9 x 77 rows
        dict(name="norm text step", op="norm", stream="bf16", branch="bf16", groups=9, rows=77, d=512, rms=False, y=True, post=False, gate="", pre=True, scale=1.0, grad=True),
        # a block with a norm on both sides and a gate for each sequence, on an fp32 stream
        dict(name="norm gated sandwich", op="norm", stream="f32", branch="bf16", groups=8, rows=4096, d=2048, rms=True, y=True, post=True, gate="groups", pre=True, scale=0.5, grad=True),
        # the first stage of the Swin student in fp32: many short rows, with a layer scale
        dict(name="norm swin stage fp32", op="norm", stream="f32", branch="f32", groups=2, rows=22533, d=96, rms=False, y=True, post=False, gate="layer", pre=True, scale=1.0, grad=True),
        # a few single tokens
        dict(name="norm single tokens", op="norm", stream="bf16", branch="bf16", groups=1, rows=4, d=4096, rms=True, y=True, post=True, gate="", pre=True, scale=1.0, grad=False),
        # the text encoder's MLP under prompt learning: frozen weights, the gradient of the input alone
        dict(name="linear text mlp", op="linear", type="bf16", m=693, k=512, n=2048, act="quick_gelu", bias=True, residual=False, grad="input"),
        # the Swin student's third stage in fp32, everything trained
        dict(name="linear swin mlp fp32", op="linear", type="f32", m=5092, k=384, n=1536, act="gelu", bias=True, residual=False, grad="all"),
        # a large layer in training, with the residual in its epilogue
        dict(name="linear large training", op="linear", type="bf16", m=16381, k=2048, n=8192, act="gelu", bias=True, residual=True, grad="all"),
        # single tokens: the weight is read for four rows
        dict(name="linear single tokens", op="linear", type="bf16", m=4, k=8192, n=2048, act="none", bias=True, residual=True, grad=""),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "norm", "linear"])
    if op == "attention":
        kind = rng.choice(["f32", "bf16", "bf16"])
        d = rng.choice([32, 64, 128, 8 * rng.randint(1, 16)])
        hkv = rng.choice([1, 2, 3, 4, 8])
        hq = hkv * rng.choice([1, 1, 2, 4])
        if rng.random() < 0.3:      # new tokens over a cache
            lq, lk, grad = rng.choice([1, 1, rng.randint(2, 16)]), _log(rng, 64, 32768), False
        else:
            lq, grad = _log(rng, 1, 4096), rng.random() < 0.75
            lk = lq if rng.random() < 0.7 else _log(rng, 1, 4096)
        most = 10 ** 8 if kind == "bf16" else 10 ** 7   # pairs of query and key over all heads
        b = max(1, min(_log(rng, 1, 64), most // (hq * lq * lk), 5 * 10 ** 8 // (lk * hkv * d)))
        return dict(op=op, type=kind, b=b, lq=lq, lk=lk, hq=hq, hkv=hkv, d=d, causal=rng.random() < 0.6, ragged=rng.random() < 0.5, grad=grad)
    if op == "norm":
        stream, branch = rng.choice([("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
        d = rng.choice([_log(rng, 16, 8192), 8 * _log(rng, 4, 1024), 8 * _log(rng, 4, 1024)])
        groups = _log(rng, 1, 16)
        rows = max(1, min(_log(rng, 1, 16384), 6 * 10 ** 7 // (groups * d)))
        y = rng.random() < 0.85
        post = y and rng.random() < 0.5
        gate = rng.choice(["", "layer", "groups"]) if y else ""
        return dict(op=op, stream=stream, branch=branch, groups=groups, rows=rows, d=d, rms=rng.random() < 0.5, y=y, post=post, gate=gate,
                    pre=(not y) or rng.random() < 0.85, scale=rng.choice([1.0, 1.0, 0.5, 1.25]), grad=rng.random() < 0.75)
    kind = rng.choice(["f32", "bf16", "bf16"])
    step = rng.choice([1, 8, 8, 32])
    m, k, n = _log(rng, 1, 16384), step * _log(rng, max(1, 16 // step), 8192 // step), step * _log(rng, max(1, 16 // step), 8192 // step)
    most = 2.5 * 10 ** 11 if kind == "bf16" else 2 * 10 ** 10
    m = max(1, min(m, int(most / (k * n))))
    return dict(op=op, type=kind, m=m, k=k, n=n, act=rng.choice(["none", "relu", "gelu", "quick_gelu", "silu"]), bias=rng.random() < 0.75,
                residual=rng.random() < 0.5, grad=rng.choice(["", "input", "all", "all"]))


# -------------------------------------------------------------------------------------------------------------------------- the inputs
def _normal(g, shape, dtype, std=1.0, grad=False):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype).requires_grad_(grad)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    c = dict(case)
    s = {"case": c}
    if c["op"] == "attention":
        t, grad = TYPES[c["type"]], c["grad"]
        s["q"] = _normal(g, (c["b"], c["lq"], c["hq"], c["d"]), t, 1.0, grad)
        s["k"] = _normal(g, (c["b"], c["lk"], c["hkv"], c["d"]), t, 1.0, grad)
        s["v"] = _normal(g, (c["b"], c["lk"], c["hkv"], c["d"]), t, 1.0, grad)
        s["scale"] = c["d"] ** -0.5
        # ragged: sequences of every length up to the buffer's, the first as long as the buffer
        n = torch.randint(0, c["lk"] + 1, (c["b"],), generator=g, device=DEV, dtype=torch.int32)
        n[0] = c["lk"]
        s["lengths"] = n if c["ragged"] else None
        s["dout"] = _normal(g, (c["b"], c["lq"], c["hq"], c["d"]), t) if grad else None
    elif c["op"] == "norm":
        ts, tb, d, grad = TYPES[c["stream"]], TYPES[c["branch"]], c["d"], c["grad"]
        shape = (c["groups"], c["rows"], d)
        kind = torch.nn.RMSNorm if c["rms"] else torch.nn.LayerNorm

        def norm():
            m = kind(d, eps=1e-5, device=DEV)
            with torch.no_grad():
                for name, p in m.named_parameters():
                    p.copy_(torch.randn(d, generator=g, device=DEV) * 0.2 + (1.0 if name == "weight" else 0.0))
            return m.requires_grad_(grad)

        s["x"] = _normal(g, shape, ts, 2.0, grad)
        s["y"] = _normal(g, shape, tb, 1.0, grad) if c["y"] else None
        s["post"] = norm() if c["post"] else None
        s["pre"] = norm() if c["pre"] else None
        # a gate of each sequence comes from the network, in the branch's type; a layer scale is a parameter, in fp32
        s["gate"] = {"": lambda: None, "layer": lambda: _normal(g, (d,), torch.float32, 0.3, grad),
                     "groups": lambda: _normal(g, (c["groups"], 1, d), tb, 0.5, grad)}[c["gate"]]()
        s["dr"] = _normal(g, shape, ts) if grad and c["y"] else None
        s["dh"] = _normal(g, shape, tb) if grad and c["pre"] else None
    else:
        t, every = TYPES[c["type"]], c["grad"] == "all"
        s["x"] = _normal(g, (c["m"], c["k"]), t, 1.0, c["grad"] != "")
        s["w"] = _normal(g, (c["n"], c["k"]), t, c["k"] ** -0.5, every)
        s["b"] = _normal(g, (c["n"],), t, 0.5, every) if c["bias"] else None
        s["res"] = _normal(g, (c["m"], c["n"]), t, 1.0, c["grad"] != "") if c["residual"] else None
        s["dy"] = _normal(g, (c["m"], c["n"]), t) if c["grad"] else None
    return s


# --------------------------------------------------------------------------------------------------------------------------- the passes
def run(state):
    if own:
        return {"attention": _own_attention, "norm": _own_norm, "linear": _own_linear}[state["case"]["op"]](state)
    with torch.no_grad():
        return {"attention": _attention, "norm": _norm, "linear": _linear}[state["case"]["op"]](state)


def _grads(named, outs, given):
    """The gradients of the leaves in `named` from those of the outputs, under their names."""
    named = {k: v for k, v in named.items() if v is not None and v.requires_grad}
    return dict(zip(named, torch.autograd.grad(outs, list(named.values()), given)))


def _own_attention(s):
    from coin_amd import layers as L

    c = s["case"]
    out = L.attention(s["q"], s["k"], s["v"], causal=c["causal"], scale=s["scale"], key_lengths=s["lengths"])
    return {"out": out, **(_grads({"dq": s["q"], "dk": s["k"], "dv": s["v"]}, [out], [s["dout"]]) if c["grad"] else {})}


def _own_norm(s):
    from coin_amd import layers as L

    c = s["case"]
    r, h = L.residual_norm(s["x"], s["y"], post_norm=s["post"], gate=s["gate"], scale=c["scale"], pre_norm=s["pre"], branch_dtype=TYPES[c["branch"]])
    out = {**({"r": r} if c["y"] else {}), **({"h": h} if c["pre"] else {})}
    if c["grad"]:
        leaves = {"dx": s["x"], "dy": s["y"], "dgate": s["gate"]}
        for at in ("post", "pre"):
            if s[at] is not None:
                leaves.update({"d%s_%s" % (at, n): p for n, p in s[at].named_parameters()})
        out.update(_grads(leaves, list(out.values()), [s["d" + n] for n in out]))
    return out


def _own_linear(s):
    from coin_amd import layers as L

    c = s["case"]
    act = {"none": L.ACT_NONE, "relu": L.ACT_RELU, "gelu": L.ACT_GELU, "quick_gelu": L.ACT_QUICK_GELU, "silu": L.ACT_SILU}[c["act"]]
    y = L.fused_linear(s["x"], s["w"], s["b"], act=act, residual=s["res"])
    return {"y": y, **(_grads({"dx": s["x"], "dw": s["w"], "db": s["b"], "dres": s["res"]}, [y], [s["dy"]]) if c["grad"] else {})}


def _attention(s):
    c = s["case"]
    b, lq, lk, hq, hkv, d = (c[n] for n in ("b", "lq", "lk", "hq", "hkv", "d"))
    t, g = TYPES[c["type"]], hq // hkv
    # [b, hkv, g * lq, d] against [b, hkv, lk, d]: the query heads of one key head are rows of one product
    rows = lambda x: x.float().view(b, lq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * lq, d)  # noqa: E731
    keys = lambda x: x.float().permute(0, 2, 1, 3).contiguous()  # noqa: E731
    back = lambda x, n: x.view(b, hkv, n, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, hkv * n, d).to(t)  # noqa: E731
    j = torch.arange(lk, device=DEV)
    n = s["lengths"].long().view(b, 1, 1) if s["lengths"] is not None else torch.full((b, 1, 1), lk, device=DEV)
    keep = j.view(1, 1, lk) < n
    if c["causal"]:
        keep = keep & (j.view(1, 1, lk) <= torch.arange(lq, device=DEV).view(1, lq, 1) + n - lq)
    keep = keep.expand(b, lq, lk).unsqueeze(1).unsqueeze(1).expand(b, 1, g, lq, lk).reshape(b, 1, g * lq, lk)
    live = (j.view(1, 1, lk, 1) < n.view(b, 1, 1, 1))
    q, k, v = rows(s["q"]) * s["scale"], torch.where(live, keys(s["k"]), 0.0), torch.where(live, keys(s["v"]), 0.0)
    p = (q @ k.transpose(-1, -2)).masked_fill_(~keep, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = p @ v
    out = {"out": back(o, g)}
    if c["grad"]:
        do = rows(s["dout"])
        dv = p.transpose(-1, -2) @ do
        ds = do @ v.transpose(-1, -2)
        ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
        out["dq"] = back((ds @ k) * s["scale"], g)
        out["dk"] = (ds.transpose(-1, -2) @ q).permute(0, 2, 1, 3).to(t)
        out["dv"] = dv.permute(0, 2, 1, 3).to(t)
    return out


def _normed(u, m, rms):
    """-> the normalised rows, 1 / their deviation, and their affine image."""
    if not rms:
        u = u - u.mean(-1, keepdim=True)
    rstd = torch.rsqrt((u * u).mean(-1, keepdim=True) + m.eps)
    n = u * rstd
    return n, rstd, n * m.weight + (0.0 if rms else m.bias)


def _normed_back(g, n, rstd, m, rms):
    w = g * m.weight
    d = w - n * (w * n).mean(-1, keepdim=True)
    return rstd * (d if rms else d - w.mean(-1, keepdim=True))


def _norm(s):
    c = s["case"]
    ts, tb, rms = TYPES[c["stream"]], TYPES[c["branch"]], c["rms"]
    r, n, f, gate = s["x"].float(), None, None, None
    if c["y"]:
        f = s["y"].float()
        if c["post"]:
            n, rstd, f = _normed(f, s["post"], rms)
        gate = s["gate"].float() if s["gate"] is not None else None
        r = r + c["scale"] * (f * gate if gate is not None else f)
    out = {"r": r.to(ts)} if c["y"] else {}
    if c["pre"]:
        m, rstd_r, h = _normed(r, s["pre"], rms)
        out["h"] = h.to(tb)
    if not c["grad"]:
        return out
    e, params = (s["dr"].float() if c["y"] else 0.0), {}
    if c["pre"]:
        dh = s["dh"].float()
        params["dpre_weight"] = (dh * m).sum((0, 1))
        if not rms:
            params["dpre_bias"] = dh.sum((0, 1))
        e = e + _normed_back(dh, m, rstd_r, s["pre"], rms)
    out["dx"] = e.to(ts)
    if c["y"]:
        df = e * c["scale"]
        if gate is not None:
            dg = df * f
            out["dgate"] = dg.sum((0, 1)) if c["gate"] == "layer" else dg.sum(1, keepdim=True).to(tb)
            df = df * gate
        if c["post"]:
            params["dpost_weight"] = (df * n).sum((0, 1))
            if not rms:
                params["dpost_bias"] = df.sum((0, 1))
            df = _normed_back(df, n, rstd, s["post"], rms)
        out["dy"] = df.to(tb)
    return {**out, **params}


def _act(z, kind, want_slope):
    """The activation and its slope."""
    if kind == "none":
        return z, None
    if kind == "relu":
        return z.clamp_min(0.0), (z > 0).to(z.dtype) if want_slope else None
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 0.7071067811865476))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327 if want_slope else None
    a = 1.702 if kind == "quick_gelu" else 1.0
    sg = torch.sigmoid(a * z)
    return z * sg, sg * (1.0 + a * z * (1.0 - sg)) if want_slope else None


def _linear(s):
    c = s["case"]
    t = TYPES[c["type"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if c["bias"]:
        z = z + s["b"].float()
    y, slope = _act(z, c["act"], c["grad"] != "")
    if c["residual"]:
        y = y + s["res"].float()
    out = {"y": y.to(t)}
    if c["grad"]:
        dz = s["dy"].float()
        if slope is not None:
            dz = dz * slope
        out["dx"] = (dz @ w).to(t)
        if c["grad"] == "all":
            out["dw"] = (dz.t() @ x).to(t)
            if c["bias"]:
                out["db"] = dz.sum(0).to(t)
        if c["residual"]:
            out["dres"] = s["dy"]
    return out


# ----------------------------------------------------------------------------------------------------------------------------- its work
def _pairs(c):
    """Pairs of a query and a key of one head that the mask leaves; of ragged keys, half the buffer's on average."""
    n = c["lk"] * (0.5 + 0.5 / c["b"] if c["ragged"] else 1.0)
    whole = c["lq"] * n
    if c["causal"]:
        q = min(c["lq"], n)
        whole = q * n - q * (q - 1) / 2.0
    return c["b"] * whole


def work(case):
    c = case
    if c["op"] == "attention":
        e = 2 if c["type"] == "bf16" else 4
        n = c["lk"] * (0.5 + 0.5 / c["b"] if c["ragged"] else 1.0)
        qs, ks = c["b"] * c["lq"] * c["hq"] * c["d"] * e, c["b"] * n * c["hkv"] * c["d"] * e
        pairs = _pairs(c) * c["hq"] * c["d"]
        # forward: two products, q k v read and out written; backward: five (the scores again), out and its gradient read, three gradients written
        return {"bytes": 2 * qs + 2 * ks + (2 * qs + 2 * c["b"] * c["lk"] * c["hkv"] * c["d"] * e if c["grad"] else 0), "flops": (14 if c["grad"] else 4) * pairs}
    if c["op"] == "norm":
        es, eb = (2 if c[n] == "bf16" else 4 for n in ("stream", "branch"))
        n = c["groups"] * c["rows"] * c["d"]
        per = es + (es + eb if c["y"] else 0) + (eb if c["pre"] else 0)
        if c["grad"]:   # gradients in and out, of the same sizes
            per += (es + eb if c["y"] else 0) + (eb if c["pre"] else 0) + es
        return {"bytes": n * per, "flops": n * (30 if c["grad"] else 12)}
    e = 2 if c["type"] == "bf16" else 4
    m, k, n = c["m"], c["k"], c["n"]
    products = {"": 1, "input": 2, "all": 3}[c["grad"]]
    size = m * k + n * k + m * n * (2 if c["residual"] else 1)
    if c["grad"]:
        size += m * n + m * k + (n * k if c["grad"] == "all" else 0)
    return {"bytes": size * e, "flops": 2 * m * n * k * products}


# ----------------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, their gradients by differentiation of the definition."""
    s = prepare(case, seed)
    c = s["case"]
    up = lambda x: None if x is None else x.detach().double().requires_grad_(x.requires_grad)  # noqa: E731
    if c["op"] == "attention":
        if c["b"] * c["hq"] * c["lq"] * c["lk"] > 1.2e9:
            return None
        q, k, v = up(s["q"]), up(s["k"]), up(s["v"])
        outs = []
        for i in range(c["b"]):     # each sequence by itself, over the keys that it has
            n = int(s["lengths"][i]) if s["lengths"] is not None else c["lk"]
            qi = q[i].transpose(0, 1)
            ki, vi = (x[i, :n].transpose(0, 1).repeat_interleave(c["hq"] // c["hkv"], 0) for x in (k, v))
            sc = torch.matmul(qi, ki.transpose(1, 2)) * s["scale"]
            first = 0
            if c["causal"]:
                sc = sc + torch.full((c["lq"], n), float("-inf"), device=DEV, dtype=torch.float64).triu(n - c["lq"] + 1)
                first = max(0, c["lq"] - n)     # the rows before it have no key
            elif n == 0:
                first = c["lq"]
            o = torch.matmul(torch.softmax(sc[:, first:], -1), vi)
            outs.append(torch.nn.functional.pad(o, (0, 0, first, 0)).transpose(0, 1))
        out = torch.stack(outs)
        res = {"out": out}
        if c["grad"]:
            res.update(_grads({"dq": q, "dk": k, "dv": v}, [out], [s["dout"].double()]))
    elif c["op"] == "norm":
        x, y, gate = up(s["x"]), up(s["y"]), up(s["gate"])
        leaves = {"dx": x, "dy": y, "dgate": gate}
        par = {}
        for at in ("post", "pre"):
            if s[at] is not None:
                par[at] = {n: up(p) for n, p in s[at].named_parameters()}
                leaves.update({"d%s_%s" % (at, n): p for n, p in par[at].items()})

        def norm(u, at):
            p = par[at]
            if c["rms"]:
                return u / torch.sqrt(u.pow(2).mean(-1, keepdim=True) + s[at].eps) * p["weight"]
            return (u - u.mean(-1, keepdim=True)) / torch.sqrt(u.var(-1, unbiased=False, keepdim=True) + s[at].eps) * p["weight"] + p["bias"]

        res, r = {}, x
        if y is not None:
            f = norm(y, "post") if c["post"] else y
            r = x + c["scale"] * (gate * f if gate is not None else f)
            res["r"] = r
        if c["pre"]:
            res["h"] = norm(r, "pre")
        if c["grad"]:
            res.update(_grads(leaves, list(res.values()), [s["d" + n].double() for n in res]))
    else:
        x, w, b, rs = up(s["x"]), up(s["w"]), up(s["b"]), up(s["res"])
        z = torch.nn.functional.linear(x, w, b)
        f = {"none": lambda u: u, "relu": torch.relu, "gelu": lambda u: u * torch.special.ndtr(u),
             "quick_gelu": lambda u: u / (1 + torch.exp(-1.702 * u)), "silu": lambda u: u / (1 + torch.exp(-u))}[c["act"]]
        y = f(z) if rs is None else rs + f(z)
        res = {"y": y}
        if c["grad"]:
            res.update(_grads({"dx": x, "dw": w, "db": b, "dres": rs}, [y], [s["dy"].double()]))
    return {k: v.detach() for k, v in res.items()}
