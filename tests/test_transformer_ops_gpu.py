"""Attention, residual norms and linear epilogues of a transformer block (coin_amd.layers) against their definitions in 64 bits.

Tolerances are derived, element by element, from what the kernels round: every product and sum in float32 (2^-24 relative a step), the
probabilities and dS to the tensors' type before they enter the second product, the slope of an activation to half precision and dz to the
tensors' type, and each output once."""
import math

import pytest
import torch

from coin_amd import layers as L
from coin_amd._lib import CoinHipError

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8}
DEV = "cuda"


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def within(got, want, tol, what):
    """|got - want| <= tol element by element (and both finite)."""
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"


# ------------------------------------------------------------------------------------------------------------------------- attention
def attention_oracle(q, k, v, causal, scale, lengths, dout=None):
    """-> {name: (value, bound)} in 64 bits."""
    b, lq, hq, d = q.shape
    lk, hkv = k.shape[1], k.shape[2]
    g, u = hq // hkv, U[q.dtype]
    n = lengths.long() if lengths is not None else torch.full((b,), lk, device=q.device)
    j, i = torch.arange(lk, device=q.device), torch.arange(lq, device=q.device)
    keep = (j[None, None, :] < n[:, None, None]).expand(b, lq, lk)
    if causal:
        keep = keep & (j[None, None, :] <= i[None, :, None] + n[:, None, None] - lq)
    keep = keep.unsqueeze(1)
    live = (j[None, :] < n[:, None])[:, :, None, None]
    hd = lambda x: x.double().transpose(1, 2)  # noqa: E731
    Q = hd(q)
    Kk, V = (hd(torch.where(live, x, torch.zeros_like(x))).repeat_interleave(g, 1) for x in (k, v))
    s = Q @ Kk.transpose(-1, -2) * scale
    ds_ = (d + 8) * 2.0 ** -24 * (Q.abs() @ Kk.abs().transpose(-1, -2)) * scale + 4 * 2.0 ** -24 * s.abs()
    s = s.masked_fill(~keep, float("-inf"))
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    # what float32 scores, exponentials and a sum of lk terms leave of p, relatively
    ep = 2 * torch.where(keep, ds_, 0.0).amax(-1, keepdim=True) + (lk + 64) * 2.0 ** -24
    o = p @ V
    A = p @ V.abs()
    eo = u * o.abs() + (u + 2 * ep) * A + 1e-30
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    res = {"out": (back(o), back(eo))}
    if dout is None:
        return res
    G = hd(dout)
    dp = G @ V.transpose(-1, -2)
    D = (G * o).sum(-1, keepdim=True)
    ds = p * (dp - D)
    # D is formed with the output and what rounding took from it (u * u), whose probabilities were rounded; dp with d products
    eD = (G.abs() * eo).sum(-1, keepdim=True) + d * 2.0 ** -24 * (G.abs() * o.abs()).sum(-1, keepdim=True)
    eds = u * ds.abs() + p * (eD + d * 2.0 ** -24 * (G.abs() @ V.abs().transpose(-1, -2))) + (2 * ep + 2.0 ** -22) * p * (dp.abs() + D.abs())
    acc_k, acc_q = (lk + 8) * 2.0 ** -24, (lq * g + 8) * 2.0 ** -24
    dq = ds @ Kk * scale
    edq = u * dq.abs() + scale * ((eds + acc_k * ds.abs()) @ Kk.abs()) + 1e-30
    grp = lambda x: x.view(b, hkv, g, lk, d).sum(2)  # noqa: E731
    dk = grp(ds.transpose(-1, -2) @ Q) * scale
    edk = u * dk.abs() + scale * grp((eds + acc_q * ds.abs()).transpose(-1, -2) @ Q.abs()) + 1e-30
    dv = grp(p.transpose(-1, -2) @ G)
    edv = u * dv.abs() + grp(((u + 2 * ep + acc_q) * p).transpose(-1, -2) @ G.abs()) + 1e-30
    res.update(dq=(back(dq), back(edq)), dk=(back(dk), back(edk)), dv=(back(dv), back(edv)))
    return res


def check_attention(q, k, v, causal, lengths, what, scale=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = L.attention(q, k, v, causal=causal, scale=scale, key_lengths=lengths)
    dout = rand(out.shape, out.dtype, 99)
    grads = torch.autograd.grad(out, [q, k, v], dout)
    with torch.no_grad():
        again = L.attention(q, k, v, causal=causal, scale=scale, key_lengths=lengths)   # the call without a gradient may split the keys
    ref = attention_oracle(q.detach(), k.detach(), v.detach(), causal, scale or q.shape[-1] ** -0.5, lengths, dout)
    within(again, *ref["out"], what + " out, no gradient")
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads):
        within(t, *ref[name], f"{what} {name}")
    return out, grads


SHAPES = [  # b, lq, lk, hq, hkv, d, causal, lengths
    (1, 1, 1, 1, 1, 8, False, None),
    (2, 1, 1, 2, 1, 64, True, [0, 1]),
    (9, 77, 77, 8, 8, 64, True, None),
    (2, 3, 700, 8, 2, 128, True, [700, 129]),            # new tokens over a ragged cache
    (3, 1, 1300, 6, 2, 96, True, [1300, 0, 257]),
    (2, 130, 67, 3, 3, 32, True, None),                  # more queries than keys: the first see nothing
    (2, 65, 129, 4, 1, 40, False, [129, 64]),
    (1, 513, 513, 2, 1, 128, True, None),
    (4, 33, 31, 5, 5, 24, False, [31, 1, 0, 17]),
    (1, 300, 9, 8, 8, 128, False, None),                 # many rows over few keys
    (2, 257, 255, 4, 2, 64, True, [255, 100]),
    (1, 2, 2050, 1, 1, 64, False, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_its_definition(shape, dtype):
    b, lq, lk, hq, hkv, d, causal, lengths = shape
    q, k, v = rand((b, lq, hq, d), dtype, 1), rand((b, lk, hkv, d), dtype, 2), rand((b, lk, hkv, d), dtype, 3)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32) if lengths else None
    check_attention(q, k, v, causal, n, str(shape))


SPLIT_SHAPES = [   # keys (forward) and rows (dK, dV) in pieces, some of them empty
    (2, 40, 1500, 4, 2, 64, True, [1500, 70]),
    (1, 200, 1030, 4, 4, 128, False, [300]),
    (1, 33, 2100, 2, 1, 32, True, [0]),
    (1, 700, 700, 4, 2, 128, True, None),
    (3, 1000, 129, 2, 1, 64, True, [129, 128, 1]),
    (1, 32, 513, 2, 2, 128, True, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SPLIT_SHAPES)
def test_attention_in_pieces(shape, dtype):
    b, lq, lk, hq, hkv, d, causal, lengths = shape
    q, k, v = rand((b, lq, hq, d), dtype, 1), rand((b, lk, hkv, d), dtype, 2), rand((b, lk, hkv, d), dtype, 3)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int32) if lengths else None
    check_attention(q, k, v, causal, n, str(shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_head_dimensions(dtype):
    for d in range(8, 129, 8) if dtype == BF16 else (4, 12, 32, 36, 64, 68, 100, 128):
        q, k, v = rand((2, 19, 2, d), dtype, d), rand((2, 70, 1, d), dtype, d + 1), rand((2, 70, 1, d), dtype, d + 2)
        check_attention(q, k, v, True, None, f"d={d}")


@pytest.mark.parametrize("std", [0.0, 1e-4, 30.0])
def test_attention_flat_and_peaked_scores(std):
    q, k, v = rand((1, 70, 2, 64), F32, 1, std), rand((1, 200, 2, 64), F32, 2, std), rand((1, 200, 2, 64), F32, 3)
    q, k = (t.to(BF16) for t in (q, k))
    check_attention(q, k, v.to(BF16), False, None, f"std {std}", scale=0.3)


def test_attention_strided_operands_and_broadcast_keys():
    qkv = rand((3, 77, 3, 4, 64), BF16, 5)
    q, k, v = qkv.unbind(2)
    check_attention(q, k, v, True, None, "views of one projection")
    qt = rand((3, 4, 50, 64), BF16, 6).transpose(1, 2)            # heads outside
    check_attention(qt, k, v, False, None, "heads outside")
    odd = rand((3, 50, 4, 67), BF16, 7)[..., 1:65]                # neither pointer nor strides of 16 bytes
    check_attention(odd, k, v, False, None, "unaligned")
    rev = rand((3, 50, 4, 64), BF16, 8).transpose(0, 1).contiguous().transpose(0, 1)
    check_attention(rev, k, v, False, None, "tokens outside")
    one = rand((1, 77, 1, 64), BF16, 9).requires_grad_()          # one key head for every sequence
    kk = one.expand(3, 77, 4, 64)
    qq = rand((3, 20, 4, 64), BF16, 10)
    out = L.attention(qq, kk, kk)
    dout = rand(out.shape, BF16, 11)
    g, = torch.autograd.grad(out, one, dout)
    ref = attention_oracle(qq, kk.detach(), kk.detach(), False, 0.125, None, dout)
    s = lambda x: x.sum((0, 2), keepdim=True)  # noqa: E731
    # the two gradients are rounded, then summed over 12 places and rounded a step at a time by the caller's expansion
    want, tol = s(ref["dk"][0] + ref["dv"][0]), s(ref["dk"][1] + ref["dv"][1])
    within(g, want, tol + 14 * 2.0 ** -8 * s(ref["dk"][0].abs() + ref["dv"][0].abs()), "broadcast keys")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_reads_nothing_behind_the_lengths(dtype):
    q, k, v = rand((3, 5, 4, 64), dtype, 1), rand((3, 200, 2, 64), dtype, 2), rand((3, 200, 2, 64), dtype, 3)
    n = torch.tensor([130, 0, 64], device=DEV, dtype=torch.int32)
    clean = check_attention(q, k, v, True, n, "clean")
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        k2, v2 = k.clone(), v.clone()
        for i, m in enumerate(n.tolist()):
            k2[i, m:] = bad
            v2[i, m:] = bad
        out, grads = check_attention(q, k2, v2, True, n, f"{bad}")
        assert torch.equal(out, clean[0]) and all(torch.equal(a, b) for a, b in zip(grads, clean[1]))
    assert torch.equal(clean[0][1], torch.zeros_like(clean[0][1])) and torch.equal(clean[1][0][1], torch.zeros_like(clean[1][0][1]))
    long = torch.tensor([1 << 30, -5, 64], device=DEV, dtype=torch.int32)   # lengths are clamped to the buffer
    torch.testing.assert_close(L.attention(q, k, v, causal=True, key_lengths=long)[2], clean[0][2], rtol=0, atol=0)


def test_attention_many_heads_over_a_long_and_nearly_empty_buffer():
    # 256 heads times the tokens behind the sequence pass 2^31: those tiles of keys have no rows to start from
    q, k, v = rand((1, 1, 256, 8), BF16, 1), rand((1, 64, 1, 8), BF16, 2), rand((1, 64, 1, 8), BF16, 3)
    lk = (1 << 23) + 300
    bufs = []
    for t in (k, v):
        buf = torch.full((1, lk, 1, 8), float("nan"), device=DEV, dtype=BF16)
        buf[:, :64] = t
        bufs.append(buf.requires_grad_())
    qq = q.clone().requires_grad_()
    out = L.attention(qq, *bufs, causal=True, key_lengths=torch.tensor([64], device=DEV))
    dout = rand(out.shape, BF16, 4)
    dq, dk, dv = torch.autograd.grad(out, [qq] + bufs, dout)
    ref = attention_oracle(q, k, v, True, 8 ** -0.5, None, dout)
    for name, t in (("out", out.detach()), ("dq", dq), ("dk", dk[:, :64]), ("dv", dv[:, :64])):
        within(t, *ref[name], name)
    assert not dk[:, 64:].any() and not dv[:, 64:].any()


def test_attention_gradient_against_differences():
    q, k, v = (rand((1, 6, 2, 8), F32, s, 0.7) for s in (1, 2, 3))
    n = torch.tensor([5], device=DEV, dtype=torch.int32)
    w = rand(q.shape, F32, 4).double()
    xs = [t.requires_grad_() for t in (q, k, v)]
    f = lambda *a: float((L.attention(*a, causal=True, key_lengths=n).double() * w).sum())  # noqa: E731
    grads = torch.autograd.grad(L.attention(*xs, causal=True, key_lengths=n), xs, w.float())
    h = 2.0 ** -6
    with torch.no_grad():
        for i, x in enumerate(xs):
            step = rand(x.shape, F32, 10 + i)
            up, down = ([t + (h * step if t is x else 0.0) for t in xs], [t - (h * step if t is x else 0.0) for t in xs])
            num = (f(*up) - f(*down)) / (2 * h)
            # central difference: h^2 / 6 of a third derivative of order 10, and float32 sums of 96 products over 2 h
            assert abs(num - float((grads[i].double() * step).sum())) < 10 * h * h + 96 * 2.0 ** -22 / h


def test_attention_packed_projection_is_the_same_call():
    qkv = rand((4, 77, 3 * 8 * 64), BF16, 3).requires_grad_()
    n = torch.tensor([77, 5, 0, 40], device=DEV)
    out = L.attention_qkv(qkv, 8, causal=True, key_lengths=n)
    dout = rand(out.shape, BF16, 4)
    g, = torch.autograd.grad(out, qkv, dout)
    p = qkv.detach().view(4, 77, 3, 8, 64).clone().requires_grad_()
    o2 = L.attention(*p.unbind(2), causal=True, key_lengths=n)
    g2, = torch.autograd.grad(o2, p, dout.view(4, 77, 8, 64))
    assert torch.equal(out, o2.reshape(out.shape)) and torch.equal(g, g2.reshape(g.shape))


# --------------------------------------------------------------------------------------------------------------------- residual norm
def make_norm(rms, d, seed, affine=True):
    m = (torch.nn.RMSNorm if rms else torch.nn.LayerNorm)(d, eps=1e-5, elementwise_affine=affine, device=DEV)
    with torch.no_grad():
        for i, p in enumerate(m.parameters()):
            p.copy_(rand((d,), F32, seed + i, 0.3) + (1 - i))
    return m


def check_norm(lead, d, ts, tb, rms, with_y, post, gate, pre, scale, affine=True, std=1.0, mean=0.0):
    x = (rand(lead + (d,), F32, 1, std) + mean).to(ts).requires_grad_()
    y = rand(lead + (d,), tb, 2, std).requires_grad_() if with_y else None
    gt = gate(lead, d, tb).requires_grad_() if gate else None
    pn, nn_ = make_norm(rms, d, 10, affine) if post else None, make_norm(rms, d, 20, affine) if pre else None
    r, h = L.residual_norm(x, y, post_norm=pn, gate=gt, scale=scale, pre_norm=nn_, branch_dtype=tb)
    outs = ([r] if with_y else []) + ([h] if pre else [])
    gos = [rand(o.shape, o.dtype, 30 + i) for i, o in enumerate(outs)]
    leaves = [t for t in (x, y, gt) if t is not None] + [p for m in (pn, nn_) if m is not None for p in m.parameters()]
    names = [n for n, t in (("dx", x), ("dy", y), ("dgate", gt)) if t is not None] + [f"d{w}_{n}" for w, m in (("post", pn), ("pre", nn_)) if m is not None for n, _ in m.named_parameters()]
    grads = dict(zip(names, torch.autograd.grad(outs, leaves, gos)))

    # 64 bits, by differentiation of the definition
    def up(t):
        return t.detach().double().requires_grad_()
    X, Y, G = up(x), up(y) if with_y else None, up(gt) if gt is not None else None
    pars = {w: {n: up(p) for n, p in m.named_parameters()} for w, m in (("post", pn), ("pre", nn_)) if m is not None}
    scales = []   # (rows, largest value of a normalised row's input, 1 / deviation) for the bounds

    def norm(t, w):
        c = t if rms else t - t.mean(-1, keepdim=True)
        rstd = (c.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        scales.append((t.detach().abs().amax(-1, keepdim=True) * rstd.detach()))
        out = c * rstd
        return out * pars[w]["weight"] + (pars[w]["bias"] if "bias" in pars[w] else 0.0) if affine else out
    R = X
    if with_y:
        F = norm(Y, "post") if post else Y
        R = X + scale * (G * F if G is not None else F)
    H = norm(R, "pre") if pre else None
    Os = ([R] if with_y else []) + ([H] if pre else [])
    Gs = dict(zip(names, torch.autograd.grad(Os, [t for t in (X, Y, G) if t is not None] + [p for w in pars.values() for p in w.values()], [g.double() for g in gos])))
    # float32 rows: a normalised value is off by 2^-20 of 1 + (largest input) / deviation at most -- 64 steps of half a unit, sums of up to
    # 8192 values in a tree of depth 19 and a handful of operations; gradients multiply that by the row's own size
    # (without a norm: x + scale * y in float32 with scale as a float32 takes three roundings of 2^-24 of |x| + |scale y|; rows of normal
    # values stay below 6 in either, so 3 * 2^-24 * (6 + 2 * 6) < 2^-18.2, and 2^-19 is taken of 1 + the row's largest result, over 2 in all rows
    # of 7 values and more)
    en = 2.0 ** -19 * (1 + sum(scales, torch.zeros(1, device=DEV, dtype=torch.float64)))
    if pre and post:
        en = en * (1 + scales[0])
    for o, O in zip(outs, Os):
        within(o.detach(), O.detach(), U[o.dtype] * O.detach().abs() + en * (1 + O.detach().abs().amax(-1, keepdim=True)), "output")
    for n in names:
        w = Gs[n]
        t = grads[n]
        assert t.dtype == dict(zip(names, leaves))[n].dtype
        if n in ("dx", "dy"):
            row = w.abs().amax(-1, keepdim=True) + (Gs["dx"].abs().amax(-1, keepdim=True) * (1 + (scales[0] if post else 0)))
            within(t, w, U[t.dtype] * w.abs() + 8 * en * row, n)
        else:   # sums over rows: float32 terms, each off by en of the row's size
            rows = 1 if n != "dgate" else None
            size = sum(g.double().abs().amax() for g in gos) * (1 + Gs["dx"].abs().amax())
            m = x.numel() // d
            within(t, w, U[t.dtype] * w.abs() + 8 * float(en.max()) * float(size) * math.sqrt(m) * (1 + float(en.max() / 2.0 ** -19)) * torch.ones_like(w) * (1 if rows else abs(scale)), n)
    return grads


LAYER = lambda lead, d, tb: rand((d,), F32, 5, 0.5)  # noqa: E731
EACH = lambda lead, d, tb: rand(lead[:1] + (1,) * (len(lead) - 1) + (d,), tb, 5, 0.5)  # noqa: E731
ROWS = lambda lead, d, tb: rand(lead + (d,), tb, 5, 0.5)  # noqa: E731


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("lead,d", [((1,), 1), ((3, 5), 7), ((9, 77), 512), ((2, 37), 96), ((700,), 136), ((3, 11), 1000), ((2, 9), 2048), ((5,), 2501), ((4, 3), 4096), ((3,), 8192)])
def test_residual_norm_matches_its_definition(lead, d, rms, types):
    for kw in (dict(with_y=True, post=False, gate=None, pre=True, scale=1.0), dict(with_y=True, post=True, gate=EACH, pre=True, scale=0.5)):
        check_norm(lead, d, *types, rms, **kw)


@pytest.mark.parametrize("kw", [
    dict(with_y=False, post=False, gate=None, pre=True, scale=1.0),
    dict(with_y=True, post=False, gate=None, pre=False, scale=0.3),
    dict(with_y=True, post=True, gate=None, pre=False, scale=1.0),
    dict(with_y=True, post=False, gate=LAYER, pre=True, scale=1.0),
    dict(with_y=True, post=True, gate=LAYER, pre=False, scale=-2.0),
    dict(with_y=True, post=True, gate=ROWS, pre=True, scale=1.0),
    dict(with_y=True, post=False, gate=EACH, pre=True, scale=1.0, affine=False),
    dict(with_y=True, post=True, gate=EACH, pre=True, scale=0.0),
    dict(with_y=True, post=True, gate=EACH, pre=True, scale=1.0, affine=False),
])
@pytest.mark.parametrize("lead,d", [((4, 50), 64), ((7, 3), 100), ((2, 3, 41), 768), ((40, 130), 16)])
def test_residual_norm_parts(kw, lead, d):
    check_norm(lead, d, F32, F32, False, **kw)
    check_norm(lead, d, F32, BF16, True, **kw)


def test_residual_norm_rows_without_spread_and_far_from_zero():
    check_norm((3, 4), 64, F32, F32, False, True, False, None, True, 1.0, std=0.0, mean=3.0)
    check_norm((3, 4), 512, F32, F32, False, True, False, None, True, 1.0, std=1.0, mean=1000.0)


def test_residual_norm_groups_that_end_inside_a_walk():
    """Gates of few and of many rows: whole inside one walk of the backward, over several, and at both ends."""
    for lead, d in (((5, 1000), 64), ((1000, 5), 64), ((3000, 1), 32), ((700, 9), 520)):
        check_norm(lead, d, F32, F32, True, True, True, EACH, True, 1.0)


def test_residual_norm_without_the_gradient_of_one_output():
    for keep in (0, 1):
        x, y = rand((9, 77, 64), BF16, 1).requires_grad_(), rand((9, 77, 64), BF16, 2).requires_grad_()
        ln = make_norm(False, 64, 3)
        out = L.residual_norm(x, y, pre_norm=ln)[keep]
        g = rand(out.shape, BF16, 4)
        gx, gy, gw = torch.autograd.grad(out, [x, y, ln.weight], g, allow_unused=True)
        X, Y = x.detach().double().requires_grad_(), y.detach().double().requires_grad_()
        O = X + Y if keep == 0 else torch.nn.functional.layer_norm(X + Y, (64,), ln.weight.detach().double(), ln.bias.detach().double(), 1e-5)
        want, = torch.autograd.grad(O, X, g.double())
        within(gx, want, 2.0 ** -8 * want.abs() + 2.0 ** -14 * want.abs().amax(), "dx")
        assert torch.equal(gx, gy) and (gw is None) == (keep == 0)


# ------------------------------------------------------------------------------------------------------------------------------ linear
ACTS = {"none": L.ACT_NONE, "relu": L.ACT_RELU, "gelu": L.ACT_GELU, "quick_gelu": L.ACT_QUICK_GELU, "silu": L.ACT_SILU}


def act64(z, name):
    if name == "none":
        return z
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid((1.702 if name == "quick_gelu" else 1.0) * z)


def check_linear(x, w, b, res, act, what):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    b = b.detach().requires_grad_() if b is not None else None
    res = res.detach().requires_grad_() if res is not None else None
    y = L.fused_linear(x, w, b, act=ACTS[act], residual=res)
    assert y.dtype == (res.dtype if res is not None else x.dtype)
    dy = rand(y.shape, y.dtype, 77)
    leaves = [t for t in (x, w, b, res) if t is not None]
    names = [n for n, t in (("dx", x), ("dw", w), ("db", b), ("dres", res)) if t is not None]
    grads = dict(zip(names, torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        assert torch.equal(L.fused_linear(x, w, b, act=ACTS[act], residual=res), y)
    u = U[x.dtype]
    X, W = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double()
    if w.dtype != x.dtype:
        W = w.detach().to(x.dtype).double()
    B = b.detach().double() if b is not None else torch.zeros(W.shape[0], device=DEV, dtype=torch.float64)
    k, n, m = X.shape[1], W.shape[0], X.shape[0]
    z = (X @ W.t() + B).requires_grad_()
    a = act64(z, act)
    slope, = torch.autograd.grad(a.sum(), z)
    z, a = z.detach(), a.detach()
    ez = (k + 8) * 2.0 ** -24 * (X.abs() @ W.abs().t() + B.abs())
    want = a + (res.detach().double().reshape(m, n) if res is not None else 0.0)
    # an activation's slope stays below 1.2; its own arithmetic in float32 costs 16 steps of its size
    within(y.detach().reshape(m, n), want, U[y.dtype] * want.abs() + 1.2 * ez + 2.0 ** -20 * (a.abs() + want.abs()) + 1e-30, what + " y")
    G = dy.double().reshape(m, n)
    dz = G * slope
    # the slope is off by half a step of its type (2^-11 for half), by its own arithmetic and, through z, by 1.1 ez; next to 0 a ReLU's slope may flip
    es = ((2.0 ** -11 if x.dtype == BF16 else 2.0 ** -24) if act != "none" else 0.0) * slope.abs() + (2.0 ** -20 + 1.1 * ez + 2.0 ** -25 if act not in ("none", "relu") else 0.0)
    if act == "relu":
        es = es + (z.abs() <= ez).double()
    ebz = G.abs() * es                       # before dz is rounded
    edz = ebz + u * (dz.abs() + ebz)
    dx = dz @ W
    within(grads["dx"].reshape(m, k), dx, u * dx.abs() + (edz + (n + 8) * 2.0 ** -24 * dz.abs()) @ W.abs() + 1e-30, what + " dx")
    dw = dz.t() @ X
    within(grads["dw"], dw, U[w.dtype] * dw.abs() + (edz + (m + 64) * 2.0 ** -24 * dz.abs()).t() @ X.abs() + 1e-30, what + " dw")
    if b is not None:
        db = dz.sum(0)
        within(grads["db"], db, U[b.dtype] * db.abs() + (ebz + (m + 8) * 2.0 ** -24 * dz.abs()).sum(0) + 1e-30, what + " db")
    if res is not None:
        assert torch.equal(grads["dres"], dy)
    assert grads["dw"].dtype == w.dtype and grads["dx"].dtype == x.dtype


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 8, 8), (3, 77, 5), (4, 2048, 256), (16, 512, 520), (17, 40, 1000), (100, 1001, 33), (693, 512, 2048), (130, 136, 264),
                                   (2000, 96, 96), (777, 64, 7), (2048, 1024, 2112), (5092, 384, 200), (3500, 264, 3601), (4000, 3400, 72), (1000, 8200, 1100), (3840, 200, 3808)])
def test_linear_sizes(m, k, n, dtype):
    i = (m + k + n) % 5
    act = list(ACTS)[i]
    x, w, b = rand((m, k), dtype, 1), rand((n, k), dtype, 2, k ** -0.5), rand((n,), dtype, 3)
    check_linear(x, w, b, rand((m, n), dtype, 4) if i % 2 else None, act, f"{m} {k} {n} {act}")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_activations(act, dtype):
    x, w, b = rand((3, 50, 72), dtype, 1, 3.0), rand((88, 72), dtype, 2, 72 ** -0.5), rand((88,), F32, 3)
    check_linear(x, w, b, None, act, act)
    check_linear(x, w, None, rand((3, 50, 88), F32, 4), act, act + " on a float32 residual")


def test_linear_strides_and_alignment():
    w = rand((136, 72), BF16, 2, 0.1)
    base = rand((60, 200), BF16, 1)
    for what, x in (("columns of a wider matrix", base[:, 8:80]), ("unaligned columns", base[:, 3:75]), ("transposed", rand((72, 60), BF16, 5).t()),
                    ("every other row", base[::2, :72]), ("one row for all", base[:1, :72].expand(60, 72)), ("reversed batch", rand((6, 10, 72), BF16, 6).transpose(0, 1))):
        check_linear(x, w, None, rand(x.shape[:-1] + (136,), BF16, 4)[..., :], "gelu", what)
    check_linear(base[:, :72], rand((72, 136), BF16, 2, 0.1).t(), None, rand((60, 300), BF16, 3)[:, 5:141], "silu", "transposed weight, unaligned residual")
    y = L.fused_linear(base[:, :72].detach().requires_grad_(), w.requires_grad_())
    g1 = torch.autograd.grad(y.sum(), w, retain_graph=True)[0]          # an expanded gradient (stride 0)
    g2 = torch.autograd.grad(y, w, torch.ones_like(y))[0]
    assert torch.equal(g1, g2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [40, 37])
def test_linear_gradients_of_some_operands_alone(n, dtype):
    """Frozen weights, a bias alone, a residual alone: each gradient is the one of the full call."""
    ts = {"x": rand((50, 64), dtype, 1), "w": rand((n, 64), dtype, 2, 0.1), "b": rand((n,), F32, 3), "res": rand((50, n), dtype, 4)}
    dy = rand((50, n), dtype, 5)
    for act in ("none", "gelu"):
        def grads(names):
            t = {k: v.detach().requires_grad_(k in names) for k, v in ts.items()}
            y = L.fused_linear(t["x"], t["w"], t["b"], act=ACTS[act], residual=t["res"])
            return dict(zip(names, torch.autograd.grad(y, [t[k] for k in names], dy)))
        full = grads(list(ts))
        for names in (["x"], ["w"], ["b"], ["res"], ["x", "b"], ["w", "res"]):
            for k, g in grads(names).items():
                assert torch.equal(g, full[k]), (act, names, k)


def test_residual_norm_gradients_of_some_operands_alone():
    ln, pn = make_norm(False, 96, 1), make_norm(False, 96, 5)
    ts = {"x": rand((4, 30, 96), F32, 1), "y": rand((4, 30, 96), BF16, 2), "gate": rand((4, 1, 96), BF16, 3)}
    g = [rand((4, 30, 96), F32, 6), rand((4, 30, 96), BF16, 7)]
    pars = {"pw": pn.weight, "pb": pn.bias, "nw": ln.weight, "nb": ln.bias}

    def grads(names):
        t = {k: v.detach().requires_grad_(k in names) for k, v in ts.items()}
        for k, p in pars.items():
            p.requires_grad_(k in names)
        r, h = L.residual_norm(t["x"], t["y"], post_norm=pn, gate=t["gate"], scale=0.7, pre_norm=ln)
        return dict(zip(names, torch.autograd.grad([r, h], [t[k] if k in t else pars[k] for k in names], g)))
    full = grads(list(ts) + list(pars))
    for names in (["x"], ["y"], ["gate"], ["pw"], ["pb", "nw"], ["nb"], ["x", "gate"], ["y", "pw"]):
        for k, v in grads(names).items():
            assert torch.equal(v, full[k]), (names, k)


def test_residual_norm_gradient_of_the_stream_alone():
    x, y = (rand((3, 40, 96), F32, i).requires_grad_() for i in (1, 2))
    gate = rand((3, 1, 96), F32, 3).requires_grad_()
    ln, post = make_norm(False, 96, 10), make_norm(False, 96, 20)
    dr = rand(x.shape, F32, 4)
    for turn in range(2):                                 # r keeps a gradient of its own; nothing is written into the caller's
        keep = dr.clone()
        gx, gy = torch.autograd.grad(L.residual_norm(x, y, pre_norm=ln)[0], [x, y], dr)
        assert torch.equal(gx, keep) and torch.equal(gy, keep) and torch.equal(dr, keep)
    gx, gy, gg, gw = torch.autograd.grad(L.residual_norm(x, y, post_norm=post, gate=gate, scale=0.5, pre_norm=ln)[0], [x, y, gate, post.weight], dr)
    X, Y, G, W, B = (t.detach().double().requires_grad_() for t in (x, y, gate, post.weight, post.bias))
    want = torch.autograd.grad(X + 0.5 * G * torch.nn.functional.layer_norm(Y, (96,), W, B, 1e-5), [X, Y, G, W], dr.double())
    assert torch.equal(gx, dr)
    for name, a, b in zip(("dy", "dgate", "dw"), (gy, gg, gw), want[1:]):
        # float32 sums of up to 120 products a value, relative to the largest
        within(a, b, 256 * 2.0 ** -24 * b.abs().amax() + 0 * b, name)
    g, = torch.autograd.grad(L.residual_norm(x, y.detach(), gate=gate.detach())[0].sum(), x)
    assert torch.equal(g, torch.ones_like(x))
    x.grad = y.grad = None
    a, b = x * 2, y * 2                                   # leaves behind other operations, accumulated in place
    L.residual_norm(a, b)[0].backward(dr)
    L.residual_norm(x * 2, y * 2)[0].backward(dr)
    assert torch.equal(x.grad, 4 * dr) and torch.equal(y.grad, 4 * dr)
    x.grad = y.grad = None
    for _ in range(2):                                    # the same gradient tensor for both leaves: neither accumulates into the other
        L.residual_norm(x, y)[0].backward(dr)
    assert torch.equal(x.grad, 2 * dr) and torch.equal(y.grad, 2 * dr) and torch.equal(dr, keep)


def test_linear_one_row_of_any_pitch():
    base = rand((3, 77), BF16, 1)
    w = rand((40, 72), BF16, 2, 0.1)
    check_linear(base[1:2, 3:75], w, None, rand((1, 40), BF16, 3), "gelu", "one row, unaligned")
    check_linear(base[:1, :72], w, None, rand((3, 45), BF16, 3)[2:, :40], "none", "one row of a pitch of 77")
    v = rand((72,), BF16, 4).requires_grad_()                       # a vector
    y = L.fused_linear(v, w, act=L.ACT_SILU, residual=rand((40,), BF16, 5))
    g, = torch.autograd.grad(y, v, rand((40,), BF16, 6))
    assert y.shape == (40,) and g.shape == (72,)


def test_rms_norm_takes_its_default_epsilon_from_its_input():
    m, q = torch.nn.RMSNorm(64, device=DEV), torch.nn.RMSNorm(64, device=DEV)
    x, y = torch.zeros(3, 64, device=DEV), torch.full((3, 64), 2.0 ** -9, device=DEV, dtype=BF16)
    r, h = L.residual_norm(x, y, post_norm=m, pre_norm=q)
    # y's epsilon is bfloat16's 2^-7: y / sqrt(2^-18 + 2^-7); r's float32's
    want = 2.0 ** -9 / (2.0 ** -18 + 2.0 ** -7) ** 0.5
    within(r, torch.full_like(r, want).double(), torch.full_like(r, 2.0 ** -22).double(), "post")
    within(h, torch.full_like(r, want / (want * want + 2.0 ** -23) ** 0.5).double(), torch.full_like(r, 2.0 ** -8).double(), "pre")


def test_linear_master_weights_through_the_shadow():
    x, w, b = rand((70, 64), BF16, 1), rand((40, 64), F32, 2, 0.1), rand((40,), F32, 3)
    check_linear(x, w, b, None, "quick_gelu", "float32 master")
    p = torch.nn.Parameter(w.clone())
    with torch.autocast("cuda", dtype=BF16):
        a = L.fused_linear(x.float(), p, b)
        with torch.no_grad():
            p.mul_(2.0)
        c = L.fused_linear(x.float(), p, b)
    assert a.dtype == BF16 and not torch.equal(a, c)


# ------------------------------------------------------------------------------------------------------------------ together, and in use
def block_of(x, ln1, ln2, wqkv, bqkv, wo, bo, w1, b1, w2, b2, heads, lengths):
    """A pre-norm transformer block on (stream, normalised stream)."""
    _, h = L.residual_norm(x, pre_norm=ln1)
    a = L.attention_qkv(L.fused_linear(h, wqkv, bqkv), heads, causal=True, key_lengths=lengths)
    x, h = L.residual_norm(x, L.fused_linear(a, wo, bo), pre_norm=ln2)
    return L.fused_linear(L.fused_linear(h, w1, b1, act=L.ACT_QUICK_GELU), w2, b2, residual=x)


def make_block(d, dtype):
    ws = [rand(s, dtype, 40 + i, 0.05) for i, s in enumerate([(3 * d, d), (3 * d,), (d, d), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)])]
    return [t.requires_grad_() for t in ws], make_norm(False, d, 60), make_norm(False, d, 70)


def block64(x, ln1, ln2, ws, heads):
    F = torch.nn.functional
    n, l, d = x.shape
    ln = lambda t, m: F.layer_norm(t, (d,), m.weight.double(), m.bias.double(), 1e-5)  # noqa: E731
    q, k, v = F.linear(ln(x, ln1), ws[0], ws[1]).view(n, l, 3, heads, d // heads).permute(2, 0, 3, 1, 4)
    s = (q @ k.transpose(-1, -2)) * (d // heads) ** -0.5 + torch.full((l, l), float("-inf"), device=DEV, dtype=torch.float64).triu(1)
    x = x + F.linear((s.softmax(-1) @ v).transpose(1, 2).reshape(n, l, d), ws[2], ws[3])
    h = F.linear(ln(x, ln2), ws[4], ws[5])
    return x + F.linear(h * torch.sigmoid(1.702 * h), ws[6], ws[7])


@pytest.mark.parametrize("dtype,tol", [(F32, 1e-5), (BF16, 2.0 ** -5)])
def test_a_block_of_them_and_its_gradients(dtype, tol):
    """tol, of each result's 2-norm: float32 keeps 2^-24 a step over some 2000-term sums; in bfloat16 about ten tensors are rounded (2^-8 at
    most each) between the leaf that is furthest away and the result, and errors of the stages add: 10 * 2^-8 < 2^-4.6; half of that is asked,
    roundings being independent."""
    d, heads = 128, 2
    ws, ln1, ln2 = make_block(d, dtype)
    x = rand((5, 77, d), dtype, 1).requires_grad_()
    y = block_of(x, ln1, ln2, *ws, heads, None)
    dy = rand(y.shape, dtype, 2)
    leaves = [x] + ws + list(ln1.parameters()) + list(ln2.parameters())
    got = torch.autograd.grad(y, leaves, dy)
    up = [t.detach().double().requires_grad_() for t in [x] + ws]
    y64 = block64(up[0], ln1, ln2, up[1:], heads)
    want = torch.autograd.grad(y64, up + list(ln1.parameters()) + list(ln2.parameters()), dy.double())
    for i, (a, b) in enumerate(zip((y,) + got, (y64,) + want)):
        rel = float((a.double() - b.double()).norm() / b.double().norm())
        assert rel < tol, (i, rel)


def test_a_block_gives_the_same_bits_twice_and_on_another_stream():
    ws, ln1, ln2 = make_block(128, BF16)
    x = rand((9, 77, 128), BF16, 1).requires_grad_()
    dy = rand(x.shape, BF16, 2)
    n = torch.tensor([77, 3, 50, 0, 1, 77, 64, 65, 9], device=DEV, dtype=torch.int32)
    leaves = [x] + ws + list(ln1.parameters()) + list(ln2.parameters())
    step = lambda: torch.autograd.grad(block_of(x, ln1, ln2, *ws, 2, n), leaves, dy)  # noqa: E731
    a = step()
    b = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a, b, c))


def test_a_block_captured_and_replayed():
    """Forward and backward recorded in one graph, and a second graph beside it; replays with the program's own work between them follow the
    inputs as the eager calls do."""
    ws, ln1, ln2 = make_block(128, BF16)
    n = torch.tensor([60, 31, 0], device=DEV, dtype=torch.int32)
    leaves = ws + list(ln1.parameters()) + list(ln2.parameters())

    def capture(x, dy):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                torch.autograd.grad(block_of(x, ln1, ln2, *ws, 2, n), [x] + leaves, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block_of(x, ln1, ln2, *ws, 2, n)
            outs = (y,) + torch.autograd.grad(y, [x] + leaves, dy)
        return graph, [o.detach() for o in outs]

    xs = [rand((3, 60, 128), BF16, 1).requires_grad_(), rand((3, 200, 128), BF16, 3).requires_grad_()]
    dys = [rand(x.shape, BF16, 2) for x in xs]
    graphs = [capture(x, dy) for x, dy in zip(xs, dys)]
    for turn in range(4):
        for i in ((0, 1) if turn % 2 else (1, 0)):
            with torch.no_grad():
                xs[i].copy_(rand(xs[i].shape, BF16, 100 * turn + i))
            graphs[i][0].replay()
            torch.cuda.synchronize()
            junk = [torch.empty(1 << 20, device=DEV).normal_() for _ in range(3)]   # the program's own allocations
            y = block_of(xs[i], ln1, ln2, *ws, 2, n)
            want = (y,) + torch.autograd.grad(y, [xs[i]] + leaves, dys[i])
            del junk
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want)), (turn, i)


# ------------------------------------------------------------------------------------------ tensors of more than 2^31 elements
def test_attention_of_a_cache_past_32_bits():
    lk, heads = 300000, 64                                # element 2^31 (byte 2^32) is token 262144
    q = rand((1, 1, heads, 128), BF16, 1).requires_grad_()
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn((1, lk, heads, 128), generator=g, device=DEV, dtype=BF16) for _ in range(2))
    k[:, 262144:] *= 1.5                                  # the largest scores lie behind it
    k.requires_grad_()
    v.requires_grad_()
    out = L.attention(q, k, v, causal=True, scale=0.5)
    dout = rand(out.shape, BF16, 3)
    grads = torch.autograd.grad(out, [q, k, v], dout)
    with torch.no_grad():
        again = L.attention(q, k, v, causal=True, scale=0.5)
    for h in (0, 31, 63):
        at = lambda t: t.detach()[:, :, h:h + 1]  # noqa: E731
        ref = attention_oracle(at(q), at(k), at(v), True, 0.5, None, at(dout))
        assert float(ref["dv"][0][:, 262144:].abs().amax()) > 0.01    # what is compared is there
        within(at(again), *ref["out"], f"out of head {h}, no gradient")
        for name, t in zip(("out", "dq", "dk", "dv"), (out,) + grads):
            within(at(t), *ref[name], f"{name} of head {h}")


def test_residual_norm_of_rows_past_32_bits():
    m, d, n = 1_100_000, 2048, 96                         # element 2^31 is in row 1048576
    g = torch.Generator(device=DEV).manual_seed(1)
    x, y = (torch.randn((m, d), generator=g, device=DEV, dtype=BF16) for _ in range(2))
    dr, dh = (torch.randn((m, d), generator=g, device=DEV, dtype=BF16) for _ in range(2))
    gate = rand((d,), BF16, 2)
    post, pre = make_norm(True, d, 10), make_norm(True, d, 20)

    def run(a, b, ga, gb):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        r, h = L.residual_norm(a, b, post_norm=post, gate=gate, scale=0.5, pre_norm=pre)
        return [t.detach() for t in (r, h) + torch.autograd.grad([r, h], [a, b], [ga, gb])]

    whole = run(x, y, dr, dh)
    for first in (0, 1048576 - n // 2, m - n):            # a row's arithmetic is its own
        s = slice(first, first + n)
        assert all(torch.equal(a[s], b) for a, b in zip(whole, run(x[s], y[s], dr[s], dh[s]))), first


@pytest.mark.parametrize("k,n,act", [(8192, 64, "none"), (64, 8192, "gelu")])
def test_linear_of_rows_past_32_bits(k, n, act):
    m, t = 300000, 100                                    # x and dx, or y, its slope and dz, have 2.46e9 elements
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((m, k), generator=g, device=DEV, dtype=BF16).requires_grad_()
    w, b = rand((n, k), BF16, 2, k ** -0.5).requires_grad_(), rand((n,), BF16, 3).requires_grad_()
    y = L.fused_linear(x, w, b, act=ACTS[act])
    dy = torch.zeros_like(y)
    dy[-t:] = rand((t, n), BF16, 4)                       # the last rows alone have a gradient
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    assert not dx[:-t].any()
    X, W, B, G = (z.detach().double() for z in (x[-t:], w, b, dy[-t:]))
    z = (X @ W.t() + B).requires_grad_()
    a = act64(z, act)
    slope, = torch.autograd.grad(a.sum(), z)
    z, a, u = z.detach(), a.detach(), U[BF16]
    ez = (k + 8) * 2.0 ** -24 * (X.abs() @ W.abs().t() + B.abs())
    within(y.detach()[-t:], a, u * a.abs() + 1.2 * ez + 2.0 ** -19 * a.abs() + 1e-30, "y")
    dz = G * slope
    ebz = G.abs() * (2.0 ** -11 * slope.abs() + 2.0 ** -20 + 1.1 * ez + 2.0 ** -25 if act != "none" else 0.0)
    edz = ebz + u * (dz.abs() + ebz)
    within(dx[-t:], dz @ W, u * (dz @ W).abs() + (edz + (n + 8) * 2.0 ** -24 * dz.abs()) @ W.abs() + 1e-30, "dx")
    within(dw, dz.t() @ X, u * (dz.t() @ X).abs() + (edz + (t + 64) * 2.0 ** -24 * dz.abs()).t() @ X.abs() + 1e-30, "dw")
    within(db, dz.sum(0), u * dz.sum(0).abs() + (ebz + (t + 8) * 2.0 ** -24 * dz.abs()).sum(0) + 1e-30, "db")


def test_sequences_of_no_tokens_and_batches_of_none():
    q, k = torch.zeros(2, 0, 4, 64, device=DEV, requires_grad=True), torch.zeros(2, 5, 4, 64, device=DEV, requires_grad=True)
    out = L.attention(q, k, k)
    assert out.shape == (2, 0, 4, 64)
    g = torch.autograd.grad(out.sum(), [q, k])
    assert torch.equal(g[1], torch.zeros_like(k))
    e = L.attention(k, q.detach(), q.detach())          # no keys: zeros
    assert torch.equal(e, torch.zeros_like(e))
    assert torch.autograd.grad(e.sum(), k)[0].abs().sum() == 0
    assert L.attention(q[:0], k[:0], k[:0]).shape == (0, 0, 4, 64)
    ln = make_norm(False, 16, 1)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    r, h = L.residual_norm(x, x, pre_norm=ln)
    gs = torch.autograd.grad([r.sum() + h.sum()], [x, ln.weight])
    assert r.shape == h.shape == (0, 16) and gs[0].shape == (0, 16) and gs[1].abs().sum() == 0
    w = torch.ones(8, 16, device=DEV, requires_grad=True)
    y = L.fused_linear(x, w, act=L.ACT_GELU)
    assert y.shape == (0, 8) and torch.autograd.grad(y.sum(), w)[0].abs().sum() == 0


def test_refusals():
    t = lambda *s, dt=F32: torch.zeros(*s, device=DEV, dtype=dt)  # noqa: E731
    ln, rn = make_norm(False, 16, 1), make_norm(True, 16, 1)
    bad = [
        lambda: L.attention(t(1, 2, 3, 64), t(1, 2, 2, 64), t(1, 2, 2, 64)),                      # 3 query heads over 2
        lambda: L.attention(t(1, 2, 2, 6), t(1, 2, 2, 6), t(1, 2, 2, 6)),                         # head dimension
        lambda: L.attention(t(1, 2, 2, 136), t(1, 2, 2, 136), t(1, 2, 2, 136)),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64, dt=BF16), t(1, 2, 2, 64)),             # types
        lambda: L.attention(t(1, 2, 2, 64, dt=torch.float16), t(1, 2, 2, 64, dt=torch.float16), t(1, 2, 2, 64, dt=torch.float16)),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 3, 2, 64)),
        lambda: L.attention(t(1, 2, 2, 64), t(2, 2, 2, 64), t(2, 2, 2, 64)),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 2, 2, 64), scale=0.0),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 2, 2, 64), scale=float("nan")),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 2, 2, 64), key_lengths=t(1)),
        lambda: L.attention(t(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 2, 2, 64), key_lengths=t(2, dt=torch.int32)),
        lambda: L.attention(t(2, 2, 64), t(2, 2, 64), t(2, 2, 64)),
        lambda: L.attention(torch.zeros(1, 2, 2, 64), t(1, 2, 2, 64), t(1, 2, 2, 64)),
        lambda: L.attention_qkv(t(1, 2, 100), 8),
        lambda: L.residual_norm(t(4, 16), t(4, 16), pre_norm=ln, post_norm=rn),
        lambda: L.residual_norm(t(4, 16)),
        lambda: L.residual_norm(t(4, 16), gate=t(16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 16), t(3, 16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 8), t(4, 8), pre_norm=ln),
        lambda: L.residual_norm(t(4, 16), t(4, 16), pre_norm=torch.nn.GroupNorm(2, 16).cuda()),
        lambda: L.residual_norm(t(4, 16, dt=BF16), t(4, 16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 16, dt=torch.float16), t(4, 16, dt=torch.float16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 6, 16), t(4, 6, 16), gate=t(6, 16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 6, 16), t(4, 6, 16), gate=t(4, 1, 8), pre_norm=ln),
        lambda: L.residual_norm(t(4, 6, 16), t(4, 6, 16), gate=t(4, 1, 16, dt=torch.float16), pre_norm=ln),
        lambda: L.residual_norm(t(4, 16), t(4, 16), pre_norm=ln, scale=float("inf")),
        lambda: L.residual_norm(t(2, 9000), t(2, 9000)),
        lambda: L.fused_linear(t(4, 16), t(8, 15)),
        lambda: L.fused_linear(t(4, 16), t(8, 16), t(7)),
        lambda: L.fused_linear(t(4, 16), t(8, 16), act=L.ACT_LEAKY_RELU),
        lambda: L.fused_linear(t(4, 16), t(8, 16), residual=t(4, 7)),
        lambda: L.fused_linear(t(4, 16), t(8, 16), residual=t(4, 8, dt=BF16)),
        lambda: L.fused_linear(t(4, 16, dt=torch.float16), t(8, 16, dt=torch.float16)),
        lambda: L.fused_linear(t(4, 16), t(8, 16, dt=BF16)),
        lambda: L.fused_linear(t(4, 16), torch.zeros(8, 16)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(CoinHipError):
            f()
            pytest.fail(f"call {i} was not refused")
