"""Attention, residual norms and linear epilogues (coin_amd.layers) where a call meets the module, the layout or the mode that it stands for:
default epsilons, wide pitches, column sums, rows that the mask leaves empty, infinities and NaN, forward-mode derivatives."""
import pytest
import torch
import torch.nn.utils.parametrize

from coin_amd import layers as L
from coin_amd._lib import CoinHipError
from norm_oracle import residual_norm64
from test_transformer_ops_gpu import BF16, DEV, F32, U, attention_oracle, check_attention, check_linear, rand, within

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------------------------------- default epsilon
@pytest.mark.parametrize("weight", [F32, BF16, None])
@pytest.mark.parametrize("ts,tb", [(F32, F32), (F32, BF16), (BF16, BF16)])
def test_rms_norm_without_an_epsilon_is_the_module(ts, tb, weight):
    """Rows of 2^-10, whose mean square 2^-20 lies between the epsilons of float32 (2^-23) and bfloat16 (2^-7): on both sides, against the
    modules that the call stands for and against the formula in 64 bits."""
    d = 64
    post, pre = (torch.nn.RMSNorm(d, elementwise_affine=weight is not None, device=DEV, dtype=weight or F32) for _ in range(2))
    x, y = (rand((5, d), F32, 1) * 2.0 ** -10).to(ts), (rand((5, d), F32, 2) * 2.0 ** -10).to(tb)
    _, h = L.residual_norm(x, pre_norm=pre, branch_dtype=tb)
    r, _ = L.residual_norm(torch.zeros_like(x), y, post_norm=post)
    norm64 = lambda t: t.double() / (t.double().pow(2).mean(-1, keepdim=True) + 2.0 ** -23).sqrt()  # noqa: E731
    for got, src, module in ((h, x, pre), (r, y, post)):
        want = norm64(src)
        # a sum of 64 squares, a root and a quotient in float32: 80 steps of 2^-24 at most; then one rounding to the result's type
        tol = (80 * 2.0 ** -24 + U[got.dtype]) * want.abs()
        within(got, want, tol, "formula")
        m = module(src)
        within(got, m.double(), 2 * tol + (U[m.dtype] + 80 * 2.0 ** -24) * want.abs(), "module")


def test_gradient_of_an_rms_norm_without_an_epsilon():
    m = torch.nn.RMSNorm(96, device=DEV)
    x = (rand((7, 96), F32, 1) * 2.0 ** -10).to(BF16).requires_grad_()
    dh = rand((7, 96), BF16, 2)
    gx, gw = torch.autograd.grad(L.residual_norm(x, pre_norm=m)[1], [x, m.weight], dh)
    X, W = x.detach().double().requires_grad_(), torch.ones(96, device=DEV, dtype=torch.float64, requires_grad=True)
    rstd = (X.pow(2).mean(-1, keepdim=True) + 2.0 ** -23).rsqrt()
    want = torch.autograd.grad(X * rstd * W, [X, W], dh.double())
    # float32 sums of 96 products: 128 steps of 2^-24 of the row's largest term; terms of dx: rstd (|dh| + |n| mean |dh n|)
    n = (X * rstd).detach()
    size = rstd.detach() * (dh.double().abs() + n.abs() * (dh.double() * n).abs().mean(-1, keepdim=True))
    within(gx, want[0], U[BF16] * want[0].abs() + 128 * 2.0 ** -24 * size, "dx")
    within(gw, want[1], 128 * 2.0 ** -24 * (dh.double() * n).abs().sum(0), "dw")


# ------------------------------------------------------------------------------------------------------------ pitches past 32 bits
@pytest.mark.parametrize("dtype,rows", [(BF16, 2048), (F32, 1024)])
def test_linear_on_the_last_token_of_each_sequence(dtype, rows):
    """x[:, -1] of [3, rows, 2048]: 260 rows of that pitch pass 2^31 bytes, and so they do for a weight and a gradient cut out the same way."""
    wide = torch.zeros(3, rows, 2048, device=DEV, dtype=dtype)
    cut = wide[:, -1]
    cut.copy_(rand((3, 2048), dtype, 1))
    assert 260 * cut.stride(0) * cut.element_size() >= 2 ** 31
    for n in (72, 37):
        check_linear(cut, rand((n, 2048), dtype, 2, 2048 ** -0.5), rand((n,), F32, 3), None, "gelu", f"last tokens, n={n}")
    check_linear(rand((5, 2048), dtype, 4), cut, None, None, "none", "a weight of wide pitch")
    x, w = rand((3, 64), dtype, 5).requires_grad_(), rand((2048, 64), dtype, 6, 0.1).requires_grad_()
    for act in (L.ACT_NONE, L.ACT_SILU):
        a, b = (torch.autograd.grad(L.fused_linear(x, w, act=act), [x, w], g) for g in (cut, cut.contiguous()))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    res = wide[:, -1, :72]                                 # the residual is read row by row, whatever its pitch
    check_linear(rand((3, 64), dtype, 8), rand((72, 64), dtype, 9, 0.1), None, res, "relu", "a residual of wide pitch")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_over_tokens_that_lie_far_apart(dtype):
    pitch = 2 ** 31 // (130 * (2 if dtype == BF16 else 4)) // 64 * 64 + 128

    def apart(n, heads, seed):
        base = torch.empty(n, pitch, device=DEV, dtype=dtype)
        t = base[:, :heads * 64].unflatten(1, (heads, 64))[None]
        t.copy_(rand(t.shape, dtype, seed))
        return t

    q, k, v = rand((1, 9, 4, 64), dtype, 1), apart(7, 2, 2), apart(7, 2, 3)
    check_attention(q, k, v, True, None, "keys far apart")
    check_attention(apart(9, 4, 4), k.contiguous(), v, False, torch.tensor([5], device=DEV, dtype=torch.int32), "queries far apart")
    qq, kk, vv = (t.contiguous().requires_grad_() for t in (q, k, v))
    dout = apart(9, 4, 5)
    a, b = (torch.autograd.grad(L.attention(qq, kk, vv), [qq, kk, vv], g) for g in (dout, dout.contiguous()))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_over_heads_that_lie_far_apart():
    """Four query heads of one key head, 2^29 bytes from one another: the gradients walk them as rows of one product."""
    base = torch.empty(4, 1 << 28, device=DEV, dtype=BF16)
    q = base[:, :9 * 64].unflatten(1, (9, 64)).transpose(0, 1)[None]
    q.copy_(rand((1, 9, 4, 64), BF16, 1))
    assert q.stride(2) == 1 << 28
    k, v = rand((1, 40, 1, 64), BF16, 2), rand((1, 40, 1, 64), BF16, 3)
    check_attention(q, k, v, True, None, "heads far apart")
    qq = q.contiguous().requires_grad_()
    a, b = (torch.autograd.grad(L.attention(qq, k, v), qq, g)[0] for g in (q, q.contiguous()))
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------- forward mode and recorded calls
def calls():
    """One call of each entry point as a function of one tensor, and that tensor."""
    w, ln = rand((16, 16), F32, 5), torch.nn.LayerNorm(16, device=DEV).requires_grad_(False)
    kv = rand((2, 7, 2, 8), F32, 6)
    x = rand((3, 16), F32, 7)
    return {
        "attention": (lambda t: L.attention(t, kv, kv), rand((2, 5, 4, 8), F32, 1)),
        "attention keys": (lambda t: L.attention(kv, t, kv), rand((2, 7, 2, 8), F32, 1)),
        "attention_qkv": (lambda t: L.attention_qkv(t, 2), rand((2, 5, 48), F32, 2)),
        "residual_norm": (lambda t: L.residual_norm(x, t, pre_norm=ln)[1], rand((3, 16), F32, 3)),
        "fused_linear": (lambda t: L.fused_linear(t, w, act=L.ACT_GELU), rand((3, 16), F32, 4)),
        "fused_linear weight": (lambda t: L.fused_linear(x, t), rand((16, 16), F32, 4)),
    }


@pytest.mark.parametrize("grad", [False, True])
def test_a_forward_mode_tangent_is_refused_not_dropped(grad):
    for name, (f, t) in calls().items():
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
            assert not dual.requires_grad
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                f(dual)
                pytest.fail(f"{name} gave a result without its tangent")
            with torch.no_grad():
                assert torch.equal(f(t), f(t.clone())), name          # operands without a tangent are as good as outside
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
            pytest.fail(f"{name} gave a result without its tangent")


def test_a_traced_call_is_refused():
    for name, (f, t) in calls().items():
        for needs in (False, True):
            with pytest.raises(CoinHipError):
                torch.jit.trace(f, (t.detach().clone().requires_grad_(needs),), check_trace=False)
                pytest.fail(f"{name} was recorded")
        assert f(t).isfinite().all()


# -------------------------------------------------------------------------------------------------- modules that are not what they seem
class _Shifted(torch.nn.LayerNorm):
    def forward(self, x):
        return super().forward(x) + 1


class _Named(torch.nn.RMSNorm):
    """A subclass that computes what its base does."""


def test_norms_that_compute_something_else_are_refused():
    x, y = rand((4, 16), F32, 1), rand((4, 16), F32, 2)
    swapped = torch.nn.LayerNorm(16, device=DEV)
    swapped.forward = lambda t: t
    hooked = [torch.nn.LayerNorm(16, device=DEV) for _ in range(3)]
    hooked[0].register_forward_hook(lambda m, i, o: 2 * o)
    hooked[1].register_forward_pre_hook(lambda m, i: (2 * i[0],))
    hooked[2].register_full_backward_hook(lambda m, gi, go: None)
    for bad in [_Shifted(16, device=DEV), swapped] + hooked:
        for kw in (dict(pre_norm=bad), dict(post_norm=bad)):
            with pytest.raises(CoinHipError):
                L.residual_norm(x, y, **kw)
                pytest.fail(f"{bad} was taken for its base")
    a, b = _Named(16, device=DEV), torch.nn.RMSNorm(16, device=DEV)
    assert torch.equal(L.residual_norm(x, y, pre_norm=a)[1], L.residual_norm(x, y, pre_norm=b)[1])
    torch.nn.utils.parametrize.register_parametrization(b, "weight", _Doubled())
    within(L.residual_norm(x, pre_norm=b)[1], 2 * L.residual_norm(x, pre_norm=a)[1].detach().double(), 2.0 ** -30 * torch.ones_like(x).double(), "parametrized")


class _Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


# ------------------------------------------------------------------------------------------------------------------ sums over the rows
WALKS = [   # rows of one gate: over many walks of the backward, a part of one, several whole ones within one, one row each
    ((5, 1000), 64), ((1000, 5), 64), ((3000, 1), 32), ((700, 9), 520), ((40000, 3), 32), ((4500, 2), 2501), ((9, 77), 512), ((2, 37), 96), ((40, 130), 16),
    ((700,), 136), ((3, 41), 768), ((7, 9), 100), ((3, 500), 4096), ((2, 700), 8192),
]


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("lead,d", WALKS)
def test_residual_norm_gradients_column_by_column(lead, d, rms, types):
    """Both norms and a gate, by layer and by group; every gradient within the bounds of norm_oracle, which are asserted to be a small part of
    the sums (a walk's rows are added one by one, then 16 walks, up to 64 + 16 workgroups: 128 levels while a walk has up to 32 rows)."""
    ts, tb = types
    kind = torch.nn.RMSNorm if rms else torch.nn.LayerNorm
    post, pre = kind(d, eps=1e-5, device=DEV), kind(d, eps=1e-5, device=DEV)
    with torch.no_grad():
        for i, p in enumerate(list(post.parameters()) + list(pre.parameters())):
            p.mul_(1.0).add_(rand((d,), F32, 20 + i, 0.3))
    x, y = rand(lead + (d,), ts, 1).requires_grad_(), rand(lead + (d,), tb, 2).requires_grad_()
    dr, dh = rand(lead + (d,), ts, 3), rand(lead + (d,), tb, 4)
    for groups in (False, True):
        gate = rand(lead[:1] + (1,) * (len(lead) - 1) + (d,) if groups else (d,), tb if groups else F32, 5, 0.5).requires_grad_()
        outs = L.residual_norm(x, y, post_norm=post, gate=gate, scale=0.7, pre_norm=pre)
        leaves = {"dx": x, "dy": y, "dgate": gate, **{f"d{w}_{n}": p for w, m in (("post", post), ("pre", pre)) for n, p in m.named_parameters()}}
        got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), [dr, dh])), r=outs[0].detach(), h=outs[1].detach())
        par = lambda m: (m.weight, getattr(m, "bias", None) if not rms else 0.0, 1e-5)  # noqa: E731
        want = residual_norm64(x, y, par(post), gate, 0.7, par(pre), rms, dr, dh, depth=128, groups=groups)
        for name, t in got.items():
            value, bound, terms = want[name]
            if name.startswith(("dgate", "dpost", "dpre")):
                # worst cases of m terms add up with m, terms of random signs with its root: 120000 rows leave the largest ratio
                assert bool((bound < 0.1 * value.abs().amax()).all()), name
            within(t, value, bound + (U[t.dtype] * value.abs() if t.dtype == BF16 else 2 * U[F32] * value.abs()), f"{name}, groups={groups}")


# ------------------------------------------------------------------------------------------------------------------ infinities and NaN
@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("d", [40, 100, 2048])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_residual_norm_keeps_a_bad_row_to_itself(bad, d, rms, types):
    """One bad value in x, y, dr or dh: rows without it keep their bits, its own row is not finite wherever the definition's is not, and so are the
    sums it enters: all columns' or its own, and its own group's gate alone."""
    ts, tb = types
    kind = torch.nn.RMSNorm if rms else torch.nn.LayerNorm
    post, pre = kind(d, eps=1e-5, device=DEV), kind(d, eps=1e-5, device=DEV)
    lead, at = (6, 11), (2, 7)
    base = [rand(lead + (d,), t, i) for i, t in enumerate((ts, tb, ts, tb))]
    gate = rand((6, 1, d), tb, 9, 0.5)
    rows = torch.ones(lead, dtype=torch.bool, device=DEV)
    rows[at] = False

    def run(ts_, f):
        x, y, g = (t.detach().requires_grad_() for t in (ts_[0], ts_[1], gate.double() if f is plain else gate))
        leaves = [x, y, g] + list(post.parameters()) + list(pre.parameters())
        outs = f(x, y, g)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [t.to(o.dtype) for t, o in zip(ts_[2:], outs)]))

    def own(x, y, g):
        return L.residual_norm(x, y, post_norm=post, gate=g, scale=0.5, pre_norm=pre)

    def plain(x, y, g):
        def norm(t, m):
            c = t if rms else t - t.mean(-1, keepdim=True)
            return c * (c.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * m.weight.double() + (0.0 if rms else m.bias.double())
        r = x.double() + 0.5 * g * norm(y.double(), post)
        return r, norm(r, pre)

    clean = run(base, own)
    for i in range(4):
        ts_ = [t.clone() for t in base]
        ts_[i][at + (3,)] = bad
        got, want = run(ts_, own), run(ts_, plain)
        for j in (0, 1, 2, 3):                                                   # r, h, dx, dy
            assert torch.equal(got[j][rows], clean[j][rows]), (i, j)
            assert not (got[j].isfinite() & ~want[j].isfinite()).any(), (i, j)    # nothing bad is made good
            assert bool(got[j][want[j].isfinite()].isfinite().all()), (i, j)      # nor the other way
        other = [k for k in range(6) if k != at[0]]
        assert torch.equal(got[4][other], clean[4][other])
        for g, w in zip(got[4:], want[4:]):
            assert torch.equal(g.isfinite(), w.isfinite()), i


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 70, 30, 4, 2, 64), (1, 300, 170, 2, 1, 128), (1, 900, 40, 2, 2, 32)])
def test_queries_that_see_no_key_may_hold_anything(shape, dtype):
    """More causal queries than keys: the first rows see nothing.  NaN in them and in their gradient reaches no other result."""
    b, lq, lk, hq, hkv, d = shape
    q, k, v = rand((b, lq, hq, d), dtype, 1), rand((b, lk, hkv, d), dtype, 2), rand((b, lk, hkv, d), dtype, 3)
    n = torch.tensor([lk - 3 * i for i in range(b)], device=DEV, dtype=torch.int32)
    dout = rand(q.shape, dtype, 4)
    dead = torch.arange(lq, device=DEV)[None, :] < lq - n[:, None]
    qb, gb = q.clone(), dout.clone()
    qb[dead] = float("nan")
    gb[dead] = float("nan")
    res = []
    for qq, gg in ((q, dout), (qb, gb)):
        ts = [t.clone().requires_grad_() for t in (qq, k, v)]
        out = L.attention(*ts, causal=True, key_lengths=n)
        with torch.no_grad():
            again = L.attention(*ts, causal=True, key_lengths=n)
        res.append([out.detach(), again] + list(torch.autograd.grad(out, ts, gg)))
    zero = torch.where(dead[:, :, None, None], torch.zeros_like(dout), dout)
    ref = attention_oracle(q, k, v, True, d ** -0.5, n, zero)
    for name, clean, bad in zip(("out", "out", "dq", "dk", "dv"), *res):
        assert not clean.isnan().any()
        within(bad, *ref[name], name)
        if name in ("out", "dq"):
            assert not bad[dead].any(), name


# ------------------------------------------------------------------------------------------------------- operands kept elsewhere meanwhile
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("keep", ["copies", "host"])
def test_operands_that_a_saved_tensor_hook_lays_out_anew(keep, dtype):
    """Copies and the host's offload give strided operands back dense: the gradients are those without a hook."""
    hook = lambda: (torch.autograd.graph.save_on_cpu() if keep == "host"  # noqa: E731
                    else torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t))
    base = rand((3, 40, 3, 4, 64), dtype, 1)
    wide = rand((3, 40, 1024), dtype, 2)[..., 128:896]
    x, w = rand((50, 200), dtype, 3)[:, 8:72], rand((96, 128), dtype, 4, 0.1)[:, 64:]
    ln = torch.nn.LayerNorm(64, device=DEV)

    def views(t):
        return L.attention(*t.unbind(2), causal=True, key_lengths=n)

    def packed(t):
        return L.attention_qkv(t, 4, causal=True)

    def linear(t):
        return L.fused_linear(t, w, act=L.ACT_GELU)

    def norm(t):
        return L.residual_norm(t, t.flip(0), post_norm=ln, pre_norm=ln)[1]

    n = torch.tensor([40, 7, 33], device=DEV, dtype=torch.int32)
    for f, src in ((views, base), (packed, wide), (linear, x), (norm, x)):
        t = src.detach().requires_grad_()
        assert f in (views,) or not t.is_contiguous()
        with hook():
            out = f(t)
        dout = rand(out.shape, out.dtype, 9)
        got, = torch.autograd.grad(out, t, dout)
        want, = torch.autograd.grad(f(t), t, dout)
        assert torch.equal(got, want), f.__name__
