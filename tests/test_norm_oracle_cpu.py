"""The bounds of tests/norm_oracle.py hold for float32 arithmetic and are small enough to notice a row, a walk or a group that is lost."""
import pytest
import torch

from norm_oracle import residual_norm64

DEPTH = 128


def case(lead, d, rms, gate, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    shape = lead + (d,)
    return dict(x=n(*shape), y=n(*shape), post=(1 + 0.3 * n(d), 0.0 if rms else 0.3 * n(d), 1e-5), pre=(1 + 0.3 * n(d), 0.0 if rms else 0.3 * n(d), 1e-5),
                gate={"layer": n(d) * 0.5, "groups": n(lead[0], *([1] * (len(lead) - 1)), d) * 0.5}[gate], scale=0.7, rms=rms, dr=n(*shape), dh=n(*shape))


def float32(c):
    """The formulas by torch's own float32 operations."""
    leaf = lambda t: t.clone().requires_grad_() if torch.is_tensor(t) else t  # noqa: E731
    x, y, gate = leaf(c["x"]), leaf(c["y"]), leaf(c["gate"])
    (pw, pb, pe), (nw, nb, ne) = (tuple(leaf(t) for t in c[k]) for k in ("post", "pre"))

    def norm(t, w, b, eps):
        t = t if c["rms"] else t - t.mean(-1, keepdim=True)
        return t * (t.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w + b

    r = x + c["scale"] * gate * norm(y, pw, pb, pe)
    h = norm(r, nw, nb, ne)
    names = {"dx": x, "dy": y, "dgate": gate, "dpost_weight": pw, "dpre_weight": nw}
    if not c["rms"]:
        names.update(dpost_bias=pb, dpre_bias=nb)
    got = dict(zip(names, torch.autograd.grad([r, h], list(names.values()), [c["dr"], c["dh"]])))
    return {"r": r.detach(), "h": h.detach(), **got}


SHAPES = [((5, 200), 64), ((150, 5), 64), ((40, 9), 130), ((3, 7), 8), ((70,), 24)]


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("gate", ["layer", "groups"])
@pytest.mark.parametrize("lead,d", SHAPES)
def test_float32_stays_within_the_bounds(lead, d, gate, rms):
    c = case(lead, d, rms, gate)
    want = residual_norm64(**c, depth=DEPTH, groups=gate == "groups")
    for name, got in float32(c).items():
        value, bound, _ = want[name]
        assert got.shape == value.shape and bool(((got.double() - value).abs() <= bound).all()), name


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("gate", ["layer", "groups"])
@pytest.mark.parametrize("lead,d", SHAPES)
def test_the_bounds_notice_what_is_lost(lead, d, gate, rms):
    """Each row by itself: without it, some column of each sum leaves its bound; no sum may be zeros; no two groups may change places."""
    want = residual_norm64(**case(lead, d, rms, gate), depth=DEPTH, groups=gate == "groups")
    for name in ("dgate", "dpost_weight", "dpre_weight") + (() if rms else ("dpost_bias", "dpre_bias")):
        value, bound, terms = want[name]
        assert bool((bound < 0.01 * value.abs().amax()).all()), name
        if name == "dgate" and gate == "groups":
            bound = bound.expand(terms.shape)
            swapped = (value.roll(1, 0) - value).abs() > want[name][1]
            assert bool(swapped.flatten(1).any(1).all()), name
        assert bool((terms.abs() > 2 * bound).any(-1).all()), name
