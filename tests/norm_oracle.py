"""residual_norm in 64 bits, each result with a bound on what float32 arithmetic may leave of it, for the tests of its sums over rows.

u = 2^-24.  A row's sums (a thread's 32 values, six exchanges, four waves) and the handful of operations around them stay within C = 64 steps; the
bounds below carry them, value by value, through the formulas.  A sum over rows adds a step for each level of the kernels' order."""
import torch

u, C = 2.0 ** -24, 64


def _norm(t, dt, w, b, eps, rms):
    """Normalised rows of t, which is off by dt -> n, its error, 1 / deviation, its relative error, affine image, its error."""
    c = t if rms else t - t.mean(-1, keepdim=True)
    rstd = 1.0 / (c.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n = c * rstd
    top = t.abs().amax(-1, keepdim=True) * rstd
    rho = (dt * n.abs()).mean(-1, keepdim=True) * rstd + C * u * (1 + top)
    dn = (dt + (0.0 if rms else dt.mean(-1, keepdim=True))) * rstd + n.abs() * rho + C * u * (n.abs() + top)
    a = n * w + b
    return n, dn, rstd, rho, a, dn * w.abs() + 2 * u * ((n * w).abs() + b.abs())


def _back(g, dg, n, dn, rstd, rho, w, rms):
    """The gradient of the rows behind `_norm` from that of its affine image, and its error."""
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    gw, dgw = g * w, dg * w.abs()
    parts = gw.abs() + n.abs() * mean((gw * n).abs()) + (0.0 if rms else mean(gw.abs()))
    v = rstd * (gw - n * mean(gw * n) - (0.0 if rms else mean(gw)))
    dv = rho * rstd * parts + rstd * (dgw + dn * mean((gw * n).abs()) + n.abs() * mean(dgw * n.abs() + gw.abs() * dn) + (0.0 if rms else mean(dgw)) + C * u * parts)
    return v, dv


def residual_norm64(x, y, post, gate, scale, pre, rms, dr, dh, depth, groups=None):
    """x, y, dr, dh [..., D]; post / pre = (weight, bias or 0, eps) or None; gate broadcastable to x or None; depth: levels of a sum over rows.
    -> {name: (value, bound, terms)}; terms: what a sum adds up, per row."""
    up = lambda t: t.detach().double() if torch.is_tensor(t) else t  # noqa: E731
    x, y, gate, dr, dh = (up(t) for t in (x, y, gate, dr, dh))
    zero = torch.zeros_like(x)
    f, df_ = y, zero
    if post:
        pw, pb, peps = up(post[0]), up(post[1]) + 0 * x, post[2]
        np_, dnp, rstdp, rhop, f, df_ = _norm(y, zero, pw, pb, peps, rms)
    s = scale * (gate if gate is not None else 1.0) + zero
    r, dr_ = x + s * f, s.abs() * df_ + 4 * u * (x.abs() + (s * f).abs())
    res = {"r": (r, dr_, None)}
    e, de = (dr if dr is not None else zero), zero
    if pre:
        nw, nb, neps = up(pre[0]), up(pre[1]) + 0 * x, pre[2]
        nr, dnr, rstdr, rhor, h, dh_err = _norm(r, dr_, nw, nb, neps, rms)
        res["h"] = (h, dh_err, None)
        if dh is not None:
            v, dv = _back(dh, zero, nr, dnr, rstdr, rhor, nw, rms)
            e, de = e + v, dv + 2 * u * (e.abs() + v.abs())
    res["dx"] = (e, de, None)

    def total(t, dt, keep=None):
        """Summed over all rows, or within each entry of the leading dimension."""
        over = tuple(range(1, t.dim() - 1)) if keep else tuple(range(t.dim() - 1))
        add = (lambda z: z.sum(over, keepdim=True) if over else z) if keep else (lambda z: z.sum(over))
        return add(t), add(dt + depth * u * t.abs()), t

    if pre and dh is not None:
        res["dpre_weight"] = total(dh * nr, dh.abs() * dnr)
        res["dpre_bias"] = total(dh, zero)
    if gate is not None:
        res["dgate"] = total(scale * e * f, abs(scale) * (de * f.abs() + e.abs() * df_ + 4 * u * (e * f).abs()), keep=groups)
    g, dg = s * e, s.abs() * (de + 4 * u * e.abs())
    if post:
        res["dpost_weight"] = total(g * np_, dg * np_.abs() + g.abs() * dnp)
        res["dpost_bias"] = total(g, dg)
        g, dg = _back(g, dg, np_, dnp, rstdp, rhop, pw, rms)
    res["dy"] = (g, dg, None)
    return res
