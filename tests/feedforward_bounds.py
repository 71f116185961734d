"""64-bit results of the feed-forward operators with elementwise error bounds.

``U`` is half a step of fp32 relative to the value (2^-24), ``half(t)`` that of type ``t``.  A sum of n terms in fp32 is
off by at most (n - 1) U sum|terms| in any order; the bounds below count these, every other fp32 operation as one U of
its result, and the last rounding as ``half(t)`` of the value.  All arithmetic here is fp64 on the CPU."""
import math

import torch

U = 2.0 ** -24


def half(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def wide(t):
    return None if t is None else t.detach().cpu().double()


def close(name, got, want, tol, dtype):
    """|got - want| <= tol + half(dtype) (|want| + tol), elementwise; the worst ratio is reported."""
    assert got.dtype == dtype and got.shape == want.shape, (name, got.dtype, got.shape, want.shape)
    lim = tol + half(dtype) * (want.abs() + tol) + 1e-38
    ratio = ((got.detach().cpu().double() - want).abs() / lim)
    assert not ratio.isnan().any(), f"{name}: NaN"
    worst = ratio.max().item() if ratio.numel() else 0.0
    assert worst <= 1.0, f"{name}: error {worst:.3g} times its bound"


def layer_norm_bounds(x, w, b, dy, eps):
    """(value, tolerance) of y, dx, dw, db for 2-D x."""
    x, w, b, dy = wide(x), wide(w), wide(b), wide(dy)
    M, C = x.shape
    w = torch.ones(C, dtype=torch.float64) if w is None else w
    b = torch.zeros(C, dtype=torch.float64) if b is None else b
    mu = x.mean(-1, keepdim=True)
    r = ((x - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mu) * r
    # mean: at most C terms, its error U C mean|x| moves every x - mu; the error of the mean of squares from that of
    # the mean is of second order (sum of x - mu is zero), the rest is relative: (C + 4) U, half of it in r
    rel = (C + 8) * U
    exh = rel * (r * x.abs().mean(-1, keepdim=True) + xh.abs()) + 2 * U * (r * (x - mu).abs())
    y = xh * w + b
    ty = exh * w.abs() + 3 * U * (xh * w).abs() + 2 * U * (b.abs() + y.abs())
    out = {"y": (y, ty)}
    if dy is None:
        return out
    g = dy * w
    mg, mq = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    ag, aq = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    emq = (C + 4) * U * aq + (g.abs() * exh).mean(-1, keepdim=True)
    dx = r * (g - mg - xh * mq)
    tdx = r * ((rel + 6 * U) * (g.abs() + mg.abs() + (xh * mq).abs()) + (C + 4) * U * ag + exh * mq.abs()
               + xh.abs() * emq + exh * emq)
    tdw = ((M + 4) * U * (dy * xh).abs() + dy.abs() * exh).sum(0)
    tdb = (M + 1) * U * dy.abs().sum(0)
    out.update(dx=(dx, tdx), dw=((dy * xh).sum(0), tdw), db=(dy.sum(0), tdb))
    return out


def _act(g, act):
    if act == "gelu":
        phi = torch.special.ndtr(g)
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def gated_bounds(x, w, b, dh, act, op: torch.dtype):
    """(value, tolerance) of h, dx, dw, db for 2-D x; ``op``: the type of the matrix operands (x and w hold it)."""
    x, w, b, dh = wide(x), wide(w), wide(b), wide(dh)
    (M, D), F = x.shape, w.shape[0] // 2
    gu = x @ w.t() + (0 if b is None else b)
    # products of D terms accumulated in fp32 (a matrix instruction may truncate: a whole step, 2 U, per addition)
    egu = 2 * U * (D + 2) * (x.abs() @ w.abs().t() + (0 if b is None else b.abs()))
    (g, u), (eg, eu) = gu.chunk(2, 1), egu.chunk(2, 1)
    a, d = _act(g, act)
    # exp, erf and the few operations behind them: 8 U (1 + |g|) absolute for the activation's values, times |g| where
    # it multiplies; |act'| <= 1.13 and |act''| <= 0.8 for all three
    ea = 1.13 * eg + 8 * U * (1 + g.abs()) ** 2
    ed = 0.8 * eg + 8 * U * (1 + g.abs()) ** 2
    h = a * u
    th = u.abs() * ea + a.abs() * eu + ea * eu + 2 * U * h.abs()
    out = {"h": (h, th)}
    if dh is None:
        return out
    dg, du = dh * u * d, dh * a
    tdg = dh.abs() * (u.abs() * ed + d.abs() * eu + ed * eu) + 3 * U * dg.abs()
    tdu = dh.abs() * ea + 2 * U * du.abs()
    dgu, tdgu = torch.cat((dg, du), 1), torch.cat((tdg, tdu), 1)
    db, tdb = dgu.sum(0), tdgu.sum(0) + (M + 1) * U * (dgu.abs() + tdgu).sum(0)
    t = tdgu + half(op) * (dgu.abs() + tdgu)     # the operand of the two products below
    big = dgu.abs() + t
    out["dx"] = (dgu @ w, t @ w.abs() + 2 * U * (2 * F + 2) * (big @ w.abs()))
    out["dw"] = (dgu.t() @ x, t.t() @ x.abs() + 2 * U * (M + 2) * (big.t() @ x.abs()))
    out["db"] = (db, tdb)
    return out
