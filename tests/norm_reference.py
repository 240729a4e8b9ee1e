"""The residual norms in float64 on the CPU, with bounds on what fp32 arithmetic may add.

``forward`` / ``backward`` return (value, bound) pairs: |kernel - value| <= bound elementwise, for
a kernel that computes in fp32 from the same inputs and rounds each result once to its type.
``U`` is fp32's rounding, 2^-24, and HALF[t] half a step of type t.  A row statistic is a sum of D
squares: at most 16 sequential additions per thread and 10 in the trees, so (with the products,
rsqrt to 2 ulp and the multiplications after it) every factor of a row carries at most K = 40
roundings; a sigmoid is 4 more.  A term's bound is then K U times the sum of the magnitudes it is
made of.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
K = 48
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# results below the normal range of fp16 are rounded to multiples of 2^-24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def _d(t):
    return None if t is None else t.detach().double().cpu()


def _rounded(value, err, dtype):
    return value, err + HALF[dtype] * (value.abs() + err) + TINY[dtype]


def rms(x, eps):
    return (x.square().mean(-1, keepdim=True) + eps).sqrt()


def plain_forward(x, w, eps, out_dtype):
    x, w = _d(x), _d(w)
    n = x / rms(x, eps) * w
    return _rounded(n, K * U * n.abs(), out_dtype)


def parts(update, post_weight, gate, scale, const, eps):
    y = _d(update)
    u = y if post_weight is None else y / rms(y, eps) * _d(post_weight)
    s = torch.ones(1, dtype=torch.float64) if gate is None else torch.sigmoid(_d(gate))
    c = const * (torch.ones(1, dtype=torch.float64) if scale is None else _d(scale))
    return y, u, s, c


def stream_of(residual, update, post_weight, gate, scale, const, eps):
    h = _d(residual)
    _, u, s, c = parts(update, post_weight, gate, scale, const, eps)
    v = h + c * s * u
    return _rounded(v, K * U * (c * s * u).abs() + U * v.abs(), residual.dtype)


def _norm_grad(x, w, eps, dn):
    """(dx, magnitude, per-row terms of dw) of x / rms(x) * w."""
    r = 1 / rms(x, eps)
    a = w * dn
    q = (a * x).mean(-1, keepdim=True)
    dx = r * (a - x * r * r * q)
    mag = r * (a.abs() + x.abs() * r * r * (a * x).abs().mean(-1, keepdim=True))
    return dx, mag, dn * x * r


def _columns(terms, mags):
    """Column sums over every row: n additions in some fixed order of at most n + 8 each."""
    t, m = terms.flatten(0, -2), mags.flatten(0, -2)
    n = t.shape[0]
    return t.sum(0), (K + min(n, 2048) + 8) * U * m.sum(0) + 2.0 ** -149


def plain_backward(x, w, eps, dn):
    dx, mag, tw = _norm_grad(_d(x), _d(w), eps, _d(dn))
    return {"dx": _rounded(dx, 2 * K * U * mag, x.dtype), "dweight": _columns(tw, tw.abs())}


def backward(stream, update, weight, post_weight, gate, scale, const, eps, dstream, dnormed):
    """Gradients from the stream that the forward returned (its norm reads the rounded values)."""
    x, w = _d(stream), _d(weight)
    y, u, s, c = parts(update, post_weight, gate, scale, const, eps)
    dn = torch.zeros_like(x) if dnormed is None else _d(dnormed)
    ds = torch.zeros_like(x) if dstream is None else _d(dstream)
    g, mag, tw = _norm_grad(x, w, eps, dn)
    g, mag = g + ds, mag + ds.abs()
    out = {"dresidual": _rounded(g, 2 * K * U * mag, stream.dtype), "dweight": _columns(tw, tw.abs())}
    if scale is not None:
        t = const * g * s * u
        out["dscale"] = _columns(t, 2 * const * mag * s * u.abs())
    if gate is not None:
        t, m = g * c * u * s * (1 - s), mag * (c * u * s).abs() * 2
        if gate.shape[-1] != x.shape[-1]:
            t, m = t.sum(-1, keepdim=True), m.sum(-1, keepdim=True)
        out["dgate"] = _rounded(t, 3 * K * U * m, gate.dtype)
    du, m = g * c * s, mag * (c * s).abs()
    if post_weight is not None:
        wp = _d(post_weight)
        dy, _, tp = _norm_grad(y, wp, eps, du)
        _, m2, mp = _norm_grad(y.abs(), wp.abs(), eps, m)
        out["dpost_weight"] = _columns(tp, 2 * mp)
        out["dupdate"] = _rounded(dy, 3 * K * U * m2, update.dtype)
    else:
        out["dupdate"] = _rounded(du, 3 * K * U * m, update.dtype)
    return out


def check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), float(((got - value).abs() / bound).max()))
