"""The layer operators in float64, step by step, for the tests (numpy; slow and plain).

Each function returns its results and, beside them, the same sums with every term's absolute value: a
rounding error of the kernels is a small multiple of u = 2^-24 of those.
"""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def silu_slope(x):
    s = sigmoid(x)
    return s * (1 + x * (1 - s))


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def layer_norm(x, w, b, eps, dy=None):
    """(y, |y|) and, with dy, (dx, dw, db) and their absolute sums."""
    n = x.shape[-1]
    mean = x.mean(-1, keepdims=True)
    var = ((x - mean) ** 2).mean(-1, keepdims=True)
    r = 1 / np.sqrt(var + eps)
    xh = (x - mean) * r
    # What the mean's and the variance's own rounding can do to xh: they are sums of |x|.
    size = np.abs(xh) + np.abs(x).mean(-1, keepdims=True) * r * (1 + np.abs(xh))
    y = xh * w + b
    ya = size * np.abs(w) + np.abs(b)
    if dy is None:
        return y, ya
    g = w * dy
    ga = np.abs(g)
    dx = r * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
    dxa = r * (
        ga + ga.mean(-1, keepdims=True) + size * (ga * size).mean(-1, keepdims=True)) * (
        1 + np.abs(x).mean(-1, keepdims=True) * r)
    rows = tuple(range(x.ndim - 1))
    grads = (dx, (dy * xh).sum(rows), dy.sum(rows))
    sums = (dxa, (np.abs(dy) * size).sum(rows), np.abs(dy).sum(rows))
    return y, ya, grads, sums


def causal_conv(x, w, b, silu, initial=None, lengths=None, dy=None, dfinal=None):
    """Dict of results: y, final and, with dy, x, weight, bias, initial (gradients); and of absolute sums."""
    batch, length, c = x.shape
    width = w.shape[1]
    lens = [length] * batch if lengths is None else [min(max(int(v), 0), length) for v in lengths]
    out = {"y": np.zeros_like(x), "final": np.zeros((batch, width - 1, c))}
    mag = {k: np.zeros_like(v) for k, v in out.items()}
    if dy is not None:
        for d in (out, mag):
            d.update(x=np.zeros_like(x), weight=np.zeros_like(w), bias=np.zeros(c),
                     initial=np.zeros((batch, width - 1, c)))
    for i in range(batch):
        m = lens[i]
        past = np.zeros((width - 1, c)) if initial is None else initial[i]
        line = np.concatenate([past, x[i, :m]])
        p, pa = np.tile(b, (m, 1)).astype(float), np.tile(np.abs(b), (m, 1)).astype(float)
        for k in range(width):
            p += w[:, k] * line[k:k + m]
            pa += np.abs(w[:, k] * line[k:k + m])
        out["y"][i, :m] = p * sigmoid(p) if silu else p
        # |d silu| <= 1.1 times the error of p, and its own error grows with |p| through e^-p
        mag["y"][i, :m] = (1 + np.abs(p)) * pa if silu else pa
        out["final"][i] = line[m:]
        if dy is None:
            continue
        q = dy[i, :m] * (silu_slope(p) if silu else 1.0)
        # the slope's derivative is at most 0.5
        qa = np.abs(dy[i, :m]) * ((1.1 + pa) * (1 + np.abs(p)) if silu else 1.0)
        for d, qq, ww, ll in ((out, q, w, line), (mag, qa, np.abs(w), np.abs(line))):
            dline = np.zeros_like(line)
            for k in range(width):
                dline[k:k + m] += ww[:, k] * qq
                d["weight"][:, k] += (qq * ll[k:k + m]).sum(0)
            if dfinal is not None:
                dline[m:] += dfinal[i] if d is out else np.abs(dfinal[i])
            d["bias"] += qq.sum(0)
            d["initial"][i], d["x"][i, :m] = dline[:width - 1], dline[width - 1:]
    return out, mag


def _scan_core(d, a, u, B, C, D, h0, lens, e, dlast, A):
    """One channel layout for everything: d, u [b, l, c]; a [b, l, c, n]; B, C [b, l, c, n] (spread over channels)."""
    batch, length, c = u.shape
    n = a.shape[3]
    on = (np.arange(length)[None] < np.asarray(lens)[:, None]).astype(float)[..., None]
    h = h0.copy()
    before, after = np.zeros((batch, length, c, n)), np.zeros((batch, length, c, n))
    for t in range(length):
        before[:, t] = h
        live = on[:, t][..., None]
        h = live * (a[:, t] * h + (d[:, t] * u[:, t])[..., None] * B[:, t]) + (1 - live) * h
        after[:, t] = h
    s = (after * C).sum(-1) + D * u
    r = {"s": s * on, "final": h}
    if e is None:
        return r
    e = e * on
    g = dlast.copy()
    G, Wt = np.zeros_like(before), np.zeros_like(before)
    for t in reversed(range(length)):
        live = on[:, t][..., None]
        now = live * (g + e[:, t][..., None] * C[:, t])
        G[:, t] = now
        Wt[:, t] = now * a[:, t] * before[:, t]
        g = live * (a[:, t] * now) + (1 - live) * g
    r["C"] = e[..., None] * after * on[..., None]
    r["B"] = G * (d * u)[..., None]
    gB = (G * B).sum(-1)
    r["u"] = d * gB + D * e
    r["dd"] = (Wt * A).sum(-1) + gB * u
    r["A"] = (Wt * d[..., None]).sum((0, 1))
    r["D"] = (e * u).sum((0, 1))
    r["initial"] = g
    return r


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus_on=False, initial=None, lengths=None,
                   dy=None, dfinal=None):
    """B, C: [b, l, groups, n].  Dicts (results, absolute sums) with y, final and, with dy, the gradients by name."""
    batch, length, c = u.shape
    n, groups = A.shape[1], B.shape[2]
    per = c // groups
    lens = [length] * batch if lengths is None else [min(max(int(v), 0), length) for v in lengths]
    raw = delta + (0.0 if delta_bias is None else delta_bias)
    d = softplus(raw) if softplus_on else raw
    a = np.exp(d[..., None] * A)
    Bs, Cs = np.repeat(B, per, 2), np.repeat(C, per, 2)
    Dv = np.zeros(c) if D is None else D
    h0 = np.zeros((batch, c, n)) if initial is None else initial
    gate = None if z is None else z * sigmoid(z)
    e = None if dy is None else (dy if z is None else dy * gate)
    dl = np.zeros((batch, c, n)) if dfinal is None else dfinal
    r = _scan_core(d, a, u, Bs, Cs, Dv, h0, lens, e, dl, A)
    ab = np.abs
    m = _scan_core(ab(d), a, ab(u), ab(Bs), ab(Cs), ab(Dv), ab(h0), lens, None if e is None else ab(e), ab(dl), ab(A))
    on = (np.arange(length)[None] < np.asarray(lens)[:, None]).astype(float)[..., None]
    out, mag = {}, {}
    for src, dst, f in ((r, out, lambda v: v), (m, mag, ab)):
        dst["y"] = src["s"] if z is None else src["s"] * f(gate)
        dst["final"] = src["final"]
        if dy is None:
            continue
        for k in ("C", "B"):
            dst[k] = src[k].reshape(batch, length, groups, per, n).sum(3)
        dst["u"], dst["A"], dst["D"], dst["initial"] = src["u"], src["A"], src["D"], src["initial"]
        dst["delta"] = src["dd"] * on * (sigmoid(raw) if softplus_on else 1.0)
        dst["delta_bias"] = dst["delta"].sum((0, 1))
        if z is not None:
            dst["z"] = f(dy) * src["s"] * f(silu_slope(z)) * on
            if dst is mag:  # the slope's own error is relative to its terms, not to their sum
                dst["z"] = ab(dy) * src["s"] * (1.1 + ab(z)) * on
    # Relative error of one factor exp(d A): the exponential's (4 u), its argument's (d is good to 12 u, the
    # product and A log2(e) to 1 u each, scaled by |d A|) and the product's with h (1 u).
    steps = 5 + 14 * float(ab(d[..., None] * A).max()) if length else 5.0
    return out, mag, steps


def scan_tolerance(length, steps, z=None):
    """Multiple of u that an absolute sum of a scan of this length may be off by: one factor per position, the
    sums over the states, channels and positions (pairwise or by blocks: at most 64 roundings on any path, and 16
    for the step size and the other factors), and the gate's e^-z."""
    return steps * length + 96 + (0 if z is None else 4 * float(np.abs(z).max()))
