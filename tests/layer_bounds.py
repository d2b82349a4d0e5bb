"""The selective scan and its gradients in float64, each value with a bound on a float32 computation's error.

The bounds follow the recurrences themselves (first order, u = 2^-24 per rounding), so they grow with what a state
remembers and not with the length of the sequence.  Torch on the inputs' device.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def _sigmoid_error(x):
    """Relative, in u: 2^(-x log2 e) by its argument (the product and the constant: 2 |x|) and its own 2^-22.5 (2.9),
    a sum (1) and a reciprocal of 2^-23 (2)."""
    return 6 + 2 * x.abs()


def _silu_slope(x):
    """s (1 + x (1 - s)) and its error in u.  1 - s has the absolute error of s and one rounding; three more behind."""
    s = torch.sigmoid(x)
    inner = 1 + x.abs() * (1 - s)
    return s * (1 + x * (1 - s)), s * ((_sigmoid_error(x) + 3) * inner + x.abs() * (_sigmoid_error(x) + 2))


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, initial=None, lengths=None, dy=None,
         dfinal=None):
    """{name: (value, bound)}: y, final and, with dy, u, delta, A, B, C, D, z, delta_bias and initial."""
    f = torch.float64
    u, delta, A, B, C, D, z, bias, h, dy, dfinal = (
        None if t is None else t.detach().to(f) for t in (u, delta, A, B, C, D, z, delta_bias, initial, dy, dfinal))
    batch, length, c = u.shape
    groups, n = B.shape[2:]
    per = c // groups
    on = torch.ones(batch, length, 1, dtype=f, device=u.device)
    if lengths is not None:
        on = (torch.arange(length, device=u.device)[None] < lengths[:, None]).to(f)[..., None]
        u, delta, z, dy = (None if t is None else torch.where(on > 0, t, 0.0) for t in (u, delta, z, dy))
        B, C = (torch.where(on[..., None] > 0, t, 0.0) for t in (B, C))
    D0 = torch.zeros(c, dtype=f, device=u.device) if D is None else D
    h = torch.zeros(batch, c, n, dtype=f, device=u.device) if h is None else h

    raw = delta if bias is None else delta + bias
    if softplus:
        # max(x, 0) + log1p(t): x is off by one rounding; t by 2 |x| + 2.9, log1p's division and series by 9 more;
        # the last sum by one.
        tail = torch.log1p(torch.exp(-raw.abs()))
        d = raw.clamp(min=0) + tail
        ed = torch.sigmoid(raw) * raw.abs() + tail * (12 + 2 * raw.abs()) + d
        slope, eslope = torch.sigmoid(raw), torch.sigmoid(raw) * (_sigmoid_error(raw) + raw.abs())
    else:
        d, ed = raw, raw.abs()
        slope, eslope = torch.ones_like(raw), torch.zeros_like(raw)
    d, ed = d * on, ed * on
    gate, egate = 1.0, 0.0
    if z is not None:
        gate = z * torch.sigmoid(z)
        egate = gate.abs() * (_sigmoid_error(z) + 1)

    def channels(t, k):  # B or C of position k for every channel
        return t[:, k].repeat_interleave(per, 1)

    def decay(k):
        """exp(d A): x = d A log2(e) is off by d's error and three roundings; 2^x by 2.9, or by the last rounding of its
        series (|x| < 1/16) and |x| times those before it."""
        x = d[:, k, :, None] * A
        a = torch.exp(x)
        return a, a * (ed[:, k, :, None] * A.abs() + 3 * x.abs() + torch.where(x.abs() > 0.043, 2.9, 1 + 4 * x.abs()))

    hs, ehs, y, ey, s_all, es_all = [h], [torch.zeros_like(h)], [], [], [], []
    for k in range(length):
        a, ea = decay(k)
        du = (d[:, k] * u[:, k])[..., None]
        Bk, Ck = channels(B, k), channels(C, k)
        eh = a * ehs[-1] + ea * h.abs() + ((ed[:, k] * u[:, k].abs())[..., None] + 2 * du.abs()) * Bk.abs()
        live = on[:, k, :, None] > 0
        h = torch.where(live, a * h + du * Bk, h)
        eh = torch.where(live, eh + h.abs(), ehs[-1])
        hs.append(h)
        ehs.append(eh)
        s = (Ck * h).sum(-1) + D0 * u[:, k]
        es = (Ck.abs() * eh).sum(-1) + (n + 4) * (Ck * h).abs().sum(-1) + 2 * (D0 * u[:, k]).abs() + s.abs()
        s_all.append(s)
        es_all.append(es)
        g, eg = (gate, egate) if z is None else (gate[:, k], egate[:, k])
        y.append(s * g * on[:, k])
        ey.append((es * abs(g) + s.abs() * eg + (s * g).abs()) * on[:, k])
    out = {"y": (torch.stack(y, 1), torch.stack(ey, 1)), "final": (hs[-1], ehs[-1])}
    if dy is not None:
        e = dy * gate
        ee = dy.abs() * egate + e.abs()
        carry = torch.zeros_like(h) if dfinal is None else dfinal.clone()
        ecarry = torch.zeros_like(h)
        dA, edA, walk = (torch.zeros_like(h) for _ in range(3))
        per_step = {k: [None] * length for k in ("u", "delta", "B", "C", "z")}
        # Sums over a group's channels: pairs, 32 lanes, warps, then a tile of at least 16 channels at a time.
        path = c // 16 + 32
        for k in reversed(range(length)):
            a, ea = decay(k)
            Bk, Ck = channels(B, k), channels(C, k)
            live = on[:, k, :, None] > 0
            ek, eek, dk, uk = (t[:, k, :, None] for t in (e, ee, d, u))
            g = Ck * ek + carry
            eg = Ck.abs() * eek + ecarry + g.abs()
            nc, enc = a * g, a * eg + ea * g.abs() + (a * g).abs()
            w = nc * hs[k]
            ew = enc * hs[k].abs() + nc.abs() * ehs[k] + w.abs()
            # dA walks through the positions from the last: a rounding of each partial sum.
            dA = torch.where(live, dA + dk * w, dA)
            walk = torch.where(live, walk + dA.abs(), walk)
            edA = torch.where(live, edA + dk.abs() * ew + ed[:, k, :, None] * w.abs(), edA)
            gB, egB = (g * Bk).sum(-1), (eg * Bk.abs()).sum(-1) + (n + 4) * (g * Bk).abs().sum(-1)
            aw, eaw = (A * w).sum(-1), (A.abs() * ew).sum(-1) + (n + 8) * (A * w).abs().sum(-1)
            v = d[:, k] * gB + D0 * e[:, k]
            ev = (d[:, k].abs() * egB + ed[:, k] * gB.abs() + (d[:, k] * gB).abs() + D0.abs() * ee[:, k]
                  + (D0 * e[:, k]).abs() + v.abs())
            dd = aw + u[:, k] * gB
            edd = eaw + u[:, k].abs() * egB + (u[:, k] * gB).abs() + dd.abs() + aw.abs()
            m = on[:, k]
            per_step["u"][k] = v * m, ev * m
            sl, esl = slope[:, k], eslope[:, k]
            per_step["delta"][k] = dd * sl * m, (edd * sl + dd.abs() * (esl + sl)) * m
            q = g * dk * uk
            eq = eg * (dk * uk).abs() + ed[:, k, :, None] * (g * uk).abs() + 2 * q.abs()
            r = ek * hs[k + 1]
            er = eek * hs[k + 1].abs() + ek.abs() * ehs[k + 1] + r.abs()
            for name, t, et in (("B", q, eq), ("C", r, er)):
                t, et = t * m[..., None], et * m[..., None]
                shape = (batch, groups, per, n)
                per_step[name][k] = t.view(shape).sum(2), (et + path * t.abs()).view(shape).sum(2)
            if z is not None:
                p, ep = _silu_slope(z[:, k])
                x = dy[:, k] * s_all[k]
                ex = dy[:, k].abs() * es_all[k] * p.abs() + x.abs() * (ep + 2 * p.abs())
                per_step["z"][k] = x * p * m, ex * m
            carry, ecarry = torch.where(live, nc, carry), torch.where(live, enc, ecarry)
        for k, v in per_step.items():
            if k != "z" or z is not None:
                out[k] = tuple(torch.stack([t[i] for t in v], 1) for i in (0, 1))
        out["initial"] = carry, ecarry
        out["A"] = dA.sum(0), (edA + walk + batch * dA.abs()).sum(0)
        # A thread adds up every other position at most, its neighbours and the sequences follow.
        many = length // 2 + 32 + batch
        if D is not None:
            x = e * u
            out["D"] = x.sum((0, 1)), (ee * u.abs() + many * x.abs()).sum((0, 1))
        if bias is not None:
            x, ex = out["delta"]
            out["delta_bias"] = x.sum((0, 1)), (ex + many * x.abs()).sum((0, 1))
    return {k: (v, 1.01 * U * e) for k, (v, e) in out.items()}  # second order


def worst(got, want, bound):
    """The largest error of `got` as a multiple of its bound: the computation's and half a step of its type."""
    t = got.dtype
    half = U if t == torch.float32 else torch.finfo(t).eps / 2
    tol = bound + half * (want.abs() + bound) + torch.finfo(t).tiny * half
    off = (got.detach().double() - want).abs()
    return float((off / tol).max()) if off.numel() else 0.0
