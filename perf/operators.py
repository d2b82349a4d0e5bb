"""Workloads of the state space layer's operators: layer norm, short causal convolution, selective scan.

Each case is one call (or one call with its gradients) of one operator, at sizes from a few tokens
to a training batch.  `run` computes it in plain torch operations, or, with `own` set, through the
package's entry points; `exact` computes it in 64 bits from the definition.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parent.parent / "bs-compiler_b200")
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _basalto():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import basalto
    return basalto


# ---- cases ------------------------------------------------------------------------------
# op: ln | conv | conv_step | scan | scan_step.   grad: the call and the gradients of all its inputs.
# lines: the sequence axis, not the channel axis, is the contiguous one.
# ragged: a batch of sequences of different lengths, padded to the longest.
# carry: a state of an earlier piece of the sequence comes in; the final state is returned.

def listed():
    return [
        # The norm in front of a layer while a handful of sequences decode: latency of one small launch.
        {"name": "ln_token", "op": "ln", "dtype": "fp16", "rows": 5, "dim": 1541, "grad": False, "wide": False},
        # The norm of a training step over 16 K tokens, with the reduction of its weights' gradients.
        {"name": "ln_train", "op": "ln", "dtype": "bf16", "rows": 16384, "dim": 4096, "grad": True, "wide": True},
        # One long prompt through the convolution, its last inputs kept for decoding.
        {"name": "conv_prompt", "op": "conv", "dtype": "bf16", "batch": 1, "length": 8192, "channels": 4096,
         "width": 4, "silu": True, "lines": False, "ragged": False, "carry": True, "grad": False},
        # The convolution of a training step.
        {"name": "conv_train", "op": "conv", "dtype": "bf16", "batch": 4, "length": 4096, "channels": 4096,
         "width": 4, "silu": True, "lines": False, "ragged": False, "carry": False, "grad": True},
        # A padded batch of odd sizes whose sequence axis is contiguous, in 32 bits.
        {"name": "conv_lines", "op": "conv", "dtype": "fp32", "batch": 3, "length": 1021, "channels": 770,
         "width": 3, "silu": False, "lines": True, "ragged": True, "carry": False, "grad": True},
        # One token for each of 64 decoding sequences.
        {"name": "conv_token", "op": "conv_step", "dtype": "bf16", "batch": 64, "channels": 4096, "width": 4,
         "silu": True},
        # One token of one sequence, odd width and channel count.
        {"name": "conv_token_one", "op": "conv_step", "dtype": "fp32", "batch": 1, "channels": 1537, "width": 3,
         "silu": False},
        # One prompt through the scan, its final state kept for decoding.
        {"name": "scan_prompt", "op": "scan", "dtype": "bf16", "batch": 1, "length": 4096, "channels": 4096,
         "states": 16, "groups": 1, "gate": True, "ragged": False, "carry": True, "grad": False},
        # The scan of a training step.
        {"name": "scan_train", "op": "scan", "dtype": "bf16", "batch": 4, "length": 2048, "channels": 4096,
         "states": 16, "groups": 1, "gate": True, "ragged": False, "carry": False, "grad": True},
        # A padded batch of odd sizes that continues from earlier states, in 32 bits, with its gradients.
        {"name": "scan_ragged", "op": "scan", "dtype": "fp32", "batch": 5, "length": 777, "channels": 514,
         "states": 12, "groups": 2, "gate": False, "ragged": True, "carry": True, "grad": True},
        # One token for each of 256 decoding sequences.
        {"name": "scan_token", "op": "scan_step", "dtype": "bf16", "batch": 256, "channels": 4096, "states": 16,
         "groups": 1, "gate": True},
        # One token for each of two sequences, odd sizes.
        {"name": "scan_token_two", "op": "scan_step", "dtype": "fp32", "batch": 2, "channels": 1030, "states": 24,
         "groups": 2, "gate": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST = 4 * 2048 * 4096 * 16  # (batch, length, channel, state) products of the largest scan


def draw(rng):
    op = rng.choice(["ln", "conv", "conv_step", "scan", "scan_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "ln":
        dim = _log(rng, 17, 8192)
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, min(16384, 16384 * 4096 // dim // 2)), "dim": dim,
                "grad": rng.random() < 0.5, "wide": rng.random() < 0.5}
    if op == "conv":
        b, c = _log(rng, 1, 8), _log(rng, 33, 4096)
        length = _log(rng, 1, min(8192, 4 * 4096 * 4096 // (b * c) // 2))
        return {"op": op, "dtype": dtype, "batch": b, "length": length, "channels": c, "width": rng.randint(2, 4),
                "silu": rng.random() < 0.7, "lines": rng.random() < 0.3, "ragged": rng.random() < 0.3,
                "carry": rng.random() < 0.4, "grad": rng.random() < 0.5}
    if op == "conv_step":
        return {"op": op, "dtype": dtype, "batch": _log(rng, 1, 128), "channels": _log(rng, 65, 4096),
                "width": rng.randint(2, 4), "silu": rng.random() < 0.7}
    groups = rng.choice([1, 1, 2])
    n = rng.choice([4, 8, 12, 16, 16, 24, 32, 64])
    if op == "scan":
        b, c = _log(rng, 1, 8), groups * _log(rng, 33, 4096 // groups)
        length = _log(rng, 1, max(1, min(8192, _MOST // (b * c * n) // 2)))
        return {"op": op, "dtype": dtype, "batch": b, "length": length, "channels": c, "states": n,
                "groups": groups, "gate": rng.random() < 0.6, "ragged": rng.random() < 0.3,
                "carry": rng.random() < 0.4, "grad": rng.random() < 0.5}
    return {"op": op, "dtype": dtype, "batch": _log(rng, 1, 128), "channels": groups * _log(rng, 33, 4096 // groups),
            "states": n, "groups": groups, "gate": rng.random() < 0.6}


# ---- inputs -----------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    op = case["op"]
    s = {"case": case}
    if op == "ln":
        m, d = case["rows"], case["dim"]
        # Activations off centre, a few channels an order of magnitude larger than the others.
        gain = 1.0 + 10.0 * (uniform(d) < 0.01).float()
        s["x"] = (normal(m, d, dtype=torch.float32) * gain + 0.3).to(dt)
        wt = torch.float32 if case["wide"] else dt  # parameters in 32 bits or in the activations' type
        s["weight"] = (1.0 + normal(d, dtype=torch.float32, scale=0.1)).to(wt)
        s["bias"] = normal(d, dtype=wt, scale=0.1)
        if case["grad"]:
            s["dy"] = normal(m, d)
    elif op in ("conv", "conv_step"):
        b, c, w = case["batch"], case["channels"], case["width"]
        s["weight"] = normal(c, w, scale=1.0 / math.sqrt(w))
        s["bias"] = normal(c, scale=0.1)
        if op == "conv_step":
            s["x"], s["state"] = normal(b, c), normal(b, w - 1, c)
            s["out_state"] = torch.empty_like(s["state"])
            return s
        length = case["length"]
        # [batch, length, channels], or a transposed [batch, channels, length]
        s["x"] = normal(b, c, length).transpose(1, 2) if case["lines"] else normal(b, length, c)
        s["initial"] = normal(b, w - 1, c) if case["carry"] else None
        if case["grad"]:
            s["dy"] = normal(b, c, length).transpose(1, 2) if case["lines"] else normal(b, length, c)
    else:
        b, c, n, k = case["batch"], case["channels"], case["states"], case["groups"]
        steps = (b, case["length"]) if op == "scan" else (b,)
        s["u"], s["delta"] = normal(*steps, c), normal(*steps, c, scale=0.5)
        s["z"] = normal(*steps, c) if case["gate"] else None
        s["B"], s["C"] = normal(*steps, k, n), normal(*steps, k, n)
        # Decay rates 1..N with learned deviations, step sizes between 1e-3 and 1e-1 at rest.
        rate = torch.arange(1, n + 1, device="cuda", dtype=torch.float32).expand(c, n)
        s["A"] = -rate * torch.exp(normal(c, n, dtype=torch.float32, scale=0.1))
        s["D"] = 1.0 + normal(c, dtype=torch.float32, scale=0.1)
        size = torch.exp(uniform(c) * math.log(100.0) + math.log(1e-3))
        s["delta_bias"] = size + torch.log(-torch.expm1(-size))
        if op == "scan_step":
            s["state"] = normal(b, c, n, dtype=torch.float32)
            s["out_state"] = torch.empty_like(s["state"])
            return s
        s["initial"] = normal(b, c, n, dtype=torch.float32) if case["carry"] else None
        if case["grad"]:
            s["dy"] = normal(*steps, c)
    if op in ("conv", "scan"):
        length = case["length"]
        s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = (uniform(case["batch"]) * (length + 1)).to(torch.int32).clamp_(max=length)
    if case["grad"]:
        for key in ("x", "weight", "bias", "u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial"):
            if s.get(key) is not None:
                s[key].requires_grad_()
    return s


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"ln": _ln, "conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step}[
            state["case"]["op"]](state)


def _own(s):
    basalto = _basalto()
    case = s["case"]
    op = case["op"]
    if op == "conv_step":
        return basalto.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"],
                                        activation="silu" if case["silu"] else None, out_state=s["out_state"])
    if op == "scan_step":
        return basalto.selective_scan_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["state"], D=s["D"],
                                           z=s["z"], delta_bias=s["delta_bias"], delta_softplus=True,
                                           out_state=s["out_state"])
    if op == "ln":
        y, names = basalto.layer_norm(s["x"], s["weight"], s["bias"]), ("x", "weight", "bias")
    elif op == "conv":
        y = basalto.causal_conv(s["x"], s["weight"], s["bias"], activation="silu" if case["silu"] else None,
                                initial_state=s["initial"], lengths=s["lengths"], return_state=case["carry"])
        names = ("x", "weight", "bias", "initial")
    else:
        y = basalto.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                   delta_bias=s["delta_bias"], delta_softplus=True, initial_state=s["initial"],
                                   lengths=s["lengths"], return_state=case["carry"])
        names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial")
    if not case["grad"]:
        return y
    leaves = [k for k in names if s[k] is not None]
    first = y[0] if isinstance(y, tuple) else y
    return y, dict(zip(leaves, torch.autograd.grad(first, [s[k] for k in leaves], s["dy"])))


def _ln(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5)
    xh = c * r
    y = (xh * w + b).to(s["x"].dtype)
    if not s["case"]["grad"]:
        return y
    dy = s["dy"].float()
    gy = dy * w
    dx = r * (gy - gy.mean(-1, keepdim=True) - xh * (gy * xh).mean(-1, keepdim=True))
    return y, {"x": dx.to(s["x"].dtype), "weight": (dy * xh).sum(0).to(s["weight"].dtype),
               "bias": dy.sum(0).to(s["bias"].dtype)}


def _live(s):
    """[batch, length, 1]: true at the positions that a padded batch really has (None: all of them)."""
    if s["lengths"] is None:
        return None
    return (torch.arange(s["case"]["length"], device="cuda") < s["lengths"][:, None])[..., None]


def _conv(s):
    case = s["case"]
    w, b, dt = s["weight"].float(), s["bias"].float(), s["x"].dtype
    width, length, batch = case["width"], case["length"], case["batch"]
    live = _live(s)
    x = s["x"].float()
    left = x.new_zeros(batch, width - 1, x.shape[2]) if s["initial"] is None else s["initial"].float()
    xp = torch.cat([left, x if live is None else torch.where(live, x, 0.0)], 1)  # inputs from -(width-1) on
    seen = xp.unfold(1, width, 1)  # [batch, length, channels, width]
    p = (seen * w).sum(-1) + b
    gate = torch.sigmoid(p) if case["silu"] else None
    y = p * gate if case["silu"] else p
    y = (y if live is None else torch.where(live, y, 0.0)).to(dt)
    out = y
    if case["carry"]:
        ends = torch.full((batch,), length, device="cuda") if s["lengths"] is None else s["lengths"].long()
        rows = ends[:, None] + torch.arange(width - 1, device="cuda")
        out = (y, torch.gather(xp, 1, rows[..., None].expand(-1, -1, xp.shape[2])).to(dt))
    if not case["grad"]:
        return out
    q = s["dy"].float()
    q = q if live is None else torch.where(live, q, 0.0)
    if case["silu"]:
        q = q * gate * (1 + p * (1 - gate))
    qp = torch.nn.functional.pad(q, (0, 0, width - 1, width - 1))
    dxp = (qp.unfold(1, width, 1) * w.flip(-1)).sum(-1)  # gradient of xp
    grads = {"x": dxp[:, width - 1:].to(dt), "weight": (q[..., None] * seen).sum((0, 1)).to(s["weight"].dtype),
             "bias": q.sum((0, 1)).to(s["bias"].dtype)}
    if live is not None:
        grads["x"] = torch.where(live, grads["x"], 0.0)
    if s["initial"] is not None:
        grads["initial"] = dxp[:, :width - 1].to(dt)
    return out, grads


def _conv_step(s):
    seen = torch.cat([s["state"], s["x"][:, None]], 1)  # [batch, width, channels]
    p = (seen.float() * s["weight"].float().t()).sum(1) + s["bias"].float()
    y = p * torch.sigmoid(p) if s["case"]["silu"] else p
    s["out_state"].copy_(seen[:, 1:])
    return y.to(s["x"].dtype), s["out_state"]


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along axis 1, by doubling the reach of every position (b becomes h)."""
    reach = 1
    while reach < a.shape[1]:
        b[:, reach:] += a[:, reach:] * b[:, :-reach]
        a[:, reach:] = a[:, reach:] * a[:, :-reach]
        reach *= 2
    return b


def _scan(s):
    case = s["case"]
    dt, live = s["u"].dtype, _live(s)
    batch, length, channels = s["u"].shape
    k, n = case["groups"], case["states"]
    u, A, D = s["u"].float(), s["A"], s["D"]
    raw = s["delta"].float() + s["delta_bias"]
    delta = _softplus(raw)
    if live is not None:  # a step of size zero leaves the state as it is
        delta = torch.where(live, delta, 0.0)
    Bx = s["B"].float().repeat_interleave(channels // k, 2)  # [batch, length, channels, states]
    Cx = s["C"].float().repeat_interleave(channels // k, 2)
    a = torch.exp(delta[..., None] * A)
    h = (delta * u)[..., None] * Bx
    if s["initial"] is not None:
        h[:, 0] += a[:, 0] * s["initial"]
    h = _recurrence(a.clone(), h)
    sums = (h * Cx).sum(-1) + D * u
    gate = torch.sigmoid(s["z"].float()) if case["gate"] else None
    y = sums * s["z"].float() * gate if case["gate"] else sums
    y = (y if live is None else torch.where(live, y, 0.0)).to(dt)
    out = (y, h[:, -1].clone()) if case["carry"] else y
    if not case["grad"]:
        return out
    dy = s["dy"].float()
    dy = dy if live is None else torch.where(live, dy, 0.0)
    grads = {}
    e = dy
    if case["gate"]:
        zf = s["z"].float()
        grads["z"] = (dy * sums * gate * (1 + zf * (1 - gate))).to(dt)
        e = dy * zf * gate
    grads["C"] = (e[..., None] * h).view(batch, length, k, channels // k, n).sum(3).to(dt)
    # The adjoint runs backwards: g[t] = C[t] e[t] + a[t+1] g[t+1].
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    g = _recurrence(later, (e[..., None] * Cx).flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if s["initial"] is None else s["initial"][:, None]
    carried = g * a * torch.cat([first, h[:, :-1]], 1)
    gB = (g * Bx).sum(-1)
    grads["B"] = (g * (delta * u)[..., None]).view(batch, length, k, channels // k, n).sum(3).to(dt)
    grads["u"] = (delta * gB + D * e).to(dt)
    ddelta = ((carried * A).sum(-1) + gB * u) * torch.sigmoid(raw)
    ddelta = ddelta if live is None else torch.where(live, ddelta, 0.0)
    grads["delta"] = ddelta.to(dt)
    grads["delta_bias"] = ddelta.sum((0, 1))
    grads["A"] = (carried * delta[..., None]).sum((0, 1))
    grads["D"] = (e * u).sum((0, 1))
    if s["initial"] is not None:
        grads["initial"] = (g[:, 0] * a[:, 0]).clone()
    return out, {key: grads[key] for key in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial")
                 if key in grads}


def _scan_step(s):
    case = s["case"]
    per = s["u"].shape[1] // case["groups"]
    u = s["u"].float()
    delta = _softplus(s["delta"].float() + s["delta_bias"])
    B, C = s["B"].float().repeat_interleave(per, 1), s["C"].float().repeat_interleave(per, 1)
    h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * u)[..., None] * B
    y = (h * C).sum(-1) + s["D"] * u
    if case["gate"]:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    s["out_state"].copy_(h)
    return y.to(s["u"].dtype), s["out_state"]


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "ln":
        m, d = case["rows"], case["dim"]
        w = 4 if case["wide"] else e
        if case["grad"]:  # x, dy in; y, dx out
            return {"bytes": 4 * m * d * e + 4 * d * w, "flops": 20 * m * d}
        return {"bytes": 2 * m * d * e + 2 * d * w, "flops": 8 * m * d}
    if op == "conv_step":
        b, c, w = case["batch"], case["channels"], case["width"]
        return {"bytes": (2 * b * c * w + c * (w + 1)) * e, "flops": b * c * (2 * w + 6)}
    if op == "conv":
        b, n, c, w = case["batch"], case["length"], case["channels"], case["width"]
        edge = 2 * b * (w - 1) * c * e if case["carry"] else 0
        if case["grad"]:
            return {"bytes": 4 * b * n * c * e + 2 * c * (w + 1) * e + edge, "flops": b * n * c * (6 * w + 14)}
        return {"bytes": 2 * b * n * c * e + c * (w + 1) * e + edge, "flops": b * n * c * (2 * w + 6)}
    b, c, n, k = case["batch"], case["channels"], case["states"], case["groups"]
    gate = 1 if case["gate"] else 0
    if op == "scan_step":
        return {"bytes": 8 * b * c * n + b * c * (3 + gate) * e + 2 * b * k * n * e + c * n * 4 + c * 8,
                "flops": b * c * (8 * n + 12)}
    t = b * case["length"]
    edge = 8 * b * c * n if case["carry"] else 0
    params = c * n * 4 + c * 8
    if case["grad"]:  # u, delta, dy (z) in; y, du, ddelta (dz) out; B, C in, dB, dC out
        return {"bytes": t * c * (6 + 2 * gate) * e + 4 * t * k * n * e + 2 * params + edge,
                "flops": t * c * (30 * n + 30)}
    return {"bytes": t * c * (3 + gate) * e + 2 * t * k * n * e + params + edge, "flops": t * c * (8 * n + 12)}


# ---- the definition in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    s = {k: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v
         for k, v in prepare(case, seed).items()}
    with torch.no_grad():
        return {"ln": _exact_ln, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
                "scan_step": _exact_scan_step}[case["op"]](case, s)


def _exact_ln(case, s):
    x = s["x"]
    d = x.shape[1]
    mean = x.sum(1) / d
    var = ((x - mean[:, None]) ** 2).sum(1) / d
    sd = (var + 1e-5).sqrt()
    xh = (x - mean[:, None]) / sd[:, None]
    y = s["weight"] * xh + s["bias"]
    if not case["grad"]:
        return y
    f = s["dy"] * s["weight"]
    dot = torch.einsum("md,md->m", f, xh)
    dx = (f - (f.sum(1) / d)[:, None] - xh * (dot / d)[:, None]) / sd[:, None]
    return y, {"x": dx, "weight": torch.einsum("md,md->d", s["dy"], xh), "bias": s["dy"].sum(0)}


def _exact_conv(case, s):
    x, w = s["x"].contiguous(), s["weight"]
    batch, length, channels = x.shape
    width = case["width"]
    lens = [length] * batch if s["lengths"] is None else s["lengths"].tolist()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    final, dfirst = x.new_zeros(batch, width - 1, channels), x.new_zeros(batch, width - 1, channels)
    dw, db = torch.zeros_like(w), torch.zeros_like(s["bias"])
    for i in range(batch):
        m = lens[i]
        past = s["initial"][i] if s["initial"] is not None else x.new_zeros(width - 1, channels)
        line = torch.cat([past, x[i, :m]])
        p = s["bias"].expand(m, channels).clone()
        for j in range(width):
            p += w[:, j] * line[j:j + m]
        sg = 1 / (1 + torch.exp(-p))
        y[i, :m] = p * sg if case["silu"] else p
        final[i] = line[m:]
        if case["grad"]:
            q = s["dy"][i, :m]
            if case["silu"]:
                q = q * (sg + p * sg * (1 - sg))
            dline = torch.zeros_like(line)
            for j in range(width):
                dline[j:j + m] += w[:, j] * q
                dw[:, j] += (q * line[j:j + m]).sum(0)
            db += q.sum(0)
            dfirst[i], dx[i, :m] = dline[:width - 1], dline[width - 1:]
    out = (y, final) if case["carry"] else y
    if not case["grad"]:
        return out
    grads = {"x": dx, "weight": dw, "bias": db}
    if s["initial"] is not None:
        grads["initial"] = dfirst
    return out, grads


def _exact_conv_step(case, s):
    p = s["bias"] + s["x"] * s["weight"][:, -1]
    for j in range(case["width"] - 1):
        p = p + s["state"][:, j] * s["weight"][:, j]
    y = p / (1 + torch.exp(-p)) if case["silu"] else p
    return y, torch.cat([s["state"][:, 1:], s["x"][:, None]], 1)


def _exact_scan(case, s):
    batch, length, channels = s["u"].shape
    n, k = case["states"], case["groups"]
    per = channels // k
    if batch * length * channels * n * 8 > 30e9 or length > 20000:
        return None
    raw = s["delta"] + s["delta_bias"]
    delta = torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0)
    lens = torch.full((batch,), length, device="cuda") if s["lengths"] is None else s["lengths"].long()
    on = [(t < lens).double()[:, None] for t in range(length)]  # [batch, 1] for each step
    h = s["initial"].clone() if s["initial"] is not None else s["u"].new_zeros(batch, channels, n)
    kept = s["u"].new_empty(length if case["grad"] else 0, batch, channels, n)  # the state before each step
    total = torch.empty_like(s["u"])

    def spread(v):  # [batch, groups, states] -> [batch, channels, states]
        return v[:, :, None].expand(batch, k, per, n).reshape(batch, channels, n)

    for t in range(length):
        if case["grad"]:
            kept[t] = h
        step = delta[:, t] * on[t]
        h = torch.exp(step[..., None] * s["A"]) * h + (step * s["u"][:, t])[..., None] * spread(s["B"][:, t])
        total[:, t] = torch.einsum("bcn,bcn->bc", h, spread(s["C"][:, t])) + s["D"] * s["u"][:, t]
    valid = torch.stack(on, 1)
    sg = 1 / (1 + torch.exp(-s["z"])) if case["gate"] else None
    y = (total * s["z"] * sg if case["gate"] else total) * valid
    out = (y, h) if case["carry"] else y
    if not case["grad"]:
        return out
    dy = s["dy"] * valid
    e = dy * s["z"] * sg if case["gate"] else dy
    r = {key: torch.zeros_like(s[key]) for key in ("u", "delta", "A", "B", "C")}
    g = torch.zeros_like(h)
    for t in reversed(range(length)):
        step = delta[:, t] * on[t]
        a = torch.exp(step[..., None] * s["A"])
        Bt, ut, before = spread(s["B"][:, t]), s["u"][:, t], kept[t]
        now = a * before + (step * ut)[..., None] * Bt
        g = g + e[:, t][..., None] * spread(s["C"][:, t])
        r["C"][:, t] = (e[:, t][..., None] * now).view(batch, k, per, n).sum(2)
        r["B"][:, t] = (g * (step * ut)[..., None]).view(batch, k, per, n).sum(2)
        gB = torch.einsum("bcn,bcn->bc", g, Bt)
        through = g * a * before
        r["u"][:, t] = gB * step + s["D"] * e[:, t]
        r["delta"][:, t] = (torch.einsum("bcn,cn->bc", through, s["A"]) + gB * ut) * on[t]
        r["A"] += (through * step[..., None]).sum(0)
        g = a * g
    r["delta"] /= 1 + torch.exp(-raw)
    r["D"] = (e * s["u"]).sum((0, 1))
    if case["gate"]:
        r["z"] = dy * total * (sg + s["z"] * sg * (1 - sg))
    r["delta_bias"] = r["delta"].sum((0, 1))
    if s["initial"] is not None:
        r["initial"] = g
    return out, {key: r[key] for key in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial") if key in r}


def _exact_scan_step(case, s):
    batch, channels = s["u"].shape
    per = channels // case["groups"]
    which = torch.arange(channels, device="cuda") // per
    raw = s["delta"] + s["delta_bias"]
    delta = torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0)
    h = s["state"] * torch.exp(torch.einsum("bc,cn->bcn", delta, s["A"]))
    h = h + torch.einsum("bc,bcn->bcn", delta * s["u"], s["B"][:, which])
    y = torch.einsum("bcn,bcn->bc", h, s["C"][:, which]) + s["D"] * s["u"]
    if case["gate"]:
        y = y * s["z"] / (1 + torch.exp(-s["z"]))
    return y, h
