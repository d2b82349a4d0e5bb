"""Layer operators on the GPU against the 64-bit reference, at the sizes, layouts and masks where they can go wrong.

Tolerances: half a step of the output's type relative to the value, plus a multiple of u = 2^-24 of the
reference's absolute sums (layer_reference): the roundings on the longest path from an input to the output.
"""
import numpy as np
import pytest
import torch

import basalto
import layer_reference as R

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def make(rng, *shape, dtype=torch.float32, scale=1.0):
    """(CUDA tensor, the same values in float64)"""
    t = torch.from_numpy(rng.standard_normal(shape) * scale).to(dtype)
    return t.cuda(), t.double().numpy()


def close(got, want, mag, k, what=""):
    """got is within half a step of its type of want + k u mag."""
    t = got.dtype
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    slack = k * R.U * mag
    half = torch.finfo(t).eps / 2 if t != torch.float32 else R.U
    tol = half * (np.abs(want) + slack) + slack + torch.finfo(t).tiny * half
    off = np.abs(g - want)
    assert np.isfinite(g).all(), what
    assert (off <= tol).all(), (what, float((off / np.maximum(tol, 1e-300)).max()))


# ---- layer norm --------------------------------------------------------------------------------
# y: mean and variance are sums of at most 16 terms in a row per thread and 10 levels across threads (long rows:
# dim / 1024 in a row), a division, a root and five more operations: 64.  dx has one more pair of such sums: 128.
# dw, db: at most rows / 8 terms in a row here, then 32 rows' worth of partial sums: 128 covers 1031 rows.
NORM = [  # rows, dim
    (1, 1), (1, 17), (3, 512), (5, 513), (2, 1541), (37, 2048), (9, 4104), (4, 8192), (3, 16384), (2, 16400), (3, 20011),
    (1031, 96), (700, 1030),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,dim", NORM)
def test_layer_norm(dtype, rows, dim):
    rng = np.random.default_rng(rows * 100003 + dim)
    dt = DT[dtype]
    wide = torch.float32 if rows % 2 else dt
    x, xr = make(rng, rows, dim, dtype=dt)
    w, wr = make(rng, dim, dtype=wide)
    b, br = make(rng, dim, dtype=wide)
    dy, dr = make(rng, rows, dim, dtype=dt)
    for t in (x, w, b):
        t.requires_grad_()
    y = basalto.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want, mag, grads, mags = R.layer_norm(xr, wr, br, 1e-5, dr)
    if dim == 1:  # x - mean is exactly zero
        assert torch.equal(y.detach(), b.detach().to(dt).expand(rows, 1)) and (dx == 0).all() and (dw == 0).all()
        return
    close(y, want, mag, 64, "y")
    close(dx, grads[0], mags[0], 128, "dx")
    close(dw, grads[1], mags[1], 128, "dw")
    close(db, grads[2], mags[2], 128, "db")
    with torch.no_grad():
        assert torch.equal(basalto.layer_norm(x, w, b), y)


def test_layer_norm_options_and_layouts():
    rng = np.random.default_rng(5)
    big, br = make(rng, 4, 6, 80, dtype=torch.bfloat16)
    x, xr = big[:, :, 8:72], br[:, :, 8:72]  # rows 80 apart, aligned
    close(basalto.layer_norm(x), *R.layer_norm(xr, 1.0, np.zeros(64), 1e-5), 64)
    x, xr = big[:, :, 3:67], br[:, :, 3:67]  # not aligned
    close(basalto.layer_norm(x, eps=0.5), *R.layer_norm(xr, 1.0, np.zeros(64), 0.5), 64)
    x, xr = big.transpose(0, 2), br.swapaxes(0, 2)  # last axis not contiguous
    close(basalto.layer_norm(x), *R.layer_norm(xr, 1.0, np.zeros(4), 1e-5), 64)
    w, wr = make(rng, 80)
    leaf = w.clone().requires_grad_()
    y = basalto.layer_norm(big, leaf)  # no bias, weight in 32 bits, x without gradient
    want, mag, grads, mags = R.layer_norm(br, wr, np.zeros(80), 1e-5, np.ones_like(br))
    close(y, want, mag, 64)
    close(torch.autograd.grad(y.sum(), leaf)[0], grads[1], mags[1], 128)  # an expanded gradient (strides 0)
    bias = torch.zeros(80, device="cuda", requires_grad=True)
    y = basalto.layer_norm(big, None, bias)
    close(torch.autograd.grad(y.sum(), bias)[0], grads[2], mags[2], 128)
    one = torch.full((2, 33), 3.0, device="cuda")  # a constant row: xh = 0
    assert (basalto.layer_norm(one) == 0).all()
    for shape in ((0, 8), (3, 0), (2, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y = basalto.layer_norm(x, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and (dw == 0).all()


def test_layer_norm_keeps_nan_and_inf_in_their_rows():
    x = torch.randn(5, 300, device="cuda")
    clean = basalto.layer_norm(x)
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    y = basalto.layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).any()
    assert torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


# ---- causal convolution ------------------------------------------------------------------------
# p: width + 1 fused operations (9 at most), silu 12 more: 32.  Gradients: q as p and 12, width products: 48.  Their
# sums over positions: at most 128 in a row per piece and a reduction over the pieces of 64 roundings: 256.
CONV = [  # batch, length, channels, width, silu, lengths, carry
    (2, 37, 40, 4, True, None, False),
    (1, 1, 8, 4, True, None, True),
    (3, 2, 24, 4, False, [2, 0, 1], True),
    (2, 130, 17, 3, True, [129, 64], True),
    (2, 67, 33, 2, False, None, False),
    (1, 100, 16, 1, True, None, True),
    (1, 75, 12, 8, True, [70], True),
    (4, 40, 64, 4, True, [40, 99, -3, 17], True),  # clamped to [0, 40]
    (1, 1500, 9, 5, False, None, False),
    (2, 1300, 16, 4, True, [1300, 1025], True),
]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("lines", [False, True])
@pytest.mark.parametrize("case", range(len(CONV)))
def test_causal_conv(dtype, lines, case):
    b, l, c, w, silu, lens, carry = CONV[case]
    rng = np.random.default_rng(case)
    dt = DT[dtype]
    x, xr = make(rng, b, l, c, dtype=dt)
    dy, dr = make(rng, b, l, c, dtype=dt)
    if lines:
        x, dy = x.transpose(1, 2).contiguous().transpose(1, 2), dy.transpose(1, 2).contiguous().transpose(1, 2)
    wt = torch.float32 if case % 2 else dt
    wg, wr = make(rng, c, w, dtype=wt, scale=0.5)
    bg, br = make(rng, c, dtype=wt)
    init, ir = make(rng, b, w - 1, c, dtype=dt) if carry else (None, None)
    df, dfr = make(rng, b, w - 1, c, dtype=dt) if carry else (None, None)
    lg = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    if lens is not None:  # what lies behind a sequence is not read
        for i, n in enumerate(lens):
            x[i, max(n, 0):] = float("nan")
            dy[i, max(n, 0):] = float("inf")
            xr[i, max(n, 0):] = 0
            dr[i, max(n, 0):] = 0
    leaves = [t.requires_grad_() for t in (x, wg, bg, init) if t is not None]
    got = basalto.causal_conv(x, wg, bg, "silu" if silu else None, init, lg, return_state=carry)
    y, final = got if carry else (got, None)
    out, mag = R.causal_conv(xr, wr, br, silu, ir, lens, dr, dfr)
    grads = torch.autograd.grad([y, final] if carry else [y], leaves, [dy, df] if carry else [dy])
    close(y, out["y"], mag["y"], 32, "y")
    assert y.stride() == x.stride() or l == 1 or c == 1
    if carry:
        close(final, out["final"], mag["final"], 0, "final")
    for name, g, k in zip(("x", "weight", "bias", "initial"), grads, (48, 256, 256, 48)):
        close(g, out[name], mag[name], k, name)


def test_causal_conv_layouts():
    rng = np.random.default_rng(11)
    big, br = make(rng, 2, 30, 80, dtype=torch.bfloat16)
    w, wr = make(rng, 32, 4, dtype=torch.bfloat16)
    for lo in (0, 8, 5):  # a slice of a wider projection: aligned and not
        x, xr = big[..., lo:lo + 32], br[..., lo:lo + 32]
        out, mag = R.causal_conv(xr, wr, np.zeros(32), True)
        close(basalto.causal_conv(x, w, activation="silu"), out["y"], mag["y"], 32)
    x, xr = big[:, ::2, ::2][..., :32], br[:, ::2, ::2][..., :32]  # neither axis contiguous
    out, mag = R.causal_conv(xr, wr, np.zeros(32), False)
    close(basalto.causal_conv(x, w), out["y"], mag["y"], 32)
    xs = big[0, :, :32].expand(3, 30, 32)  # one sequence for the whole batch (stride 0), and its gradient
    leaf = big[0, :, :32].clone().requires_grad_()
    y = basalto.causal_conv(leaf.expand(3, 30, 32), w)
    out, mag = R.causal_conv(np.repeat(br[:1, :, :32], 3, 0), wr, np.zeros(32), False, dy=np.ones((3, 30, 32)))
    close(y, out["y"], mag["y"], 32)
    g = torch.autograd.grad(y.float().sum(), leaf)[0]
    # three equal gradients, each rounded to bf16 and then summed by autograd in bf16: 3 more half steps
    want = out["x"].sum(0)
    assert (np.abs(g.double().cpu().numpy() - want) <= 2.0 ** -8 * 6 * (np.abs(want) + 1e-3) + 1e-2).all()
    assert torch.equal(basalto.causal_conv(xs, w)[1], basalto.causal_conv(xs[:1], w)[0])
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w0 = torch.zeros(shape[2], 4, device="cuda", requires_grad=True)
        init = torch.ones(shape[0], 3, shape[2], device="cuda", requires_grad=True)
        y, final = basalto.causal_conv(x, w0, initial_state=init, return_state=True)
        assert y.shape == x.shape and torch.equal(final, init) or 0 not in (shape[1],)
        gx, gw, gi = torch.autograd.grad([y.sum(), final.sum()], (x, w0, init))
        assert gx.shape == x.shape and (gw == 0).all() and gi.shape == init.shape


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("b,c,w,silu", [(1, 1, 1, True), (1, 1537, 3, False), (5, 40, 2, True), (64, 4096, 4, True),
                                        (3, 24, 8, True), (7, 129, 4, True)])
def test_causal_conv_step(dtype, b, c, w, silu):
    rng = np.random.default_rng(b + c)
    dt = DT[dtype]
    x, xr = make(rng, b, c, dtype=dt)
    s, sr = make(rng, b, w - 1, c, dtype=dt)
    wg, wr = make(rng, c, w, dtype=dt, scale=0.5)
    bg, br = make(rng, c, dtype=dt)
    act = "silu" if silu else None
    out, mag = R.causal_conv(xr[:, None], wr, br, silu, sr)
    other = torch.empty_like(s)
    y, new = basalto.causal_conv_step(x, s, wg, bg, act, out_state=other)
    assert new is other
    close(y, out["y"][:, 0], mag["y"][:, 0], 32)
    close(new, out["final"], mag["final"], 0)
    assert np.array_equal(s.double().cpu().numpy(), sr)  # untouched
    pool = torch.full((b, 2, w - 1, c), 7.0, dtype=dt, device="cuda")  # a slice of a layer-major pool, in place
    pool[:, 1] = s
    y2, new = basalto.causal_conv_step(x, pool[:, 1], wg, bg, act)
    assert torch.equal(y2, y) and torch.equal(pool[:, 1], other) and (pool[:, 0] == 7).all()


# ---- selective scan ----------------------------------------------------------------------------
SCAN = [  # batch, length, channels, states, groups, gate, D, bias, softplus, lengths, carry
    (2, 37, 40, 16, 1, True, True, True, True, None, False),
    (1, 1, 1, 1, 1, False, False, False, False, None, True),
    (2, 16, 64, 16, 1, True, True, True, True, None, True),
    (3, 50, 34, 12, 2, False, True, True, True, [50, 0, 17], True),
    (1, 33, 66, 4, 1, True, True, False, True, None, True),
    (2, 20, 30, 5, 3, False, False, True, True, [7, 20], False),
    (1, 64, 24, 64, 2, True, True, True, True, None, True),
    (2, 19, 18, 32, 1, False, True, False, False, None, False),
    (4, 48, 16, 16, 4, True, True, True, True, [48, 99, -1, 33], True),
    (1, 200, 8, 16, 1, True, True, True, True, None, False),
    (2, 40, 7, 17, 1, True, False, True, True, [40, 16], True),
    (1, 18, 136, 8, 1, True, True, True, True, None, True),
]
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial")


def scan_inputs(case, dt):
    b, l, c, n, g, gate, skip, bias, softplus, lens, carry = SCAN[case]
    rng = np.random.default_rng(case + 50)
    t, r = {}, {}
    for k, shape, on, d, s in (("u", (b, l, c), True, dt, 1), ("delta", (b, l, c), True, dt, 0.5),
                               ("B", (b, l, g, n), True, dt, 1), ("C", (b, l, g, n), True, dt, 1),
                               ("D", (c,), skip, torch.float32, 1), ("z", (b, l, c), gate, dt, 1),
                               ("initial", (b, c, n), carry, torch.float32, 1), ("dy", (b, l, c), True, dt, 1),
                               ("dfinal", (b, c, n), carry, torch.float32, 1)):
        t[k], r[k] = make(rng, *shape, dtype=d, scale=s) if on else (None, None)
    a = torch.from_numpy(-np.exp(rng.uniform(-3, 1, (c, n)))).float()
    t["A"], r["A"] = a.cuda(), a.double().numpy()
    db = torch.from_numpy(rng.uniform(-6, -1, c)).float()
    t["delta_bias"], r["delta_bias"] = (db.cuda(), db.double().numpy()) if bias else (None, None)
    if not softplus:
        t["delta"], r["delta"] = t["delta"].abs(), np.abs(r["delta"])
    t["lengths"] = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    if lens is not None:  # nothing behind a sequence is read
        for i, m in enumerate(lens):
            for k in ("u", "delta", "z", "dy", "B", "C"):
                if t[k] is not None:
                    t[k][i, max(m, 0):] = float("nan")
                    r[k][i, max(m, 0):] = 0
    return t, r, softplus, lens, carry


def call_scan(t, softplus, carry):
    return basalto.selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["delta_bias"], softplus,
                                  t["initial"], t["lengths"], carry)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(SCAN)))
def test_selective_scan(dtype, case):
    t, r, softplus, lens, carry = scan_inputs(case, DT[dtype])
    leaves = {k: t[k].requires_grad_() for k in NAMES if t[k] is not None}
    got = call_scan(t, softplus, carry)
    y, final = got if carry else (got, None)
    grads = torch.autograd.grad([y, final] if carry else [y], list(leaves.values()),
                                [t["dy"], t["dfinal"]] if carry else [t["dy"]])
    out, mag, steps = R.selective_scan(r["u"], r["delta"], r["A"], r["B"], r["C"], r["D"], r["z"], r["delta_bias"],
                                       softplus, r["initial"], lens, r["dy"], r["dfinal"])
    k = R.scan_tolerance(r["u"].shape[1], steps, r["z"])
    close(y, out["y"], mag["y"], k, "y")
    if carry:
        close(final, out["final"], mag["final"], k, "final")
    for name, g in zip(leaves, grads):
        close(g, out[name], mag[name], 2 * k, name)  # a factor exp(d A) of the states and one of the adjoint
    with torch.no_grad():
        again = call_scan(t, softplus, carry)
    assert torch.equal(again[0] if carry else again, y)


@pytest.mark.parametrize("batch,channels,length", [(1, 64, 700), (1, 16, 3000), (2, 520, 260)])
def test_long_scans(batch, channels, length):
    """Lengths and widths where work is split along the sequence, against the same scan in short pieces."""
    rng = np.random.default_rng(length)
    n = 16
    u, ur = make(rng, batch, length, channels, dtype=torch.bfloat16)
    d, dr = make(rng, batch, length, channels, dtype=torch.bfloat16, scale=0.5)
    z, zr = make(rng, batch, length, channels, dtype=torch.bfloat16)
    B, Br = make(rng, batch, length, 1, n, dtype=torch.bfloat16)
    C, Cr = make(rng, batch, length, 1, n, dtype=torch.bfloat16)
    dy, gr = make(rng, batch, length, channels, dtype=torch.bfloat16)
    A = torch.from_numpy(-np.exp(rng.uniform(-2, 1, (channels, n)))).float()
    D, Dr = make(rng, channels)
    bias = torch.full((channels,), -3.0)
    init, ir = make(rng, batch, channels, n)
    lens = [length - 5 * i - 1 for i in range(batch)]
    lg = torch.tensor(lens, dtype=torch.int32, device="cuda")
    Ag, bg = A.cuda(), bias.cuda()
    leaves = [t.requires_grad_() for t in (u, d, Ag, B, C, D, z, bg, init)]
    y, final = basalto.selective_scan(u, d, Ag, B, C, D, z, bg, True, init, lg, True)
    df, dfr = make(rng, batch, channels, n)
    grads = torch.autograd.grad([y, final], leaves, [dy, df])
    out, mag, steps = R.selective_scan(ur, dr, A.double().numpy(), Br, Cr, Dr, zr, bias.double().numpy(), True, ir, lens,
                                       gr, dfr)
    # A contribution has decayed to nothing long before it crosses all positions: with steps of at least e^-6 and
    # rates of at least e^-2 a factor of e^-16 is reached after 50000 / 1 positions only, so all positions count.
    k = R.scan_tolerance(length, steps, zr)
    close(y, out["y"], mag["y"], k, "y")
    close(final, out["final"], mag["final"], k, "final")
    for name, g in zip(NAMES, grads):
        close(g, out[name], mag[name], 2 * k, name)


def test_scan_layouts():
    """Slices of wider projections, [b, l, n] without a group axis, expanded inputs, unaligned starts."""
    rng = np.random.default_rng(3)
    b, l, c, n = 2, 21, 24, 8
    wide, wr = make(rng, b, l, 2 * c + 3, dtype=torch.bfloat16)
    proj, pr = make(rng, b, l, 2 * n + 5, dtype=torch.bfloat16)
    A = torch.from_numpy(-np.exp(rng.uniform(-2, 1, (c, n)))).float()
    for lo in (0, 3):
        u, z, B, C = wide[..., lo:lo + c], wide[..., lo + c:lo + 2 * c], proj[..., 5:5 + n], proj[..., 5 + n:]
        y = basalto.selective_scan(u, u, A.cuda(), B, C, z=z, delta_softplus=True)
        ur, zr = wr[..., lo:lo + c], wr[..., lo + c:lo + 2 * c]
        out, mag, steps = R.selective_scan(ur, ur, A.double().numpy(), pr[:, :, None, 5:5 + n], pr[:, :, None, 5 + n:],
                                           z=zr, softplus_on=True)
        close(y, out["y"], mag["y"], R.scan_tolerance(l, steps, zr))
        full = basalto.selective_scan(u.contiguous(), u.contiguous(), A.cuda(), B.contiguous(), C.contiguous(),
                                      z=z.contiguous(), delta_softplus=True)
        assert torch.equal(full, y)
    u = wide[..., :c]
    Be = proj[:1, :, 5:5 + n].expand(b, l, n)  # one B for the whole batch
    same = basalto.selective_scan(u, u, A.cuda(), Be, Be, delta_softplus=True)
    assert torch.equal(same, basalto.selective_scan(u, u, A.cuda(), Be.contiguous(), Be.contiguous(),
                                                    delta_softplus=True))
    ut = u.transpose(1, 2).contiguous().transpose(1, 2)  # sequence axis contiguous: copied
    assert torch.equal(basalto.selective_scan(ut, u, A.cuda(), Be, Be, delta_softplus=True), same)
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        u = torch.zeros(shape, device="cuda", requires_grad=True)
        A0 = torch.zeros(shape[2], 4, device="cuda", requires_grad=True)
        B0 = torch.zeros(*shape[:2], 4, device="cuda")
        h0 = torch.ones(shape[0], shape[2], 4, device="cuda", requires_grad=True)
        y, final = basalto.selective_scan(u, u, A0, B0, B0, initial_state=h0, return_state=True)
        assert y.shape == u.shape and torch.equal(final, h0)
        gu, gA, gh = torch.autograd.grad([y.sum(), final.sum()], (u, A0, h0))
        assert gu.shape == u.shape and (gA == 0).all() and (gh == 1).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("b,c,n,g,gate,full", [(1, 1, 1, 1, False, False), (2, 1030, 24, 2, False, True),
                                               (5, 48, 16, 1, True, True), (3, 33, 5, 3, True, False),
                                               (2, 64, 64, 1, True, True), (7, 40, 8, 4, False, True)])
def test_selective_scan_step(dtype, b, c, n, g, gate, full):
    rng = np.random.default_rng(b * c)
    dt = DT[dtype]
    u, ur = make(rng, b, c, dtype=dt)
    d, dr = make(rng, b, c, dtype=dt)
    B, Br = make(rng, b, g, n, dtype=dt)
    C, Cr = make(rng, b, g, n, dtype=dt)
    z, zr = make(rng, b, c, dtype=dt) if gate else (None, None)
    h, hr = make(rng, b, c, n)
    A = torch.from_numpy(-np.exp(rng.uniform(-3, 1, (c, n)))).float()
    D, Dr = make(rng, c) if full else (None, None)
    bias, biasr = make(rng, c) if full else (None, None)
    out, mag, steps = R.selective_scan(ur[:, None], dr[:, None], A.double().numpy(), Br[:, None], Cr[:, None], Dr,
                                       None if zr is None else zr[:, None], biasr, True, hr)
    k = R.scan_tolerance(1, steps, zr)
    other = torch.empty_like(h)
    y, new = basalto.selective_scan_step(u, d, A.cuda(), B, C, h, D, z, bias, True, out_state=other)
    assert new is other and np.array_equal(h.double().cpu().numpy(), hr)
    close(y, out["y"][:, 0], mag["y"][:, 0], k)
    close(new, out["final"], mag["final"], k)
    pool = torch.full((b, 2, c, n + 3), 7.0, device="cuda")
    pool[:, 1, :, :n] = h
    y2, _ = basalto.selective_scan_step(u, d, A.cuda(), B, C, pool[:, 1, :, :n], D, z, bias, True)
    close(y2, out["y"][:, 0], mag["y"][:, 0], k)
    close(pool[:, 1, :, :n], out["final"], mag["final"], k)
    assert (pool[:, 0] == 7).all() and (pool[:, 1, :, n:] == 7).all()


def test_extreme_values():
    """Steps that overflow the exponential either way, zero steps, and NaN that must not vanish."""
    c, n = 8, 4
    A = -torch.ones(c, n, device="cuda")
    B = torch.ones(1, 3, n, device="cuda")
    u = torch.ones(1, 3, c, device="cuda")
    big = torch.full((1, 3, c), 1e4, device="cuda")
    assert (basalto.selective_scan(u, big, A, B, B, delta_softplus=True) == 1e4 * n).all()  # exp(-1e4) = 0
    assert (basalto.selective_scan(u, -big, A, B, B, delta_softplus=True) == 0).all()  # softplus(-1e4) = 0
    y, h = basalto.selective_scan(u, -big, A, B, B, return_state=True)  # exp(+1e4) = inf, as the definition says
    assert torch.isnan(y[0, 2]).all() or torch.isinf(y[0, 2]).all()
    zero = torch.zeros(1, 3, c, device="cuda")
    h0 = torch.randn(1, c, n, device="cuda")
    y, h = basalto.selective_scan(u, zero, A, B, B, initial_state=h0, return_state=True)
    assert torch.equal(h, h0)
    for k in range(3):
        parts = [u.clone(), zero.clone() + 0.1, B.clone()]
        parts[k][0, 1, 0] = float("nan")
        y = basalto.selective_scan(parts[0], parts[1], A, parts[2], B)
        assert torch.isfinite(y[0, 0]).all() and torch.isnan(y[0, 1:, 0]).all()
    z = torch.tensor([-1e4, -200.0, 0.0, 200.0, 1e4, 1.0, -1.0, 30.0], device="cuda").expand(1, 3, c)
    y = basalto.selective_scan(u, zero, A, B, B, D=torch.ones(c, device="cuda"), z=z)
    want = torch.nn.functional.silu(z.double())
    assert (y.double() - want).abs().max() <= 1e-5 * 1e4 and torch.isfinite(y).all()
    w = torch.ones(c, 1, device="cuda")
    assert torch.isfinite(basalto.causal_conv(z.contiguous(), w, activation="silu")).all()


# ---- refusals that need a device ---------------------------------------------------------------
def test_step_refusals():
    x, s, w = torch.zeros(2, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    with pytest.raises(ValueError, match="state"):
        basalto.causal_conv_step(x, s[:, :2], w)
    with pytest.raises(ValueError, match="contiguous"):
        basalto.causal_conv_step(x, torch.zeros(2, 8, 3, device="cuda").transpose(1, 2), w)
    with pytest.raises(ValueError, match="one address"):
        basalto.causal_conv_step(x, s[:1].expand(2, 3, 8), w)
    pool = torch.zeros(3, 3, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        basalto.causal_conv_step(x, pool[:2], w, out_state=pool[1:])
    with pytest.raises(RuntimeError, match="differentiable"):
        basalto.causal_conv_step(x.clone().requires_grad_(), s, w)
    A, B, h = torch.zeros(8, 4, device="cuda"), torch.zeros(2, 4, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        basalto.selective_scan_step(x, x, A, B, B, torch.zeros(2, 4, 8, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError, match="one address"):
        basalto.selective_scan_step(x, x, A, B, B, h[:, :1].expand(2, 8, 4))
    with pytest.raises(TypeError, match="state"):
        basalto.selective_scan_step(x, x, A, B, B, h.bfloat16())
    with pytest.raises(RuntimeError, match="on cpu"):
        basalto.selective_scan_step(x, x, A.cpu(), B, B, h)
    with pytest.raises(RuntimeError, match="on cpu"):
        basalto.layer_norm(x, torch.ones(8))


# ---- a layer: norm, convolution and scan together -------------------------------------------------
class Layer(torch.nn.Module):
    """x + out(scan(conv(in(norm(x))))) with projections between, as a state space layer uses the operators."""

    def __init__(self, width, channels, states, rank=4, dtype=torch.float32):
        super().__init__()
        torch.manual_seed(0)
        self.c, self.n, self.r = channels, states, rank

        def p(*s, scale=0.2, d=dtype):
            return torch.nn.Parameter((torch.randn(*s) * scale).to(d))

        self.norm_w, self.norm_b = p(width, d=torch.float32), p(width, d=torch.float32)
        self.inp, self.out = p(2 * channels, width), p(width, channels)
        self.conv_w, self.conv_b = p(channels, 4), p(channels)
        self.proj, self.dt = p(rank + 2 * states, channels), p(channels, rank)
        self.A = torch.nn.Parameter(-torch.exp(torch.randn(channels, states) * 0.3))
        self.D, self.bias = p(channels, d=torch.float32), p(channels, d=torch.float32)

    def _parts(self, v):
        q = v @ self.proj.t()
        r, B, C = q.split([self.r, self.n, self.n], -1)
        return r @ self.dt.t(), B, C

    def forward(self, x, lengths=None, conv0=None, h0=None, state=False):
        v, z = (basalto.layer_norm(x, self.norm_w, self.norm_b) @ self.inp.t()).chunk(2, -1)
        v = basalto.causal_conv(v, self.conv_w, self.conv_b, "silu", conv0, lengths, state)
        v, conv = v if state else (v, None)
        d, B, C = self._parts(v)
        y = basalto.selective_scan(v, d, self.A, B, C, self.D, z, self.bias, True, h0, lengths, state)
        y, h = y if state else (y, None)
        x = x + y @ self.out.t()
        return (x, conv, h) if state else x

    @torch.no_grad()
    def step(self, x, conv, h):
        v, z = (basalto.layer_norm(x, self.norm_w, self.norm_b) @ self.inp.t()).chunk(2, -1)
        v, _ = basalto.causal_conv_step(v, conv, self.conv_w, self.conv_b, "silu")
        d, B, C = self._parts(v)
        y, _ = basalto.selective_scan_step(v, d, self.A, B, C, h, self.D, z, self.bias, True)
        return x + y @ self.out.t()


def test_prompt_then_tokens_equals_one_pass():
    """A ragged prompt, carried on token by token, against the whole sequences in one call."""
    layer = Layer(24, 40, 16).cuda().eval()
    x = torch.randn(3, 40, 24, device="cuda")
    lens = [20, 0, 33]
    with torch.no_grad():
        whole = layer(x)
        padded = x[:, :33].clone()
        for i, m in enumerate(lens):
            padded[i, m:] = 1e30  # never read by the operators
        y, conv, h = layer(padded, torch.tensor(lens, dtype=torch.int32, device="cuda"), state=True)
        for i, m in enumerate(lens):
            assert torch.allclose(y[i, :m], whole[i, :m], rtol=1e-4, atol=1e-5)
        for k in range(7):
            tok = torch.stack([x[i, m + k] for i, m in enumerate(lens)])
            got = layer.step(tok, conv, h)
            want = torch.stack([whole[i, m + k] for i, m in enumerate(lens)])
            # 40 positions of fp32 arithmetic in another order, values of order one
            assert torch.allclose(got, want, rtol=1e-4, atol=1e-5), k
        first, conv, h = layer(x[:, :17], state=True)  # in two pieces
        second = layer(x[:, 17:], None, conv, h)
        assert torch.allclose(torch.cat([first, second], 1), whole, rtol=1e-4, atol=1e-5)


def test_layer_gradients_match_differences():
    layer = Layer(8, 12, 4).cuda()
    x = torch.randn(2, 19, 8, device="cuda", requires_grad=True)
    goal = torch.randn(2, 19, 8, device="cuda")
    params = [x, *layer.parameters()]
    grads = torch.autograd.grad((layer(x) * goal).sum(), params)
    for p, g in zip(params, grads):
        v = torch.randn_like(p)
        h = 1e-2 / max(1.0, float(v.norm()))
        with torch.no_grad():
            q = p.detach().clone()
            p.copy_(q + h * v)
            up = (layer(x).double() * goal).sum()
            p.copy_(q - h * v)
            down = (layer(x).double() * goal).sum()
            p.copy_(q)
        num, ana = float(up - down) / (2 * h), float((g * v).sum())
        # fp32 values of order 100 over 2 h = 2e-3 or more: 1e-2 absolute; curvature: h^2
        assert abs(num - ana) <= 2e-2 * max(1.0, abs(ana)), (tuple(p.shape), num, ana)


# ---- streams, graphs, devices ---------------------------------------------------------------------
def test_side_stream_and_stream_argument():
    layer = Layer(16, 32, 16).cuda()
    x = torch.randn(2, 50, 16, device="cuda")
    with torch.no_grad():
        want = layer(x)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = layer(x)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        s.wait_stream(torch.cuda.current_stream())
        y = basalto.layer_norm(x, stream=s)
        u = basalto.causal_conv(x, torch.ones(16, 4, device="cuda"), stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(y, basalto.layer_norm(x))
        assert torch.equal(u, basalto.causal_conv(x, torch.ones(16, 4, device="cuda")))


def test_captured_forward_and_backward():
    """Calls captured into two graphs, replayed with new inputs in turn."""
    layer = Layer(16, 32, 16).cuda()
    params = list(layer.parameters())
    xs = [torch.randn(2, 50, 16, device="cuda") for _ in range(2)]
    goal = torch.randn(2, 50, 16, device="cuda")

    def work(x):
        leaf = x.detach().requires_grad_()
        y = layer(leaf)
        return [y.detach(), *torch.autograd.grad(y, [leaf, *params], goal)]

    want = [[t.clone() for t in work(x)] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, ins = [], [], []
    for _ in range(2):
        buf = torch.zeros_like(xs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work(buf)
        graphs.append(g)
        outs.append(out)
        ins.append(buf)
    for turn in range(3):
        for i in range(2):
            ins[i].copy_(xs[(i + turn) % 2])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], want[(i + turn) % 2]):
                assert torch.equal(a, b)


def test_captured_decoding():
    layer = Layer(16, 32, 16).cuda().eval()
    x = torch.randn(4, 3, 16, device="cuda")
    conv, h = torch.zeros(4, 3, 32, device="cuda"), torch.zeros(4, 32, 16, device="cuda")
    want = [layer.step(x[:, k], conv, h).clone() for k in range(3)]
    tok, conv2, h2 = x[:, 0].clone(), torch.zeros_like(conv), torch.zeros_like(h)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer.step(tok, conv2, h2)
    conv2.zero_()
    h2.zero_()
    for k in range(3):
        tok.copy_(x[:, k])
        g.replay()
        assert torch.equal(out, want[k]), k
    assert torch.equal(h2, h) and torch.equal(conv2, conv)


def test_same_bits_every_time():
    t, _, softplus, _, carry = scan_inputs(0, torch.bfloat16)
    leaves = [t[k].requires_grad_() for k in NAMES if t[k] is not None]
    runs = []
    for _ in range(3):
        y = call_scan(t, softplus, carry)
        runs.append([y, *torch.autograd.grad(y, leaves, t["dy"])])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one():
    x = torch.randn(3, 40, device="cuda:1")
    assert torch.equal(basalto.layer_norm(x).cpu(), basalto.layer_norm(x.to("cuda:0")).cpu())
