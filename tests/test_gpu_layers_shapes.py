"""The kernels' shapes for real layers' sizes: every lane shape of the scan, the norm's ring through several rounds,
the sums over many partial rows."""
import numpy as np
import pytest
import torch

import basalto
import layer_bounds
import layer_reference as R
from test_gpu_layers import DT, close, make

pytestmark = pytest.mark.gpu
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial")


# ---- layer norm ------------------------------------------------------------------------------------
# More rows than the resident blocks hold in all stages of their rings.  Tolerances as for fewer rows: y 64, dx 128;
# dw, db: at most rows / 148 terms in a row per slot, 2368 / 32 partial rows and 5 levels: 128.
@pytest.mark.parametrize("rows,dim,dtype", [
    (20003, 96, "fp32"), (20003, 96, "bf16"),      # a warp per row
    (6001, 2048, "fp16"),                          # 128 threads
    (2501, 4096, "bf16"), (2501, 4096, "fp32"),    # 256
    (1100, 8192, "bf16"),                          # 512
    (700, 16384, "bf16"), (500, 16384, "fp32"),    # 1024
    (9001, 99, "bf16"), (1900, 4095, "fp16"),      # not aligned: a row ahead in registers
])
def test_layer_norm_in_many_rounds(rows, dim, dtype):
    rng = np.random.default_rng(rows + dim)
    dt = DT[dtype]
    x, xr = make(rng, rows, dim, dtype=dt)
    w, wr = make(rng, dim)
    b, br = make(rng, dim)
    dy, dr = make(rng, rows, dim, dtype=dt)
    for t in (x, w, b):
        t.requires_grad_()
    y = basalto.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want, mag, grads, mags = R.layer_norm(xr, wr, br, 1e-5, dr)
    close(y, want, mag, 64, "y")
    close(dx, grads[0], mags[0], 128, "dx")
    close(dw, grads[1], mags[1], 128, "dw")
    close(db, grads[2], mags[2], 128, "db")
    basalto.check_device_errors()


# ---- causal convolution ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("lines", [False, True])
def test_convolution_gradients_from_many_pieces(dtype, lines):
    """500 partial rows (8 with the sequence contiguous); the tolerances are those of fewer, with 500 / 32 + 5
    roundings more on the way into a sum."""
    rng = np.random.default_rng(7)
    b, n, c, width = 4, 2000, 24, 4
    dt = DT[dtype]
    x, xr = make(rng, b, n, c, dtype=dt)
    dy, dr = make(rng, b, n, c, dtype=dt)
    w, wr = make(rng, c, width, dtype=dt, scale=0.5)
    bias, br = make(rng, c, dtype=dt)
    if lines:
        x, dy = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, dy))
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    y = basalto.causal_conv(x, w, bias, "silu")
    grads = torch.autograd.grad(y, leaves, dy)
    out, mag = R.causal_conv(xr, wr, br, True, dy=dr)
    close(y, out["y"], mag["y"], 32, "y")
    for name, g, k in zip(("x", "weight", "bias"), grads, (48, 256, 256)):
        close(g, out[name], mag[name], k, name)


def test_empty_convolutions():
    """No sequences, no positions, no channels: the state and its gradient pass through."""
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.zeros(shape[2], 4, device="cuda", requires_grad=True)
        init = torch.randn(shape[0], 3, shape[2], device="cuda", requires_grad=True)
        up = torch.randn(shape[0], 3, shape[2], device="cuda")
        y, final = basalto.causal_conv(x, w, initial_state=init, return_state=True)
        assert y.shape == x.shape and torch.equal(final, init)
        gx, gw, gi = torch.autograd.grad([y, final], (x, w, init), [torch.zeros_like(y), up])
        assert gx.shape == x.shape and gw.shape == w.shape and (gw == 0).all() and torch.equal(gi, up)


# ---- selective scan ------------------------------------------------------------------------------------
# The lane shapes follow the work per scheduler (148 SMs): forward 16 states 64 and 192 channel-state pairs, 32 states
# 192; backward 384.
SHAPES = [  # batch, length, channels, states, groups, lengths
    (1, 33, 4096, 16, 1, None),           # forward: one channel per lane
    (1, 35, 4097, 16, 1, [20]),           # the same, copied element by element in 16 bits
    (2, 33, 4096, 16, 1, [33, 0]),        # forward: two channels
    (4, 36, 4096, 16, 1, [36, 16, 99, 3]),  # both directions
    (5, 19, 3330, 12, 2, [19, 1, 18, 7, 16]),  # the same, in words
    (1, 33, 4096, 32, 1, None),           # 32 states
    (2, 34, 4096, 32, 1, [34, 31]),
    (2, 18, 4094, 24, 2, None),
    (2, 33, 4096, 4, 1, [5, 33]),
    (2, 33, 4096, 8, 2, [33, 32]),
    (1, 33, 2048, 64, 1, None),
    (2, 20, 1026, 64, 2, [20, 4]),
]


def inputs(seed, batch, length, channels, states, groups, lengths, dt, rates=(-3, 1), steps=(-6, -1)):
    """exp of `rates`: -A; of `steps`: about the step sizes."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.empty(*shape, device="cuda").uniform_(lo, hi, generator=g)

    f32 = torch.float32
    t = {"u": normal(batch, length, channels), "delta": normal(batch, length, channels, scale=0.5),
         "A": -torch.exp(uniform(*rates, channels, states)), "B": normal(batch, length, groups, states),
         "C": normal(batch, length, groups, states), "D": normal(channels, dtype=f32),
         "z": normal(batch, length, channels), "delta_bias": uniform(*steps, channels),
         "initial": normal(batch, channels, states, dtype=f32), "dy": normal(batch, length, channels),
         "dfinal": normal(batch, channels, states, dtype=f32)}
    t["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return t


def check(t):
    leaves = [t[k].requires_grad_() for k in NAMES]
    y, final = basalto.selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["delta_bias"], True,
                                      t["initial"], t["lengths"], True)
    grads = torch.autograd.grad([y, final], leaves, [t["dy"], t["dfinal"]])
    want = layer_bounds.scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["delta_bias"], True,
                             t["initial"], t["lengths"], t["dy"], t["dfinal"])
    for name, got in zip(("y", "final", *NAMES), (y, final, *grads)):
        off = layer_bounds.worst(got, *want[name])
        assert off <= 1, (name, off)
    basalto.check_device_errors()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_every_lane_shape(dtype, shape):
    check(inputs(shape, *SHAPES[shape], DT[dtype]))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("batch,length,channels,states,groups", [(1, 3001, 16, 16, 1), (2, 1200, 40, 5, 2),
                                                                (1, 2000, 24, 32, 1)])
def test_long_memories(dtype, batch, length, channels, states, groups):
    """Decays of 1 - 2^-12 to 1 - 2^-5 over thousands of positions, with gradients."""
    check(inputs(length, batch, length, channels, states, groups, None, DT[dtype], rates=(-3, 0), steps=(-6, -4)))
