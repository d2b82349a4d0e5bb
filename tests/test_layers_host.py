"""Layer operators without a GPU: the 64-bit reference against differences, refusals, workspace sizes."""
import ctypes

import numpy as np
import pytest
import torch

import basalto
import layer_reference as R
from basalto import _abi


def _difference(f, x, g, rng, h=1e-6):
    """Directional derivative of f at x against the gradient g."""
    v = rng.standard_normal(x.shape)
    num = (f(x + h * v) - f(x - h * v)) / (2 * h)
    # central differences: f64 rounding 2^-52 |f| / h and a third derivative times h^2, both below 1e-8 here
    assert abs(num - (g * v).sum()) <= 1e-6 * max(1.0, abs(num)), (num, (g * v).sum())


def test_reference_layer_norm_gradients_match_differences():
    rng = np.random.default_rng(0)
    x, w, b, dy = (rng.standard_normal(s) for s in ((5, 7), (7,), (7,), (5, 7)))
    _, _, (dx, dw, db), _ = R.layer_norm(x, w, b, 1e-5, dy)
    _difference(lambda v: (R.layer_norm(v, w, b, 1e-5)[0] * dy).sum(), x, dx, rng)
    _difference(lambda v: (R.layer_norm(x, v, b, 1e-5)[0] * dy).sum(), w, dw, rng)
    _difference(lambda v: (R.layer_norm(x, w, v, 1e-5)[0] * dy).sum(), b, db, rng)


@pytest.mark.parametrize("silu", [False, True])
def test_reference_causal_conv_gradients_match_differences(silu):
    rng = np.random.default_rng(1)
    a = {"x": rng.standard_normal((3, 6, 4)), "w": rng.standard_normal((4, 3)), "b": rng.standard_normal(4),
         "initial": rng.standard_normal((3, 2, 4))}
    dy, df, lens = rng.standard_normal((3, 6, 4)), rng.standard_normal((3, 2, 4)), [6, 0, 1]
    out, _ = R.causal_conv(**a, silu=silu, lengths=lens, dy=dy, dfinal=df)

    def loss(name, v):
        o, _ = R.causal_conv(**{**a, name: v}, silu=silu, lengths=lens)
        return (o["y"] * dy).sum() + (o["final"] * df).sum()

    for name, key in (("x", "x"), ("w", "weight"), ("b", "bias"), ("initial", "initial")):
        _difference(lambda v: loss(name, v), a[name], out[key], rng)


@pytest.mark.parametrize("gate,groups", [(True, 1), (False, 2)])
def test_reference_scan_gradients_match_differences(gate, groups):
    rng = np.random.default_rng(2)
    b, l, c, n = 3, 5, 4, 3
    a = {"u": rng.standard_normal((b, l, c)), "delta": rng.standard_normal((b, l, c)),
         "A": -np.exp(rng.standard_normal((c, n))), "B": rng.standard_normal((b, l, groups, n)),
         "C": rng.standard_normal((b, l, groups, n)), "D": rng.standard_normal(c),
         "delta_bias": rng.standard_normal(c), "initial": rng.standard_normal((b, c, n)),
         "z": rng.standard_normal((b, l, c)) if gate else None}
    dy, df, lens = rng.standard_normal((b, l, c)), rng.standard_normal((b, c, n)), [5, 0, 2]
    out, _, _ = R.selective_scan(**a, softplus_on=True, lengths=lens, dy=dy, dfinal=df)

    def loss(name, v):
        o, _, _ = R.selective_scan(**{**a, name: v}, softplus_on=True, lengths=lens)
        return (o["y"] * dy).sum() + (o["final"] * df).sum()

    for name in a:
        if a[name] is not None:
            _difference(lambda v: loss(name, v), a[name], out[name], rng)


def test_reference_conv_equals_torch():
    rng = np.random.default_rng(3)
    x, w, b = rng.standard_normal((2, 9, 5)), rng.standard_normal((5, 4)), rng.standard_normal(5)
    out, _ = R.causal_conv(x, w, b, True)
    t = torch.nn.functional.conv1d(torch.from_numpy(x).transpose(1, 2), torch.from_numpy(w)[:, None],
                                   torch.from_numpy(b), padding=3, groups=5)[..., :9]
    want = torch.nn.functional.silu(t).transpose(1, 2).numpy()
    assert np.abs(out["y"] - want).max() <= 1e-13


# ---- refusals (all of them before any device work) ---------------------------------------------
def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_layer_norm_refusals():
    x = _t(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        basalto.layer_norm(x)
    with pytest.raises(TypeError, match="float64"):
        basalto.layer_norm(x.double())
    with pytest.raises(ValueError, match="weight"):
        basalto.layer_norm(x, _t(7))
    with pytest.raises(TypeError, match="weight"):
        basalto.layer_norm(x, _t(8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="one type"):
        basalto.layer_norm(x.bfloat16(), _t(8), _t(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="eps"):
        basalto.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        basalto.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="axis"):
        basalto.layer_norm(torch.tensor(1.0))


def test_causal_conv_refusals():
    x, w = _t(2, 5, 8), _t(8, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        basalto.causal_conv(x, w)
    with pytest.raises(ValueError, match="batch, length, channels"):
        basalto.causal_conv(x[0], w)
    with pytest.raises(ValueError, match="width"):
        basalto.causal_conv(x, _t(8, 9))
    with pytest.raises(ValueError, match="width"):
        basalto.causal_conv(x, _t(8, 0))
    with pytest.raises(ValueError, match="weight"):
        basalto.causal_conv(x, _t(7, 4))
    with pytest.raises(ValueError, match="bias"):
        basalto.causal_conv(x, w, _t(7))
    with pytest.raises(ValueError, match="activation"):
        basalto.causal_conv(x, w, activation="gelu")
    with pytest.raises(ValueError, match="initial_state"):
        basalto.causal_conv(x, w, initial_state=_t(2, 4, 8))
    with pytest.raises(TypeError, match="initial_state"):
        basalto.causal_conv(x, w, initial_state=_t(2, 3, 8, dtype=torch.float16))
    with pytest.raises(TypeError, match="lengths"):
        basalto.causal_conv(x, w, lengths=torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="lengths"):
        basalto.causal_conv(x, w, lengths=torch.tensor([1], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        basalto.causal_conv_step(x[:, 0], _t(2, 3, 8), w)


def test_selective_scan_refusals():
    u, A, B = _t(2, 5, 8), _t(8, 4), _t(2, 5, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        basalto.selective_scan(u, u, A, B, B)
    with pytest.raises(TypeError, match="float64"):
        basalto.selective_scan(u.double(), u, A, B, B)
    with pytest.raises(TypeError, match="A must be"):
        basalto.selective_scan(u, u, A.bfloat16(), B, B)
    with pytest.raises(ValueError, match="states"):
        basalto.selective_scan(u, u, _t(8, 65), B, B)
    with pytest.raises(ValueError, match="delta"):
        basalto.selective_scan(u, u[:, :4], A, B, B)
    with pytest.raises(ValueError, match="groups"):
        basalto.selective_scan(u, u, A, _t(2, 5, 3, 4), _t(2, 5, 3, 4))
    with pytest.raises(ValueError, match="C must"):
        basalto.selective_scan(u, u, A, B, _t(2, 5, 3))
    with pytest.raises(TypeError, match="B must"):
        basalto.selective_scan(u, u, A, B.half(), B)
    with pytest.raises(TypeError, match="D must"):
        basalto.selective_scan(u, u, A, B, B, D=_t(8, dtype=torch.float16))
    with pytest.raises(ValueError, match="z must"):
        basalto.selective_scan(u, u, A, B, B, z=_t(2, 5, 7))
    with pytest.raises(TypeError, match="initial_state"):
        basalto.selective_scan(u, u, A, B, B, initial_state=_t(2, 8, 4, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="CUDA"):
        basalto.selective_scan_step(u[:, 0], u[:, 0], A, B[:, 0], B[:, 0], _t(2, 8, 4))


def test_c_entries_refuse_before_any_device_work():
    lib, P = _abi.lib(), ctypes.byref
    nd = _abi.CNormDesc(dtype=_abi.BST_F32, param_dtype=_abi.BST_F32, rows=2, dim=8, x_row=8, y_row=8, eps=1e-5)
    call = lambda d, *p: lib.bst_layer_norm_forward(P(d) if d else None, *p, None, None, None)  # noqa: E731
    assert call(None, 16, None, None, 32) == _abi.BST_ERR_INVALID
    assert call(nd, None, None, None, 32) == _abi.BST_ERR_INVALID
    nd.dtype = _abi.BST_F64
    assert call(nd, 16, None, None, 32) == _abi.BST_ERR_UNSUPPORTED
    nd.dtype, nd.param_dtype = _abi.BST_BF16, _abi.BST_F16
    assert call(nd, 16, None, None, 32) == _abi.BST_ERR_UNSUPPORTED
    nd.dtype = nd.param_dtype = _abi.BST_F32
    nd.rows = -1
    assert call(nd, 16, None, None, 32) == _abi.BST_ERR_INVALID
    nd.rows = 0
    assert call(nd, None, None, None, None) == _abi.BST_OK
    nd.rows = 2
    # the backward pass insists on its workspace
    n = ctypes.c_int64()
    assert lib.bst_layer_norm_workspace(P(nd), P(n)) == _abi.BST_OK and n.value >= 2 * 8 * 4
    assert lib.bst_layer_norm_backward(P(nd), 16, None, 16, 16, 16, 16, 16, None, 16, n.value - 1,
                                       None) == _abi.BST_ERR_INVALID
    assert b"workspace" in lib.bst_last_error()

    cd = _abi.CConvDesc(dtype=_abi.BST_BF16, param_dtype=_abi.BST_BF16, width=4, batch=2, length=5, channels=8)
    conv = lambda: lib.bst_causal_conv_forward(P(cd), None, 16, None, None, None, 32, None, None)  # noqa: E731
    assert conv() == _abi.BST_ERR_INVALID
    cd.width = 9
    assert conv() == _abi.BST_ERR_UNSUPPORTED
    cd.width, cd.batch = 4, 65536
    assert conv() == _abi.BST_ERR_UNSUPPORTED
    cd.batch = 0
    assert conv() == _abi.BST_OK
    cd.batch = 2
    assert lib.bst_causal_conv_backward(P(cd), 16, 16, None, None, None, 16, None, 16, 16, None, None, None, 0,
                                        None) == _abi.BST_ERR_INVALID

    sd = _abi.CScanDesc(dtype=_abi.BST_F32, batch=2, length=5, channels=8, states=4, groups=3)
    room = lambda what=1: lib.bst_scan_workspace(P(sd), what, P(n))  # noqa: E731
    assert room() == _abi.BST_ERR_INVALID  # groups do not divide the channels
    sd.groups = 2
    assert room() == _abi.BST_OK and room(7) == _abi.BST_ERR_INVALID
    sd.states = 65
    assert room() == _abi.BST_ERR_UNSUPPORTED
    sd.states = 0
    assert room() == _abi.BST_ERR_UNSUPPORTED
    sd.states = 4
    assert lib.bst_scan_forward(P(sd), *[None] * 14) == _abi.BST_ERR_INVALID
    assert lib.bst_scan_step(P(sd), *[None] * 9, 0, 0, None, None, 0, 0, None) == _abi.BST_ERR_INVALID


@pytest.mark.parametrize("n", [1, 4, 5, 16, 17, 64])
@pytest.mark.parametrize("length", [0, 1, 16, 17, 1000])
def test_saved_state_size_agrees_with_the_library(n, length):
    from basalto.layers import scan_saved_bytes
    sd = _abi.CScanDesc(dtype=_abi.BST_F32, batch=3, length=length, channels=10, states=n, groups=1)
    got = ctypes.c_int64()
    _abi.check(_abi.lib().bst_scan_workspace(ctypes.byref(sd), _abi.BST_SCAN_SAVED, ctypes.byref(got)))
    assert got.value == scan_saved_bytes(3, length, 10, n)


def test_custom_operators_trace_without_a_gpu():
    """Shapes and layouts of the operators on fake tensors, as Dynamo asks for them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 8, 5, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
        w = torch.empty(8, 4, device="cuda", dtype=torch.bfloat16)
        y, final = torch.ops.basalto.causal_conv(x, w, None, True, None, None)
        assert y.shape == x.shape and y.stride(1) == 1 and final.shape == (2, 3, 8)
        y, mean, rstd = torch.ops.basalto.layer_norm(torch.empty(2, 5, 8, device="cuda"), None, None, 1e-5)
        assert y.shape == (2, 5, 8) and mean.shape == rstd.shape == (10,)
        u, A, B = torch.empty(2, 5, 8, device="cuda"), torch.empty(8, 4, device="cuda"), torch.empty(2, 5, 1, 4,
                                                                                                     device="cuda")
        y, final, saved = torch.ops.basalto.selective_scan(u, u, A, B, B, None, None, None, True, None, None, True)
        assert y.shape == u.shape and final.shape == (2, 8, 4) and saved.numel() == 2 * 1 * 8 * 4 * 4
