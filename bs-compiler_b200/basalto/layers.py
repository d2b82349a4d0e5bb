"""Operators of a state space layer over the C ABI: layer norm, short causal convolution, selective scan.

    layer_norm            y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis
    causal_conv           short causal depthwise convolution along the sequence, optionally with silu
    selective_scan        h_t = exp(d_t A) h_{t-1} + d_t u_t B_t,  y_t = (C_t h_t + D u_t) silu(z_t)
    causal_conv_step, selective_scan_step     one position for every sequence, with carried states

They run on CUDA tensors in float32, bfloat16 or float16, on the current stream of the tensors' device (or
on `stream=`: the outputs are then that stream's); arithmetic, statistics and scan states are float32.  The
first three are differentiable, once, in reverse mode.  Under torch.compile, torch.jit.trace and make_fx they appear
in the graph as the custom operators torch.ops.basalto.*; the two step functions mutate a state, run outside of
compiled graphs and refuse to be traced.

Errors: RuntimeError for tensors that are not on one CUDA device and for what the library refuses
(`_abi.BasaltoError`), TypeError for element types, ValueError for shapes.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _abi, _rust

_DT = {torch.float32: _abi.BST_F32, torch.bfloat16: _abi.BST_BF16, torch.float16: _abi.BST_F16}
_NO_GUARD = contextlib.nullcontext()


# ---- arguments ---------------------------------------------------------------------------
def _type(name, t):
    code = _DT.get(t.dtype)
    if code is None:
        raise TypeError(f"basalto.{name} runs in float32, bfloat16 or float16, got {t.dtype}")
    return code


def _need(name, what, t, shape, dtype, device):
    """`t` is a tensor of this shape, element type and device."""
    if t.shape == shape and t.dtype == dtype and t.device == device:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"basalto.{name}: {what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"basalto.{name}: {what} must be {dtype}, got {t.dtype}")
    raise RuntimeError(f"basalto.{name}: {what} is on {t.device}, the input on {device}")


def _cuda(name, t):
    if not t.is_cuda:
        raise RuntimeError(f"basalto.{name} needs CUDA tensors")


def _param(name, what, t, shape, x):
    """A parameter: the input's type or float32.  Returns its type code."""
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise TypeError(f"basalto.{name}: {what} must be {x.dtype} or float32, got {t.dtype}")
    _need(name, what, t, shape, t.dtype, x.device)
    return _DT[t.dtype]


def _same_params(name, a, b):
    if a is not None and b is not None and a.dtype != b.dtype:
        raise TypeError(f"basalto.{name}: weight and bias must have one type")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _guard(t):
    """Makes the tensor's device current for the launch (nothing to do when it already is)."""
    i = t.get_device()
    return _NO_GUARD if i == torch._C._cuda_getDevice() else torch.cuda.device(i)


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _empty(t):
    """A new contiguous tensor like t (a third of the host time of torch.empty with t's shape, type and device)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _dense(t):
    """`t`, or a copy of it, with its last axis contiguous."""
    if t is None or t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] <= 1:
        return t
    return t.contiguous()


def _lengths(name, lengths, batch, device):
    if lengths is not None:
        _need(name, "lengths", lengths, (batch,), torch.int32, device)


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_tangents(name, *ts):
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"basalto.{name} has no forward-mode derivative")


def _tracing():
    """Whether torch operators are being recorded (torch.jit.trace, make_fx): a launch would be missing there."""
    if torch._C._is_tracing():
        return True
    # make_fx works through a dispatch mode, or before dispatch through a function mode.
    if torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack():
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        return get_proxy_mode() is not None
    return False


def _recorded(name, stream, *ts):
    """Whether this call becomes a custom operator of a graph: under Dynamo or in a trace."""
    if not torch.compiler.is_compiling():
        _no_tangents(name, *ts)
        if not _tracing():
            return False
    if stream is not None:
        raise RuntimeError(f"basalto.{name}: stream= is not available in compiled graphs and traces")
    return True


def _on(stream, fn, *args):
    """fn(*args) with `stream` current; the caching allocator learns that the inputs are used there."""
    if stream.device != args[0].device:  # the kernels would run on another stream, unordered with this one
        raise RuntimeError(f"basalto.{fn.__name__}: stream= is on {stream.device}, the input on {args[0].device}")
    with torch.cuda.stream(stream):
        out = fn(*args)
    for t in args:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            t.record_stream(stream)
    return out


# ---- layer norm ----------------------------------------------------------------------------
def _rows(x):
    """x as [rows, dim] with contiguous rows at one distance (a copy where its strides do not allow it)."""
    if not x.numel():
        return x.reshape(0, x.shape[-1])
    if x.dim() != 2:
        try:
            x = x.view(-1, x.shape[-1])
        except RuntimeError:
            x = x.contiguous().view(-1, x.shape[-1])
    return _dense(x)


def _norm_forward(x, weight, bias, eps, stats):
    x2 = _rows(x)
    m, n = x2.shape
    p = weight if weight is not None else bias
    y = _empty(x)
    mean = rstd = None
    if stats:
        mean = torch.empty(m, dtype=torch.float32, device=x.device)
        rstd = torch.empty(m, dtype=torch.float32, device=x.device)
    with _guard(x):
        rc = _rust.layer_norm_forward(_DT[x.dtype], _DT[x.dtype if p is None else p.dtype], (m, n, x2.stride(0), n),
                                      eps, x2.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(mean),
                                      _ptr(rstd), _stream(x))
    if rc:
        _abi.check(rc)
    return y, mean, rstd


def _norm_backward(dy, x, weight, mean, rstd, bias_dtype, want_w, want_b):
    """(dx, dweight, dbias); bias_dtype: the bias' type, where it has one."""
    x2, g2 = _rows(x), _rows(dy)
    m, n = x2.shape
    pt = weight.dtype if weight is not None else (bias_dtype or x.dtype)
    dx = _empty(x)
    dw = torch.empty(n, dtype=pt, device=x.device) if want_w else None
    db = torch.empty(n, dtype=pt, device=x.device) if want_b else None
    code, pcode, dims = _DT[x.dtype], _DT[pt], (m, n, x2.stride(0), n, g2.stride(0), n)
    with _guard(x):
        ws = None
        if want_w or want_b:
            ws = torch.empty(_rust.layer_norm_workspace(code, pcode, dims, 0.0), dtype=torch.uint8, device=x.device)
        rc = _rust.layer_norm_backward(code, pcode, dims, 0.0, x2.data_ptr(), _ptr(weight), g2.data_ptr(),
                                       mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws),
                                       0 if ws is None else ws.numel(), _stream(x))
    if rc:
        _abi.check(rc)
    return dx, dw, db


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        _, want_w, want_b, _ = ctx.needs_input_grad
        return (*_norm_backward(dy, x, weight, mean, rstd, ctx.bias_dtype, want_w, want_b), None)


def _norm_args(name, x, weight, bias, eps):
    _type(name, x)
    if x.dim() < 1:
        raise ValueError("basalto.layer_norm needs at least one axis")
    if not eps >= 0:
        raise ValueError("basalto.layer_norm: eps must be non-negative")
    for what, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _param(name, what, p, (x.shape[-1],), x)
    _same_params(name, weight, bias)


def layer_norm(x, weight=None, bias=None, eps=1e-5, stream=None):
    """Layer norm over the last axis of x.  weight, bias: [dim], of x's type or float32 (both of one type).

    Statistics and arithmetic are float32 whatever the type; the biased variance is taken around the mean, in
    a second sweep.  Rows may lie at any distance; other layouts are copied first."""
    name, eps = "layer_norm", float(eps)
    _norm_args(name, x, weight, bias, eps)
    if _recorded(name, stream, x, weight, bias):
        return torch.ops.basalto.layer_norm(x, weight, bias, eps)[0]
    _cuda(name, x)
    if stream is not None:
        return _on(stream, layer_norm, x, weight, bias, eps)
    weight, bias = _dense(weight), _dense(bias)
    if _wants_grad(x, weight, bias):
        return _Norm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ---- causal convolution ----------------------------------------------------------------------
def _lines(x):
    """Whether the sequence axis of [batch, length, channels] is the contiguous one; None: neither is."""
    if x.stride(2) == 1 or x.shape[2] <= 1:
        return 0
    return 1 if x.stride(1) == 1 or x.shape[1] <= 1 else None


def _conv_layout(x, lines=None):
    """(x or a copy of it, lines) in a layout that the kernels take: the given one, or x's own."""
    if lines is None:
        lines = _lines(x)
        if lines is not None:
            return x, lines
    else:
        axis = 1 if lines else 2
        if x.stride(axis) == 1 or x.shape[axis] <= 1:
            return x, lines
    return (x.transpose(1, 2).contiguous().transpose(1, 2), 1) if lines else (x.contiguous(), 0)


def _conv_empty(x, lines, strides=None):
    b, n, c = x.shape
    if strides is not None:
        return torch.empty_strided((b, n, c), strides, dtype=x.dtype, device=x.device)
    if lines:
        return torch.empty(b, c, n, dtype=x.dtype, device=x.device).transpose(1, 2)
    return _empty(x)


def _step_of(x, lines):
    return x.stride(2) if lines else x.stride(1)


def _conv_forward(x, weight, bias, silu, initial, lengths, want_state, strides=None):
    """strides: of y, with either axis contiguous (None: x's layout)."""
    x, lines = _conv_layout(x, None if strides is None else int(strides[2] != 1))
    y = _conv_empty(x, lines, strides)
    b, n, c = x.shape
    width = weight.shape[1]
    final = torch.empty(b, width - 1, c, dtype=x.dtype, device=x.device) if want_state else None
    with _guard(x):
        rc = _rust.causal_conv_forward(
            _DT[x.dtype], _DT[weight.dtype], width, silu, lines,
            (b, n, c, x.stride(0), _step_of(x, lines), y.stride(0), _step_of(y, lines)), x.data_ptr(),
            weight.data_ptr(), _ptr(bias), _ptr(initial), _ptr(lengths), y.data_ptr(), _ptr(final), _stream(x))
    if rc:
        _abi.check(rc)
    return y, final


def _conv_backward(dy, dfinal, x, weight, bias, silu, initial, lengths, want_bias, want_initial):
    """(dx, dweight, dbias, dinitial)"""
    x, lines = _conv_layout(x)
    dy, _ = _conv_layout(dy, lines)
    dfinal = None if dfinal is None else dfinal.contiguous()
    dx = _conv_empty(x, lines)
    b, n, c = x.shape
    width = weight.shape[1]
    dw = torch.empty(c, width, dtype=weight.dtype, device=x.device)
    db = torch.empty(c, dtype=weight.dtype, device=x.device) if want_bias else None
    dinit = torch.empty(b, width - 1, c, dtype=x.dtype, device=x.device) if want_initial else None
    head = (_DT[x.dtype], _DT[weight.dtype], width, silu, lines,
            (b, n, c, x.stride(0), _step_of(x, lines), 0, 0, dy.stride(0), _step_of(dy, lines), dx.stride(0),
             _step_of(dx, lines)))
    with _guard(x):
        ws = torch.empty(_rust.causal_conv_workspace(*head), dtype=torch.uint8, device=x.device)
        rc = _rust.causal_conv_backward(*head, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial),
                                        _ptr(lengths), dy.data_ptr(), _ptr(dfinal), dx.data_ptr(), dw.data_ptr(),
                                        _ptr(db), _ptr(dinit), ws.data_ptr(), ws.numel(), _stream(x))
    if rc:
        _abi.check(rc)
    return dx, dw, db, dinit


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, initial, lengths, want_state, strides):
        y, final = _conv_forward(x, weight, bias, silu, initial, lengths, want_state, strides)
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return (y, final) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal=None):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        need = ctx.needs_input_grad
        dx, dw, db, dinit = _conv_backward(dy, dfinal, x, weight, bias, ctx.silu, initial, lengths, need[2], need[4])
        return dx, dw, db, None, dinit, None, None, None


def _conv_args(name, x, weight, bias, activation):
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= 8:
        raise ValueError(f"basalto.{name}: weight must be [channels, width] with a width of 1 to 8, "
                         f"got {tuple(weight.shape)}")
    if activation not in (None, "silu"):
        raise ValueError(f"basalto.{name}: activation must be None or 'silu', got {activation!r}")
    c = x.shape[-1]
    _param(name, "weight", weight, (c, weight.shape[1]), x)
    if bias is not None:
        _param(name, "bias", bias, (c,), x)
    _same_params(name, weight, bias)
    return 1 if activation else 0


def _conv_sequence_args(name, x, weight, bias, activation, initial_state, lengths):
    _type(name, x)
    if x.dim() != 3:
        raise ValueError(f"basalto.causal_conv: x must be [batch, length, channels], got {tuple(x.shape)}")
    silu = _conv_args(name, x, weight, bias, activation)
    b, _, c = x.shape
    if initial_state is not None:
        _need(name, "initial_state", initial_state, (b, weight.shape[1] - 1, c), x.dtype, x.device)
    _lengths(name, lengths, b, x.device)
    return silu


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, lengths=None, return_state=False,
                stream=None):
    """Causal depthwise convolution y[b, t, c] = act(bias[c] + sum_k weight[c, k] x[b, t - width + 1 + k, c]).

    x: [batch, length, channels], with the channel axis or (a transposed [batch, channels, length]) the sequence
    axis contiguous; y has the same layout, anything else is copied first.  weight: [channels, width], width 1 to
    8; bias: [channels]; both of x's type or float32.  activation: None or "silu".
    initial_state: [batch, width - 1, channels], the inputs before the first (default: zeros).
    lengths: int32 [batch], the real length of each sequence of a padded batch (clamped to [0, length]); y is
    zero behind it and x is not read there.
    return_state: also return the last width - 1 inputs before each sequence's end, for the next piece of the
    sequence or for causal_conv_step."""
    name = "causal_conv"
    silu = _conv_sequence_args(name, x, weight, bias, activation, initial_state, lengths)
    if _recorded(name, stream, x, weight, bias, initial_state):
        y, final = torch.ops.basalto.causal_conv(x, weight, bias, bool(silu), initial_state, lengths)
        return (y, final) if return_state else y
    _cuda(name, x)
    if stream is not None:
        return _on(stream, causal_conv, x, weight, bias, activation, initial_state, lengths, return_state)
    weight, bias, lengths = weight.contiguous(), _dense(bias), _dense(lengths)
    if initial_state is not None:
        initial_state = initial_state.contiguous()
    if _wants_grad(x, weight, bias, initial_state):
        return _Conv.apply(x, weight, bias, silu, initial_state, lengths, bool(return_state), None)
    y, final = _conv_forward(x, weight, bias, silu, initial_state, lengths, return_state)
    return (y, final) if return_state else y


def _causal_conv_in(strides, x, weight, bias, activation):
    """causal_conv whose y has these strides (either its channels or its positions are 1 apart)."""
    _type("causal_conv", x)
    silu = _conv_args("causal_conv", x, weight, bias, activation)
    _no_tangents("causal_conv", x, weight, bias)
    _cuda("causal_conv", x)
    weight, bias = weight.contiguous(), _dense(bias)
    if _wants_grad(x, weight, bias):
        return _Conv.apply(x, weight, bias, silu, None, None, False, strides)
    return _conv_forward(x, weight, bias, silu, None, None, False, strides)[0]


def _no_grad_step(name, *ts):
    if _wants_grad(*ts):
        raise RuntimeError(f"basalto.{name} is not differentiable: call it under torch.no_grad()")
    _no_tangents(name, *ts)
    if _tracing():
        raise RuntimeError(f"basalto.{name} writes to its state and cannot be traced")


def _out_state(name, state, out_state):
    """The tensor that receives the new state: `state` itself, or a buffer that shares no memory with it."""
    if out_state is None or out_state is state:
        return state
    _need(name, "out_state", out_state, state.shape, state.dtype, state.device)
    at, to = state.data_ptr(), out_state.data_ptr()
    if at == to and state.stride() == out_state.stride():
        return out_state
    if state.is_contiguous() and out_state.is_contiguous():
        meet = abs(at - to) < state.nbytes
    else:
        meet = state.numel() and _spans_meet(state, out_state)
    if meet:
        raise ValueError(f"basalto.{name}: out_state overlaps state")
    return out_state


def _spans_meet(a, b):
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in
                                                                        zip(t.shape, t.stride())))
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _distinct(name, what, t):
    """Every entry of a tensor that is written has an address of its own."""
    reach = 0
    for s, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            if s <= reach:
                raise ValueError(f"basalto.{name}: {what} maps several entries to one address")
            reach += (n - 1) * s


def causal_conv_step(x, state, weight, bias=None, activation=None, out_state=None, stream=None):
    """One position of causal_conv for every sequence: x [batch, channels], state [batch, width - 1, channels]
    (oldest input first) -> (y [batch, channels], new state).

    The new state replaces `state` in place, or goes to `out_state` (which shares no memory with it).  The state's
    rows are contiguous; sequences may lie at any distance."""
    if torch.compiler.is_compiling():
        return _eager_conv_step(x, state, weight, bias, activation, out_state, stream)
    name = "causal_conv_step"
    code = _type(name, x)
    if x.dim() != 2:
        raise ValueError(f"basalto.causal_conv_step: x must be [batch, channels], got {tuple(x.shape)}")
    silu = _conv_args(name, x, weight, bias, activation)
    b, c = x.shape
    width = weight.shape[1]
    _need(name, "state", state, (b, width - 1, c), x.dtype, x.device)
    _no_grad_step(name, x, state, weight, bias)
    _cuda(name, x)
    out = _out_state(name, state, out_state)
    if stream is not None:
        return _on(stream, causal_conv_step, x, state, weight, bias, activation, out)
    for t in (state, out):
        if not t.is_contiguous() and ((c > 1 and t.stride(2) != 1) or (width > 2 and t.stride(1) != c)):
            raise ValueError("basalto.causal_conv_step: the state's rows must be contiguous")
    if not out.is_contiguous():
        _distinct(name, "the state", out)
    x, weight, bias = _dense(x), weight.contiguous(), _dense(bias)
    y = _empty(x)
    with _guard(x):
        rc = _rust.causal_conv_step(code, _DT[weight.dtype], width, silu, b, c, x.stride(0), c, x.data_ptr(),
                                    state.data_ptr(), state.stride(0), weight.data_ptr(), _ptr(bias), y.data_ptr(),
                                    out.data_ptr(), out.stride(0), _stream(x))
    if rc:
        _abi.check(rc)
    increment_version(out)  # autograd's check on saved tensors sees the write
    return y, out


_eager_conv_step = torch.compiler.disable(causal_conv_step)


# ---- selective scan ----------------------------------------------------------------------------
def scan_saved_bytes(batch, length, channels, states):
    """Bytes that a scan keeps for its backward pass: every 16th state, padded to a power of two."""
    pad = 4
    while pad < states:
        pad *= 2
    return batch * ((length + 15) // 16) * channels * pad * 4


def _scan_head(u, delta, z, y, dy, B, C, softplus):
    """(dtype, softplus, the description's sizes and strides)"""
    b, n, c = u.shape

    def two(t):
        return (0, 0) if t is None else (t.stride(0), t.stride(1))

    return (_DT[u.dtype], softplus,
            (b, n, c, B.shape[3], B.shape[2], *two(u), *two(delta), *two(z), *two(y), *two(dy), B.stride(0),
             B.stride(1), B.stride(2), C.stride(0), C.stride(1), C.stride(2)))


def _scan_forward(u, delta, A, B, C, D, z, bias, softplus, initial, lengths, want_state, want_saved):
    u, delta, z, B, C = _dense(u), _dense(delta), _dense(z), _dense(B), _dense(C)
    dev = u.device
    b, n, c = u.shape
    y = _empty(u)
    final = torch.empty(b, c, A.shape[1], dtype=torch.float32, device=dev) if want_state else None
    head = _scan_head(u, delta, z, y, None, B, C, softplus)
    with _guard(u):
        saved = None
        if want_saved:
            saved = torch.empty(_rust.scan_workspace(*head, _abi.BST_SCAN_SAVED), dtype=torch.uint8, device=dev)
        rc = _rust.scan_forward(*head, u.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
                                _ptr(D), _ptr(z), _ptr(bias), _ptr(initial), _ptr(lengths), y.data_ptr(), _ptr(final),
                                _ptr(saved), _stream(u))
    if rc:
        _abi.check(rc)
    return y, final, saved


def _scan_backward(dy, dfinal, u, delta, A, B, C, D, z, bias, softplus, lengths, saved, want_initial):
    """(du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dinitial)"""
    u, delta, z, B, C, dy = _dense(u), _dense(delta), _dense(z), _dense(B), _dense(C), _dense(dy)
    dfinal = None if dfinal is None else dfinal.contiguous()
    dev = u.device
    du, ddelta, dA, dB, dC = _empty(u), _empty(u), _empty(A), _empty(B), _empty(C)
    dz = None if z is None else _empty(u)
    dD = None if D is None else _empty(D)
    dbias = None if bias is None else _empty(bias)
    dinit = None
    if want_initial:
        dinit = torch.empty(u.shape[0], u.shape[2], A.shape[1], dtype=torch.float32, device=dev)
    head = _scan_head(u, delta, z, None, dy, B, C, softplus)
    with _guard(u):
        ws = torch.empty(_rust.scan_workspace(*head, _abi.BST_SCAN_BACKWARD), dtype=torch.uint8, device=dev)
        rc = _rust.scan_backward(*head, u.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
                                 _ptr(D), _ptr(z), _ptr(bias), _ptr(lengths), dy.data_ptr(), _ptr(dfinal),
                                 saved.data_ptr(), du.data_ptr(), ddelta.data_ptr(), dA.data_ptr(), dB.data_ptr(),
                                 dC.data_ptr(), _ptr(dD), _ptr(dz), _ptr(dbias), _ptr(dinit), ws.data_ptr(),
                                 ws.numel(), _stream(u))
    if rc:
        _abi.check(rc)
    return du, ddelta, dA, dB, dC, dD, dz, dbias, dinit


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, softplus, initial, lengths, want_state):
        y, final, saved = _scan_forward(u, delta, A, B, C, D, z, bias, softplus, initial, lengths, want_state, True)
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, lengths, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (y, final) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal=None):
        u, delta, A, B, C, D, z, bias, lengths, saved = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros(u.shape, dtype=u.dtype, device=u.device)
        du, ddelta, dA, dB, dC, dD, dz, dbias, dinit = _scan_backward(
            dy, dfinal, u, delta, A, B, C, D, z, bias, ctx.softplus, lengths, saved, ctx.needs_input_grad[9])
        return du, ddelta, dA, dB, dC, dD, dz, dbias, None, dinit, None, None


def _scan_args(name, u, delta, A, B, C, D, z, delta_bias):
    """Checks what a scan and a step have in common; returns B and C as [.., groups, states]."""
    c = u.shape[-1]
    if A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        raise ValueError(f"basalto.{name}: A must be [channels, states] with 1 to 64 states, got {tuple(A.shape)}")
    n = A.shape[1]
    f32, dev = torch.float32, u.device
    _need(name, "A", A, (c, n), f32, dev)
    _need(name, "delta", delta, u.shape, u.dtype, dev)
    if z is not None:
        _need(name, "z", z, u.shape, u.dtype, dev)
    if D is not None:
        _need(name, "D", D, (c,), f32, dev)
    if delta_bias is not None:
        _need(name, "delta_bias", delta_bias, (c,), f32, dev)
    if B.dim() == u.dim():
        B = B.unsqueeze(-2)
    if C.dim() == u.dim():
        C = C.unsqueeze(-2)
    groups = B.shape[-2] if B.dim() == u.dim() + 1 else 0
    if groups < 1 or c % groups:
        raise ValueError(f"basalto.{name}: B must be [.., states] or [.., groups, states] with groups that divide "
                         f"the {c} channels, got {tuple(B.shape)}")
    shape = (*u.shape[:-1], groups, n)
    _need(name, "B", B, shape, u.dtype, dev)
    _need(name, "C", C, shape, u.dtype, dev)
    return B, C


def _scan_sequence_args(name, u, delta, A, B, C, D, z, delta_bias, initial_state, lengths):
    _type(name, u)
    if u.dim() != 3:
        raise ValueError(f"basalto.selective_scan: u must be [batch, length, channels], got {tuple(u.shape)}")
    B, C = _scan_args(name, u, delta, A, B, C, D, z, delta_bias)
    b, _, c = u.shape
    if initial_state is not None:
        _need(name, "initial_state", initial_state, (b, c, A.shape[1]), torch.float32, u.device)
    _lengths(name, lengths, b, u.device)
    return B, C


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
                   lengths=None, return_state=False, stream=None):
    """Selective state space scan, per batch entry and channel c with the states n:

        d_t = softplus(delta_t + delta_bias)  (or delta_t + delta_bias without delta_softplus)
        h_t[n] = exp(d_t A[c, n]) h_{t-1}[n] + d_t u_t B_t[n]
        y_t = (sum_n C_t[n] h_t[n] + D[c] u_t) * z_t * sigmoid(z_t)     (no z: no gate)

    u, delta, z: [batch, length, channels]; B, C: [batch, length, states], or [batch, length, groups, states] with
    channels / groups neighbouring channels on one of them; all of one type.  A: [channels, states] (1 to 64
    states), D, delta_bias: [channels], initial_state: [batch, channels, states] (default: zeros), all float32.
    The last axes are contiguous, the others lie as they like; other layouts are copied first.
    lengths: int32 [batch], the real lengths of a padded batch (clamped to [0, length]): y is zero behind them and
    nothing is read there.  return_state: also return the state after each sequence's last position, float32
    [batch, channels, states], for the next piece of the sequence or for selective_scan_step."""
    name = "selective_scan"
    B, C = _scan_sequence_args(name, u, delta, A, B, C, D, z, delta_bias, initial_state, lengths)
    if _recorded(name, stream, u, delta, A, B, C, D, z, delta_bias, initial_state):
        # Dynamo makes another graph for inputs with gradients; a trace has to serve those too.
        save = not torch.compiler.is_compiling() or _wants_grad(u, delta, A, B, C, D, z, delta_bias, initial_state)
        y, final, _ = torch.ops.basalto.selective_scan(u, delta, A, B, C, D, z, delta_bias, bool(delta_softplus),
                                                       initial_state, lengths, save)
        return (y, final) if return_state else y
    _cuda(name, u)
    if stream is not None:
        return _on(stream, selective_scan, u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, lengths,
                   return_state)
    softplus = 1 if delta_softplus else 0
    A, D, delta_bias, lengths = A.contiguous(), _dense(D), _dense(delta_bias), _dense(lengths)
    if initial_state is not None:
        initial_state = initial_state.contiguous()
    if _wants_grad(u, delta, A, B, C, D, z, delta_bias, initial_state):
        return _Scan.apply(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, lengths, bool(return_state))
    y, final, _ = _scan_forward(u, delta, A, B, C, D, z, delta_bias, softplus, initial_state, lengths, return_state,
                                False)
    return (y, final) if return_state else y


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=False,
                        out_state=None, stream=None):
    """One position of selective_scan for every sequence: u, delta, z [batch, channels], B, C [batch, states] or
    [batch, groups, states], state [batch, channels, states] float32 -> (y [batch, channels], new state).

    The new state replaces `state` in place, or goes to `out_state` (which shares no memory with it).  The state's
    last axis is contiguous; sequences and channels may lie at any distance."""
    if torch.compiler.is_compiling():
        return _eager_scan_step(u, delta, A, B, C, state, D, z, delta_bias, delta_softplus, out_state, stream)
    name = "selective_scan_step"
    code = _type(name, u)
    if u.dim() != 2:
        raise ValueError(f"basalto.selective_scan_step: u must be [batch, channels], got {tuple(u.shape)}")
    B, C = _scan_args(name, u, delta, A, B, C, D, z, delta_bias)
    b, c = u.shape
    n = A.shape[1]
    _need(name, "state", state, (b, c, n), torch.float32, u.device)
    _no_grad_step(name, u, delta, A, B, C, state, D, z, delta_bias)
    _cuda(name, u)
    out = _out_state(name, state, out_state)
    if stream is not None:
        return _on(stream, selective_scan_step, u, delta, A, B, C, state, D, z, delta_bias, delta_softplus, out)
    if n > 1 and (state.stride(2) != 1 or out.stride(2) != 1):
        raise ValueError("basalto.selective_scan_step: the state's last axis must be contiguous")
    if not out.is_contiguous():
        _distinct(name, "the state", out)
    u, delta, z, B, C = _dense(u), _dense(delta), _dense(z), _dense(B), _dense(C)
    A, D, delta_bias = A.contiguous(), _dense(D), _dense(delta_bias)
    y = _empty(u)
    with _guard(u):
        (Bb, Bg, _), (Cb, Cg, _) = B.stride(), C.stride()
        rc = _rust.scan_step(code, 1 if delta_softplus else 0, b, c, n, B.shape[1], u.stride(0), delta.stride(0),
                             0 if z is None else z.stride(0), c, Bb, Bg, Cb, Cg,
                             u.data_ptr(), delta.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(D),
                             _ptr(z), _ptr(delta_bias), state.data_ptr(), state.stride(0), state.stride(1),
                             y.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), _stream(u))
    if rc:
        _abi.check(rc)
    increment_version(out)
    return y, out


_eager_scan_step = torch.compiler.disable(selective_scan_step)
