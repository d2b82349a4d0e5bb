"""The layer operators as torch.library custom operators, so that graphs built by Dynamo keep them as nodes.

basalto.layer_norm, causal_conv and selective_scan call these while a graph is being compiled or traced and their own
kernels' launchers otherwise; results and gradients are the same.  They can be called by their own names, so each
makes the functions' checks of its arguments, on real and on fake tensors.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import layers as L


# ---- layer norm ------------------------------------------------------------------------------
def _norm_rows(x):
    return x.numel() // x.shape[-1] if x.shape[-1] else 0


def _norm_grad_args(dy, x, weight, mean, rstd, bias):
    name = "layer_norm_backward"
    L._norm_args(name, x, weight, bias, 0.0)
    L._need(name, "dy", dy, x.shape, x.dtype, x.device)
    for what, t in (("mean", mean), ("rstd", rstd)):
        L._need(name, what, t, (_norm_rows(x),), torch.float32, x.device)


@torch.library.custom_op("basalto::layer_norm", mutates_args=())
def layer_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> tuple[Tensor, Tensor, Tensor]:
    L._norm_args("layer_norm", x, weight, bias, eps)
    L._cuda("layer_norm", x)
    return L._norm_forward(x, L._dense(weight), L._dense(bias), eps, True)


@layer_norm.register_fake
def _(x, weight, bias, eps):
    L._norm_args("layer_norm", x, weight, bias, eps)
    stat = x.new_empty(_norm_rows(x), dtype=torch.float32)
    return x.new_empty(x.shape), stat, torch.empty_like(stat)


@torch.library.custom_op("basalto::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: Tensor, x: Tensor, weight: Optional[Tensor], mean: Tensor, rstd: Tensor,
                        bias: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor]:
    _norm_grad_args(dy, x, weight, mean, rstd, bias)
    L._cuda("layer_norm_backward", x)
    mean, rstd = L._dense(mean), L._dense(rstd)
    dx, dw, db = L._norm_backward(dy, x, L._dense(weight), mean, rstd, None if bias is None else bias.dtype,
                                  weight is not None, bias is not None)
    return dx, x.new_empty(0) if dw is None else dw, x.new_empty(0) if db is None else db


@layer_norm_backward.register_fake
def _(dy, x, weight, mean, rstd, bias):
    _norm_grad_args(dy, x, weight, mean, rstd, bias)
    return (x.new_empty(x.shape), x.new_empty(0) if weight is None else weight.new_empty(weight.shape),
            x.new_empty(0) if bias is None else bias.new_empty(bias.shape))


def _norm_context(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1], output[2])
    ctx.mark_non_differentiable(output[1], output[2])


def _norm_grad(ctx, dy, _mean, _rstd):
    x, weight, bias, mean, rstd = ctx.saved_tensors
    dx, dw, db = torch.ops.basalto.layer_norm_backward(dy, x, weight, mean, rstd, bias)
    return dx, None if weight is None else dw, None if bias is None else db, None


layer_norm.register_autograd(_norm_grad, setup_context=_norm_context)


# ---- causal convolution ------------------------------------------------------------------------
def _conv_args(name, x, weight, bias, silu, initial, lengths):
    L._conv_sequence_args(name, x, weight, bias, "silu" if silu else None, initial, lengths)


def _conv_grad_args(dy, dfinal, x, weight, bias, silu, initial, lengths):
    name = "causal_conv_backward"
    _conv_args(name, x, weight, bias, silu, initial, lengths)
    L._need(name, "dy", dy, x.shape, x.dtype, x.device)
    L._need(name, "dfinal", dfinal, (x.shape[0], weight.shape[1] - 1, x.shape[2]), x.dtype, x.device)


@torch.library.custom_op("basalto::causal_conv", mutates_args=())
def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool, initial: Optional[Tensor],
                lengths: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    _conv_args("causal_conv", x, weight, bias, silu, initial, lengths)
    L._cuda("causal_conv", x)
    return L._conv_forward(x, weight.contiguous(), L._dense(bias), int(silu),
                           None if initial is None else initial.contiguous(), L._dense(lengths), True)


@causal_conv.register_fake
def _(x, weight, bias, silu, initial, lengths):
    _conv_args("causal_conv", x, weight, bias, silu, initial, lengths)
    return L._conv_empty(x, L._lines(x) or 0), x.new_empty(x.shape[0], weight.shape[1] - 1, x.shape[2])


@torch.library.custom_op("basalto::causal_conv_backward", mutates_args=())
def causal_conv_backward(dy: Tensor, dfinal: Tensor, x: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool,
                         initial: Optional[Tensor], lengths: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    _conv_grad_args(dy, dfinal, x, weight, bias, silu, initial, lengths)
    L._cuda("causal_conv_backward", x)
    dx, dw, db, dinit = L._conv_backward(dy, dfinal, x, weight.contiguous(), L._dense(bias), int(silu),
                                         None if initial is None else initial.contiguous(), L._dense(lengths),
                                         bias is not None, initial is not None)
    return dx, dw, x.new_empty(0) if db is None else db, x.new_empty(0) if dinit is None else dinit


@causal_conv_backward.register_fake
def _(dy, dfinal, x, weight, bias, silu, initial, lengths):
    _conv_grad_args(dy, dfinal, x, weight, bias, silu, initial, lengths)
    return (L._conv_empty(x, L._lines(x) or 0), weight.new_empty(weight.shape),
            x.new_empty(0) if bias is None else bias.new_empty(bias.shape),
            x.new_empty(0) if initial is None else initial.new_empty(initial.shape))


def _conv_context(ctx, inputs, output):
    x, weight, bias, silu, initial, lengths = inputs
    ctx.save_for_backward(x, weight, bias, initial, lengths)
    ctx.silu = silu


def _conv_grad(ctx, dy, dfinal):
    x, weight, bias, initial, lengths = ctx.saved_tensors
    dx, dw, db, dinit = torch.ops.basalto.causal_conv_backward(dy, dfinal, x, weight, bias, ctx.silu, initial, lengths)
    return dx, dw, None if bias is None else db, None, None if initial is None else dinit, None


causal_conv.register_autograd(_conv_grad, setup_context=_conv_context)


# ---- selective scan ------------------------------------------------------------------------------
def _scan_args(name, u, delta, A, B, C, D, z, delta_bias, initial, lengths):
    if B.dim() != 4 or C.dim() != 4:
        raise ValueError(f"basalto.{name}: B and C must be [batch, length, groups, states]")
    L._scan_sequence_args(name, u, delta, A, B, C, D, z, delta_bias, initial, lengths)


def _scan_grad_args(dy, dfinal, u, delta, A, B, C, D, z, delta_bias, lengths, saved):
    name = "selective_scan_backward"
    _scan_args(name, u, delta, A, B, C, D, z, delta_bias, None, lengths)
    b, n, c = u.shape
    L._need(name, "dy", dy, u.shape, u.dtype, u.device)
    L._need(name, "dfinal", dfinal, (b, c, A.shape[1]), torch.float32, u.device)
    L._need(name, "saved", saved, (L.scan_saved_bytes(b, n, c, A.shape[1]),), torch.uint8, u.device)


@torch.library.custom_op("basalto::selective_scan", mutates_args=())
def selective_scan(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor],
                   z: Optional[Tensor], delta_bias: Optional[Tensor], softplus: bool, initial: Optional[Tensor],
                   lengths: Optional[Tensor], save: bool) -> tuple[Tensor, Tensor, Tensor]:
    _scan_args("selective_scan", u, delta, A, B, C, D, z, delta_bias, initial, lengths)
    L._cuda("selective_scan", u)
    y, final, saved = L._scan_forward(u, delta, A.contiguous(), B, C, L._dense(D), z, L._dense(delta_bias),
                                      int(softplus), None if initial is None else initial.contiguous(),
                                      L._dense(lengths), True, save)
    return y, final, u.new_empty(0, dtype=torch.uint8) if saved is None else saved


@selective_scan.register_fake
def _(u, delta, A, B, C, D, z, delta_bias, softplus, initial, lengths, save):
    _scan_args("selective_scan", u, delta, A, B, C, D, z, delta_bias, initial, lengths)
    b, n, c = u.shape
    room = L.scan_saved_bytes(b, n, c, A.shape[1]) if save else 0
    return (u.new_empty(u.shape), u.new_empty(b, c, A.shape[1], dtype=torch.float32),
            u.new_empty(room, dtype=torch.uint8))


@torch.library.custom_op("basalto::selective_scan_backward", mutates_args=())
def selective_scan_backward(dy: Tensor, dfinal: Tensor, u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor,
                            D: Optional[Tensor], z: Optional[Tensor], delta_bias: Optional[Tensor], softplus: bool,
                            lengths: Optional[Tensor], saved: Tensor) -> list[Tensor]:
    _scan_grad_args(dy, dfinal, u, delta, A, B, C, D, z, delta_bias, lengths, saved)
    L._cuda("selective_scan_backward", u)
    saved = saved.contiguous()
    out = L._scan_backward(dy, dfinal, u, delta, A.contiguous(), B, C, L._dense(D), z, L._dense(delta_bias),
                           int(softplus), L._dense(lengths), saved, True)
    return [u.new_empty(0) if t is None else t for t in out]


@selective_scan_backward.register_fake
def _(dy, dfinal, u, delta, A, B, C, D, z, delta_bias, softplus, lengths, saved):
    _scan_grad_args(dy, dfinal, u, delta, A, B, C, D, z, delta_bias, lengths, saved)
    def like(t):
        return u.new_empty(0) if t is None else t.new_empty(t.shape)

    return [like(u), like(delta), like(A), like(B), like(C), like(D), like(z), like(delta_bias),
            A.new_empty(u.shape[0], *A.shape)]


def _scan_context(ctx, inputs, output):
    u, delta, A, B, C, D, z, delta_bias, softplus, initial, lengths, _ = inputs
    ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, lengths, output[2])
    ctx.softplus = softplus
    ctx.initial = initial is not None


def _scan_grad(ctx, dy, dfinal, _saved):
    u, delta, A, B, C, D, z, delta_bias, lengths, saved = ctx.saved_tensors
    du, dd, dA, dB, dC, dD, dz, dbias, dinit = torch.ops.basalto.selective_scan_backward(
        dy, dfinal, u, delta, A, B, C, D, z, delta_bias, ctx.softplus, lengths, saved)
    return (du, dd, dA, dB, dC, None if D is None else dD, None if z is None else dz,
            None if delta_bias is None else dbias, None, dinit if ctx.initial else None, None, None)


selective_scan.register_autograd(_scan_grad, setup_context=_scan_context)
