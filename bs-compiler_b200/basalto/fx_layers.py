"""Layer operators in the graphs that Dynamo hands the backend.

`route(gm)` looks for nodes that the layer kernels can run on CUDA tensors in float32, bfloat16 or float16:

* F.layer_norm over the last axis;
* F.conv1d that is depthwise and causal: stride and dilation 1, groups = channels, 1 to 8 taps, and either padded
  by taps - 1 on both sides and cut back to the sequence ([..., :length]), or over an F.pad(x, (taps - 1, 0)) of
  zeros; a silu of the result that nothing else reads goes into the same kernel.

It replaces them and returns how many it replaced.  Their gradients are the kernels' own.  Shapes, types and strides
are those of Dynamo's example values; nodes without them, or with symbolic sizes, are left alone.  No other node is
removed, a replacement stands where the layer norm or the convolution stood, and a pad is read through only if nothing
can write to its source: in-place operations of the graph keep their effect and their order.
`has_layer_ops(gm)`: whether the user's code itself called one of the custom operators torch.ops.basalto.*.
"""
from __future__ import annotations

import operator

import torch
import torch.nn.functional as F

from . import layers

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_SILU = {F.silu, torch.ops.aten.silu.default}
_PAD = {F.pad, getattr(torch._C._nn, "pad", F.pad)}
_CONV = {F.conv1d, torch.conv1d}
_MOST_SEQUENCES = 65535  # of a convolution's launch


def _value(n):
    """The example tensor of a node, if its sizes are plain numbers."""
    v = n.meta.get("example_value") if isinstance(n, torch.fx.Node) else None
    if not isinstance(v, torch.Tensor) or v.layout is not torch.strided or v.is_nested:
        return None
    if any(not isinstance(s, int) for s in (*v.shape, *v.stride())):
        return None
    return v


def _usable(*values):
    return all(v is not None and v.is_cuda and v.dtype in _TYPES and v.device == values[0].device for v in values)


def _arg(n, i, name, default=None):
    return n.args[i] if len(n.args) > i else n.kwargs.get(name, default)


def _param_ok(p, x):
    """A parameter node that the kernels take with x (None: absent)."""
    if p is None:
        return True
    v = _value(p)
    return _usable(x, v) and v.dtype in (x.dtype, torch.float32)


def _same_type(*ps):
    return len({_value(p).dtype for p in ps if p is not None}) <= 1


def _layer_norm(n):
    x = _value(_arg(n, 0, "input"))
    shape = _arg(n, 1, "normalized_shape")
    w, b, eps = _arg(n, 2, "weight"), _arg(n, 3, "bias"), _arg(n, 4, "eps", 1e-5)
    if x is None or not _usable(x) or not isinstance(eps, (int, float)) or not eps >= 0:
        return None
    shape = (shape,) if isinstance(shape, int) else shape
    if not isinstance(shape, (tuple, list)) or not _keeps_type(n, x):
        return None
    if x.dim() < 1 or tuple(shape) != (x.shape[-1],) or not (_param_ok(w, x) and _param_ok(b, x) and _same_type(w, b)):
        return None
    return layers.layer_norm, (_arg(n, 0, "input"), w, b, float(eps))


def _keeps_type(n, x):
    """The node's result has its input's element type (autocast can make it another one: left alone)."""
    v = _value(n)
    return v is not None and v.dtype == x.dtype


def _one(v, want):
    return v == want or (isinstance(v, (tuple, list)) and len(v) == 1 and v[0] == want)


def conv_channels_first(x, weight, bias, activation, strides):
    """causal_conv of x [batch, channels, length] with conv1d's weight [channels, 1, taps], its result in the strides
    that the graph's code was traced with."""
    args = x.transpose(1, 2), weight.squeeze(1), bias, activation
    b, c, n = strides
    if c == 1 or n == 1:
        return layers._causal_conv_in((b, n, c), *args).transpose(1, 2)
    y = layers.causal_conv(*args).transpose(1, 2)
    return torch.empty_strided(y.shape, strides, dtype=y.dtype, device=y.device).copy_(y)


def _pad_stays(pad, conv, src):
    """Whether the convolution may read the source of an F.pad instead of its copy: nothing can write to either before
    it does, nor to the source behind it (the gradients read it again)."""
    nodes = list(pad.graph.nodes)
    i, j = nodes.index(pad), nodes.index(conv)
    return all(map(_reads_only, nodes[i + 1:j])) and not any(_writes_to(m, src) for m in nodes[j + 1:])


def _causal_conv(n):
    """(nodes of the pattern, x, weight, bias) of a causal depthwise convolution at conv1d node n."""
    x, w, b = _arg(n, 0, "input"), _arg(n, 1, "weight"), _arg(n, 2, "bias")
    stride, pad = _arg(n, 3, "stride", 1), _arg(n, 4, "padding", 0)
    dilation, groups = _arg(n, 5, "dilation", 1), _arg(n, 6, "groups", 1)
    xv, wv = _value(x), _value(w)
    if xv is None or wv is None or not _usable(xv, wv) or xv.dim() != 3 or wv.dim() != 3:
        return None
    if xv.shape[0] > _MOST_SEQUENCES:
        return None
    c, taps = xv.shape[1], wv.shape[2]
    if groups != c or tuple(wv.shape) != (c, 1, taps) or not 1 <= taps <= 8 or not (_one(stride, 1) and
                                                                                    _one(dilation, 1)):
        return None
    if not (_param_ok(w, xv) and _param_ok(b, xv) and _same_type(w, b) and _keeps_type(n, xv)):
        return None
    if _one(pad, 0) and isinstance(x, torch.fx.Node) and x.target in _PAD and x.op == "call_function":
        spec = _arg(x, 1, "pad")
        src = _value(_arg(x, 0, "input"))
        zeros = _arg(x, 2, "mode", "constant") == "constant" and _arg(x, 3, "value") in (None, 0, 0.0)
        if (src is not None and zeros and isinstance(spec, (tuple, list)) and tuple(spec) == (taps - 1, 0)
                and _pad_stays(x, n, src)):
            return [x, n], _arg(x, 0, "input"), w, b
        return None
    if taps == 1 and _one(pad, 0):
        return [n], x, w, b
    if not _one(pad, taps - 1) or len(n.users) != 1:
        return None
    cut = next(iter(n.users))
    if cut.op != "call_function" or cut.target is not operator.getitem:
        return None
    idx = cut.args[1]
    if not isinstance(idx, tuple) or len(idx) not in (2, 3):
        return None
    lead, last = idx[:-1], idx[-1]
    whole = all(i is Ellipsis or (isinstance(i, slice) and i == slice(None, None, None)) for i in lead)
    if not whole or (len(idx) == 2 and lead[0] is not Ellipsis):
        return None
    length = xv.shape[2]
    if not isinstance(last, slice) or last.start not in (None, 0) or last.step not in (None, 1):
        return None
    if last.stop != length and not (taps > 1 and last.stop == 1 - taps):
        return None
    return [n, cut], x, w, b


# What may stand between a pattern's F.pad and its convolution: operations that write to nothing.
_VIEWS = {"chunk", "contiguous", "detach", "expand", "permute", "reshape", "size", "split", "squeeze", "to", "transpose",
          "unsqueeze", "view"}
_READERS = {operator.getitem, operator.add, operator.sub, operator.mul, operator.truediv, operator.neg, F.layer_norm,
            layers.layer_norm, conv_channels_first} | _PAD | _CONV
# Python's operators that write in place.
_WRITERS = {"setitem", "delitem", "iadd", "iand", "iconcat", "ifloordiv", "ilshift", "imatmul", "imod", "imul", "ior",
            "ipow", "irshift", "isub", "itruediv", "ixor"}


def _reads_only(n):
    return n.op in ("placeholder", "get_attr") or n.target in (_VIEWS if n.op == "call_method" else _READERS)


def _writes_to(n, value):
    """Whether a node may write in place to the memory of `value`: an operation that is named or asked to write in
    place, or one that is not torch's own, with an argument in that memory."""
    name = n.target if isinstance(n.target, str) else getattr(n.target, "__name__", "")
    module = getattr(n.target, "__module__", None) or ""
    if n.op == "output" or _reads_only(n):
        return False
    if n.op == "call_method":
        writes = name.endswith("_") and (not name.endswith("__") or name.startswith(("__i", "__set")))
    elif isinstance(n.target, torch._ops.OpOverload):
        writes = n.target._schema.is_mutable
    elif module in ("_operator", "operator"):
        writes = name in _WRITERS
    else:
        own = not isinstance(n.target, torch._ops.HigherOrderOperator) and (module.startswith("torch") or
                                                                            hasattr(torch, name))
        writes = name.endswith("_") or n.op != "call_function" or not own
    if not (writes or n.kwargs.get("out") is not None or n.kwargs.get("inplace") or any(a is True for a in n.args[1:])):
        return False
    memory = value.untyped_storage()._cdata
    return any(isinstance(v, torch.Tensor) and v.layout is torch.strided and v.untyped_storage()._cdata == memory
               for v in (a.meta.get("example_value") for a in n.all_input_nodes))


def _replace(gm, nodes, at, fn, args):
    """fn(*args) in place of the last of a pattern's nodes (in the graph's order).  It stands where node `at` read the
    inputs: what later nodes write to them does not reach it.  Nodes that nothing else reads are erased, and no
    others: Dynamo's graphs hold the user's in-place operations as nodes without users."""
    last = nodes[-1]
    with gm.graph.inserting_before(at):
        new = gm.graph.call_function(fn, args)
    new.meta = dict(last.meta)
    last.replace_all_uses_with(new)
    for n in reversed(nodes):
        if not n.users:
            gm.graph.erase_node(n)


def has_layer_ops(gm: torch.fx.GraphModule) -> bool:
    return any(n.op == "call_function" and getattr(n.target, "namespace", str(n.target).split(".")[0]) == "basalto"
               for n in gm.graph.nodes)


def route(gm: torch.fx.GraphModule) -> int:
    """Replace what the layer kernels can run, in place; returns how many nodes were replaced."""
    count = 0
    for n in list(gm.graph.nodes):
        if n.op != "call_function":
            continue
        if n.target is F.layer_norm:
            hit = _layer_norm(n)
            if hit:
                _replace(gm, [n], n, *hit)
                count += 1
        elif n.target in _CONV:
            hit = _causal_conv(n)
            if hit:
                nodes, x, w, b = hit
                act = None
                if len(nodes[-1].users) == 1:
                    user = next(iter(nodes[-1].users))
                    if user.op == "call_function" and user.target in _SILU and not user.kwargs.get("inplace") and \
                            len(user.args) == 1:
                        nodes, act = [*nodes, user], "silu"
                if _value(nodes[-1]) is None:
                    continue
                _replace(gm, nodes, n, conv_channels_first, (x, w, b, act, tuple(_value(nodes[-1]).stride())))
                count += 1
    if count:
        gm.recompile()
    return count
