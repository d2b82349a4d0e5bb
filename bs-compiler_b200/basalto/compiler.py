"""The `"basalto"` torch.compile backend.

Drop-in for the reference's backend (python/basalto/compiler.py:6-97): registered under
the same name, and for stencil graphs it calls the same interceptor entry point,
`basalto._rust.PyBasaltoInterceptor().compile_and_execute(op, dtype, shape, strides, job_id,
device_ptr_x, device_ptr_y, device_ptr_z)`.  The differences are deliberate:

* The reference writes the kernel's result into a throw-away `zeros_like(x)` and returns the
  unmodified graph, so every call really runs eager PyTorch (compiler.py:77-95).  This
  backend returns a callable that launches the sm_100a kernel on the current CUDA stream and
  returns its output.
* The reference always runs the isotropic box of the op's radius; this backend recovers the
  exact stencil (offsets, coefficients and operation order) from the FX graph and passes it
  to the interceptor as a `program`, so the output equals eager torch bit for bit.

BASALTO_FP_CONTRACT=1 compiles stencils with fused multiply-add folding (the arithmetic of
the reference's GPU kernel, `StencilProgram.contract`); by default every operation is
rounded separately, as eager torch does.

Graphs that are not single-input linear stencils (including the reference's matmul /
attention / softmax branches, compiler.py:10-75) are returned unchanged and run eagerly,
which is exactly what the reference does for them; set BASALTO_FALLBACK_EAGER=0 to make
that an error instead.  Stencil graphs called with CPU tensors raise: the kernels run on
CUDA devices only.

BASALTO_MODEL_OPS=1 also sends the layer norms and causal depthwise convolutions of such a graph
to the layer kernels (fx_layers.route), with their gradients; the rest of it runs eagerly.  It is
off by default, because their results differ from eager torch's by rounding.  Graphs in which the
user's code calls basalto.layer_norm, causal_conv or selective_scan run those on the kernels in any
case.  With BASALTO_FALLBACK_EAGER=0 a graph that has such a node is no error.
"""
from __future__ import annotations

import logging
import os
import threading

import torch
import torch.fx

from . import _rust
from .fx_extract import Unsupported, extract
from .fx_layers import has_layer_ops, route

log = logging.getLogger("basalto")

_tls = threading.local()


def _fp_contract() -> bool:
    return os.environ.get("BASALTO_FP_CONTRACT", "0") == "1"


def _model_ops() -> bool:
    return os.environ.get("BASALTO_MODEL_OPS", "0") == "1"


def _extract(gm, args):
    prog, tin = extract(gm, args)
    if _fp_contract():
        prog = prog.contracted()
    return prog, tin


def _job_id():
    return os.environ.get("SLURM_JOB_ID") or os.environ.get("PBS_JOBID") or os.environ.get("LSB_JOBID")


def _interceptor():
    # One interceptor per thread keeps its plan cache warm across graphs and calls.
    it = getattr(_tls, "interceptor", None)
    if it is None:
        it = _tls.interceptor = _rust.PyBasaltoInterceptor()
    return it


def _dtype_name(t: torch.Tensor) -> str:
    return str(t.dtype).split(".")[-1]  # "float32" / "float64", as compiler.py:80


class StencilCallable:
    """What the backend returns for a stencil graph: launches the kernel per call."""

    def __init__(self, gm: torch.fx.GraphModule, program, tin: int, example_shape):
        self.gm = gm
        self.tin = tin
        shape = tuple(example_shape)
        self._programs = {shape: (program, program.pack(shape))}

    def program_for(self, args):
        """(program, packed C descriptor) for the call's grid shape."""
        x = args[self.tin]
        key = tuple(x.shape)
        entry = self._programs.get(key)
        if entry is None:  # a dynamic-shape graph called with new sizes
            prog, _ = _extract(self.gm, args)
            entry = self._programs[key] = (prog, prog.pack(key))
        return entry

    def __call__(self, *args):
        prog, packed = self.program_for(args)
        x = args[self.tin]
        if not x.is_cuda:
            raise RuntimeError("basalto: stencil kernels run on CUDA tensors; got a tensor on " + str(x.device))
        out_shape = prog.out_shape(x.shape)
        if prog.boundary == "zero":
            y = torch.empty_like(x)  # same strides as x (what the interceptor assumes)
        else:
            y = torch.empty(out_shape, dtype=x.dtype, device=x.device)
        if x.numel() == 0 or y.numel() == 0:
            return (y,)
        with torch.cuda.device(x.device):
            _interceptor().compile_and_execute(
                "stencil", _dtype_name(x), list(x.shape), list(x.stride()), _job_id(),
                x.data_ptr(), y.data_ptr(), 0,
                program=packed, stream=torch.cuda.current_stream(x.device).cuda_stream)
        return (y,)


def basalto_backend(gm: torch.fx.GraphModule, example_inputs):
    if not example_inputs:
        return gm
    try:
        prog, tin = _extract(gm, list(example_inputs))
    except Unsupported as e:
        if _model_ops() and route(gm):
            return gm
        if has_layer_ops(gm):
            return gm
        if os.environ.get("BASALTO_FALLBACK_EAGER", "1") == "0":
            raise RuntimeError(f"basalto: graph is not a supported stencil ({e})") from e
        log.info("basalto: running graph eagerly (%s)", e)
        return gm
    return StencilCallable(gm, prog, tin, example_inputs[tin].shape)


torch._dynamo.register_backend(name="basalto")(basalto_backend)
