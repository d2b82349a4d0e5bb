"""Calls of the layer operators around their kernels: streams, traces, forward-mode derivatives, version counters."""
import ctypes
import threading
import types

import pytest
import torch

import basalto
from basalto import _abi, layers


def strided_lengths(values, device="cpu"):
    """One column of a table, as a scheduler keeps it."""
    table = torch.full((len(values), 3), -7, dtype=torch.int32, device=device)
    table[:, 1] = torch.tensor(values, dtype=torch.int32)
    return table[:, 1]


def parameters(x):
    c = x.shape[2]
    return (torch.ones(c, 4, device=x.device), -torch.ones(c, 4, device=x.device),
            torch.ones(*x.shape[:2], 4, device=x.device))


def conv_and_scan(x, w, A, B, lengths, stream=None):
    return [basalto.causal_conv(x, w, lengths=lengths, stream=stream),
            basalto.selective_scan(x, x, A, B, B, lengths=lengths, stream=stream)]


def test_strided_lengths_are_copied_on_the_stream_of_the_kernel(monkeypatch):
    """What reaches the other stream is the caller's tensor, not a copy made on the current one."""
    lengths, seen = strided_lengths([3, 5]), []
    monkeypatch.setattr(layers, "_cuda", lambda *_: None)
    monkeypatch.setattr(layers, "_on", lambda stream, fn, *args: seen.append(args))
    x = torch.zeros(2, 5, 8)
    conv_and_scan(x, *parameters(x), lengths, stream="another")
    assert len(seen) == 2 and all(any(a is lengths for a in args) for args in seen)


@pytest.mark.gpu
def test_strided_lengths_on_another_stream():
    """The current stream is busy; the other one must not wait for it, nor read what it has not written yet."""
    x, lengths = torch.randn(3, 40, 16, device="cuda"), strided_lengths([17, 0, 33], "cuda")
    params = parameters(x)
    want = conv_and_scan(x, *params, lengths)
    junk = [torch.full((3,), 40, dtype=torch.int32, device="cuda") for _ in range(64)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    del junk  # what the allocator hands out next holds 40s
    torch.cuda._sleep(20_000_000)  # about 10 ms
    got = conv_and_scan(x, *params, lengths, side)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_strided_lengths_in_compiled_graphs():
    x, lengths = torch.randn(3, 40, 16, device="cuda", requires_grad=True), strided_lengths([17, 0, 33], "cuda")
    params = parameters(x)
    want = conv_and_scan(x, *params, lengths)
    torch._dynamo.reset()
    got = torch.compile(conv_and_scan, backend="basalto", fullgraph=True, dynamic=False)(x, *params, lengths)
    grads = [torch.autograd.grad(sum(y.sum() for y in r), x)[0] for r in (got, want)]
    for a, b in zip([*got, grads[0]], [*want, grads[1]]):
        assert torch.equal(a, b)


def test_streams_of_other_devices_are_refused(monkeypatch):
    """The launch goes to the input's device: with another device's stream it would not run on that stream."""
    monkeypatch.setattr(layers, "_cuda", lambda *_: None)
    x = torch.zeros(2, 5, 8)
    other = types.SimpleNamespace(device=torch.device("cuda", 1))
    w, A, B = parameters(x)
    for call in (lambda: basalto.layer_norm(x, stream=other), lambda: basalto.causal_conv(x, w, stream=other),
                 lambda: basalto.selective_scan(x, x, A, B, B, stream=other),
                 lambda: basalto.causal_conv_step(x[:, 0], torch.zeros(2, 3, 8), w, stream=other),
                 lambda: basalto.selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], torch.zeros(2, 8, 4),
                                                     stream=other)):
        with pytest.raises(RuntimeError, match="stream= is on cuda:1, the input on cpu"):
            call()


# ---- forward-mode derivatives and traces ----------------------------------------------------------
def all_calls(x):
    """Every operator as a function of its first input, x [2, 5, 8]."""
    c = x.shape[2]
    w, A, B = parameters(x)
    conv0, h0 = torch.zeros(2, 3, c, device=x.device), torch.zeros(2, c, 4, device=x.device)
    return {"layer_norm": lambda x: basalto.layer_norm(x),
            "causal_conv": lambda x: basalto.causal_conv(x, w),
            "selective_scan": lambda x: basalto.selective_scan(x, x, A, B, B),
            "causal_conv_step": lambda x: basalto.causal_conv_step(x[:, 0], conv0, w)[0],
            "selective_scan_step": lambda x: basalto.selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], h0)[0]}


@pytest.mark.parametrize("op", sorted(all_calls(torch.zeros(2, 5, 8))))
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_derivatives_are_refused(op, dev):
    """They would be lost without a word: the result comes from a kernel that knows no tangents."""
    x = torch.randn(2, 5, 8, device=dev)
    fn = all_calls(x)[op]
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fn(dual)
        if dev == "cuda":
            assert torch.isfinite(fn(x)).all()  # others may run meanwhile
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(fn, (x,), (torch.ones_like(x),))


def test_a_trace_on_fake_tensors_holds_the_operators():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode():
        x = torch.empty(2, 5, 8, device="cuda")
        for op, fn in all_calls(x).items():
            for pre in (False, True):
                if op.endswith("step"):
                    with pytest.raises(RuntimeError, match="traced"):
                        make_fx(fn, pre_dispatch=pre)(x)
                else:
                    graph = make_fx(fn, pre_dispatch=pre)(x).graph
                    assert any(str(n.target) == f"basalto.{op}.default" for n in graph.nodes)
                    with pytest.raises(RuntimeError, match="stream="):
                        make_fx(lambda x: basalto.layer_norm(x, stream="another"), pre_dispatch=pre)(x)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["layer_norm", "causal_conv", "selective_scan"])
def test_traces_run_the_kernels(op):
    """torch.jit.trace and make_fx on real tensors, replayed with others; the traced graph has gradients."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, other = torch.randn(2, 5, 8, device="cuda"), torch.randn(2, 5, 8, device="cuda", requires_grad=True)
    fn = all_calls(x)[op]
    want = fn(other)
    grad = torch.autograd.grad(want.sum(), other)[0]
    for trace in (torch.jit.trace(fn, x), make_fx(fn)(x)):
        got = trace(other)
        assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got.sum(), other)[0], grad)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["causal_conv_step", "selective_scan_step"])
def test_steps_refuse_traces(op):
    x = torch.randn(2, 5, 8, device="cuda")
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(all_calls(x)[op], x)


# ---- states written in place -----------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("inference", [False, True])
def test_steps_count_as_writes_to_their_state(inference):
    x = torch.randn(2, 5, 8, device="cuda")
    w, A, B = parameters(x)
    with torch.inference_mode(inference):
        states = [torch.zeros(2, 3, 8, device="cuda"), torch.zeros(2, 8, 4, device="cuda")]
        others = [torch.zeros_like(s) for s in states]
        for out in (states, others):
            basalto.causal_conv_step(x[:, 0], states[0], w, out_state=out[0])
            basalto.selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], states[1], out_state=out[1])
    if not inference:
        assert [s._version for s in states + others] == [1] * 4
        # A state that a differentiable call has kept for its gradients is not written unnoticed.
        leaf = w.clone().requires_grad_()
        y = basalto.causal_conv(x, leaf, initial_state=states[0])
        with torch.no_grad():
            basalto.causal_conv_step(x[:, 0], states[0], w)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


# ---- C callers on several threads --------------------------------------------------------------------
@pytest.mark.gpu
def test_c_calls_on_two_threads():
    """Rows of two lengths through the same kernels, which need different amounts of shared memory (ctypes lets the
    calls run at the same time)."""
    lib, rows, dims = _abi.lib(), 4, (12000, 8200)

    def caller(dim, failures):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            x, dy = torch.randn(2, rows, dim, device="cuda").unbind()
            y, dx = torch.empty_like(x), torch.empty_like(x)
            mean, rstd = torch.empty(2, rows, device="cuda").unbind()
        d = _abi.CNormDesc(dtype=_abi.BST_F32, param_dtype=_abi.BST_F32, rows=rows, dim=dim, x_row=dim, y_row=dim,
                           dy_row=dim, dx_row=dim, eps=1e-5)
        p = [ctypes.c_void_p(t.data_ptr()) for t in (x, y, mean, rstd, dy, dx)]
        st = ctypes.c_void_p(stream.cuda_stream)
        for _ in range(2000):
            rc = lib.bst_layer_norm_forward(ctypes.byref(d), p[0], None, None, p[1], p[2], p[3], st)
            rc = rc or lib.bst_layer_norm_backward(ctypes.byref(d), p[0], None, p[4], p[2], p[3], p[5], None, None,
                                                   None, 0, st)
            if rc:
                failures.append((dim, rc, lib.bst_last_error()))
                break
        stream.synchronize()
        want = torch.nn.functional.layer_norm(x.double(), (dim,))
        # the mean's and the variance's sums (12 terms in a row, 10 levels), a root, a division: 64 half steps of
        # values to 6
        if not failures and (y - want).abs().max() > 6 * 64 * 2.0 ** -24:
            failures.append((dim, "wrong values"))

    failures = []
    threads = [threading.Thread(target=caller, args=(dim, failures)) for dim in dims]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


# ---- custom operators called by their own names -------------------------------------------------------
def test_statistics_of_the_norm_carry_no_gradient():
    """torch.ops.basalto.layer_norm also returns mean and 1/std, whose gradients its backward pass does not have:
    a loss on them is refused instead of getting zeros."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 5, 8, device="cuda", requires_grad=True)
        y, mean, rstd = torch.ops.basalto.layer_norm(x, None, None, 1e-5)
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad


@pytest.mark.parametrize("fake", [False, True])
def test_custom_operators_check_their_arguments(fake):
    """A wrong shape or type would be read out of range: refused before any launch, as by the functions."""
    import contextlib

    from torch._subclasses.fake_tensor import FakeTensorMode
    o = torch.ops.basalto
    with FakeTensorMode() if fake else contextlib.nullcontext():
        def t(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda" if fake else "cpu")

        x, w, p, A, B, h = t(2, 5, 8), t(8, 4), t(8), t(8, 4), t(2, 5, 1, 4), t(2, 8, 4)
        stat, saved, half = t(10), t(2 * 8 * 4 * 4, dtype=torch.uint8), torch.bfloat16
        lens = t(2, dtype=torch.int64)

        def conv(x=x, w=w, bias=None, initial=None, lengths=None):
            return o.causal_conv(x, w, bias, True, initial, lengths)

        def scan(u=x, delta=x, A=A, B=B, C=B, D=None, z=None, bias=None, initial=None, lengths=None):
            return o.selective_scan(u, delta, A, B, C, D, z, bias, True, initial, lengths, True)

        def scan_grad(dy=x, dfinal=h, u=x, delta=x, A=A, B=B, saved=saved, lengths=None):
            return o.selective_scan_backward(dy, dfinal, u, delta, A, B, B, None, None, None, True, lengths, saved)

        refused = [
            lambda: o.layer_norm(x, t(7), None, 1e-5), lambda: o.layer_norm(x, p.to(half), None, 1e-5),
            lambda: o.layer_norm(x, None, None, -1.0), lambda: o.layer_norm(x.double(), None, None, 1e-5),
            lambda: o.layer_norm_backward(t(2, 5, 7), x, p, stat, stat, p),
            lambda: o.layer_norm_backward(x.to(half), x, p, stat, stat, p),
            lambda: o.layer_norm_backward(x, x, p, t(9), stat, p),
            lambda: conv(w=t(7, 4)), lambda: conv(w=t(8, 9)), lambda: conv(bias=t(7)), lambda: conv(initial=t(2, 2, 8)),
            lambda: conv(lengths=lens),
            lambda: o.causal_conv_backward(t(2, 4, 8), t(2, 3, 8), x, w, None, True, None, None),
            lambda: o.causal_conv_backward(x, t(2, 2, 8), x, w, None, True, None, None),
            lambda: scan(delta=t(2, 5, 7)), lambda: scan(A=t(8, 65)), lambda: scan(B=t(2, 5, 4), C=t(2, 5, 4)),
            lambda: scan(C=t(2, 5, 1, 3)), lambda: scan(D=t(7)), lambda: scan(z=t(2, 4, 8)), lambda: scan(bias=t(7)),
            lambda: scan(initial=t(2, 8, 3)), lambda: scan(lengths=lens),
            lambda: scan_grad(dy=t(2, 4, 8)), lambda: scan_grad(dfinal=t(2, 8, 3)), lambda: scan_grad(saved=saved[:-1]),
            lambda: scan_grad(B=t(2, 4, 1, 4)), lambda: scan_grad(saved=t(0, dtype=torch.uint8)),
        ]
        for call in refused:
            with pytest.raises((ValueError, TypeError)):
                call()
        if fake:
            o.layer_norm_backward(x, x, p, stat, stat, p)
            o.causal_conv_backward(x, t(2, 3, 8), x, w, None, True, None, None)
            scan(), scan_grad()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 0), (0, 8), (2, 0, 8), (2, 3, 0), (5,)])
def test_norm_of_empty_rows_has_the_shapes_of_its_fake(shape):
    x = torch.randn(shape, device="cuda", requires_grad=True)
    torch.library.opcheck(torch.ops.basalto.layer_norm.default, (x, None, None, 1e-5),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_compiled_graphs_of_changing_lengths():
    """One graph for every length and batch (symbolic sizes), with gradients."""
    def f(x, w, A, B, lengths):
        v = basalto.causal_conv(basalto.layer_norm(x), w, activation="silu", lengths=lengths)
        return basalto.selective_scan(v, x, A, B, B, delta_softplus=True, lengths=lengths)

    torch._dynamo.reset()
    compiled = torch.compile(f, backend="basalto", fullgraph=True, dynamic=True)
    for batch, length in ((2, 40), (3, 17), (5, 64)):
        x = torch.randn(batch, length, 16, device="cuda", requires_grad=True)
        w, A, B = parameters(x)
        lengths = torch.full((batch,), length - 3, dtype=torch.int32, device="cuda")
        y, want = compiled(x, w, A, B, lengths), f(x, w, A, B, lengths)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(want.sum(), x)[0])
