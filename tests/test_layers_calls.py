"""Calls of the layer operators around their kernels: streams, traces, forward-mode derivatives, version counters."""
import pytest
import torch

import basalto
from basalto import layers


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
