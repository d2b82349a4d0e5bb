"""Layer operators under torch.compile(backend="basalto"): routing of a graph's own nodes, custom operators."""
import pytest
import torch
import torch.nn.functional as F

import basalto
from basalto import fx_layers
from basalto.compiler import basalto_backend

C, L = 6, 11


class Block(torch.nn.Module):
    def __init__(self, taps=4, pad="both", dtype=torch.float32):
        super().__init__()
        torch.manual_seed(0)
        self.norm = torch.nn.LayerNorm(C)
        self.conv = torch.nn.Conv1d(C, C, taps, groups=C, padding=taps - 1 if pad == "both" else 0)
        self.pad, self.taps = pad, taps
        self.to(dtype)

    def forward(self, x):  # [batch, length, channels]
        v = self.norm(x).transpose(1, 2)
        if self.pad == "both":
            v = self.conv(v)[..., :x.shape[1]]
        else:
            v = self.conv(F.pad(v, (self.taps - 1, 0)))
        return F.silu(v).transpose(1, 2)


def graph_of(fn, *args):
    """The FX graph that Dynamo builds for fn (fake CUDA tensors: nothing runs)."""
    got = []

    def spy(gm, ex):
        got.append(gm)
        return lambda *a: gm(*a)

    torch._dynamo.reset()
    torch.compile(fn, backend=spy, dynamic=False)(*args)
    return got[0]


def as_cuda(gm):
    """Marks the example values as CUDA tensors, as they would be with a GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    mode = FakeTensorMode()
    for n in gm.graph.nodes:
        v = n.meta.get("example_value")
        if isinstance(v, torch.Tensor):
            with mode:
                n.meta["example_value"] = torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device="cuda")
    return gm


def targets(gm):
    return [n.target for n in gm.graph.nodes if n.op == "call_function"]


@pytest.mark.parametrize("pad", ["both", "left"])
def test_routes_layer_norm_and_causal_convolution(pad):
    m = Block(pad=pad)
    gm = as_cuda(graph_of(m, torch.randn(2, L, C)))
    assert fx_layers.route(gm) == 2
    t = targets(gm)
    assert basalto.layer_norm in t and fx_layers.conv_channels_first in t
    assert not any(f in t for f in (F.layer_norm, torch.conv1d, F.conv1d, F.silu))


def test_leaves_cpu_tensors_and_other_convolutions_alone():
    assert fx_layers.route(graph_of(Block(), torch.randn(2, L, C))) == 0
    w = torch.randn(C, 1, 4)
    cases = [
        lambda x: F.conv1d(x, w, padding=3, groups=C),                          # not cut back
        lambda x: F.conv1d(x, w, padding=3, groups=C)[..., 1:L + 1],            # cut elsewhere
        lambda x: F.conv1d(x, w, padding=3, groups=C)[..., :L - 1],             # cut too short
        lambda x: F.conv1d(x, w, padding=3, groups=C, dilation=2)[..., :L],     # dilated
        lambda x: F.conv1d(x, w, padding=3, groups=C, stride=2)[..., :L],       # strided
        lambda x: F.conv1d(x, torch.cat([w] * C, 1), padding=3)[..., :L],       # not depthwise
        lambda x: F.conv1d(F.pad(x, (2, 1)), w, groups=C),                      # not causal
        lambda x: F.conv1d(F.pad(x, (3, 0), value=1.0), w, groups=C),           # not zeros
        lambda x: F.conv1d(F.pad(x, (9, 0)), torch.randn(C, 1, 10), groups=C),  # ten taps
        lambda x: F.layer_norm(x, (C, L)),                                      # two axes
    ]
    for fn in cases:
        assert fx_layers.route(as_cuda(graph_of(fn, torch.randn(2, C, L)))) == 0
    double = torch.randn(2, L, C, dtype=torch.float64)
    assert fx_layers.route(as_cuda(graph_of(Block(dtype=torch.float64), double))) == 0


def test_leaves_autocast_regions_alone():
    """Under autocast a layer norm answers in fp32 and a convolution in bf16, whatever their input's type."""
    m = Block()
    gm = as_cuda(graph_of(m, torch.randn(2, L, C)))
    for n in gm.graph.nodes:
        if n.op == "call_function" and n.target in (F.layer_norm, torch.conv1d, F.conv1d):
            n.meta["example_value"] = n.meta["example_value"].to(torch.bfloat16)
    assert fx_layers.route(gm) == 0


def test_off_by_default(monkeypatch):
    monkeypatch.delenv("BASALTO_MODEL_OPS", raising=False)
    m = Block()
    gm = as_cuda(graph_of(m, torch.randn(2, L, C)))
    before = targets(gm)
    assert basalto_backend(gm, [torch.randn(2, L, C)]) is gm and targets(gm) == before
    monkeypatch.setenv("BASALTO_MODEL_OPS", "1")
    assert basalto_backend(gm, [torch.randn(2, L, C)]) is gm and targets(gm) != before


@pytest.mark.gpu
@pytest.mark.parametrize("pad", ["both", "left"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled_block_runs_on_the_kernels(monkeypatch, pad, dtype):
    monkeypatch.setenv("BASALTO_MODEL_OPS", "1")
    m = Block(pad=pad, dtype=dtype).cuda()
    x = torch.randn(2, L, C, device="cuda", dtype=dtype, requires_grad=True)
    goal = torch.randn(2, L, C, device="cuda", dtype=dtype)
    torch._dynamo.reset()
    cf = torch.compile(m, backend="basalto", dynamic=False)
    n0 = basalto.launch_count()
    y = cf(x)
    assert basalto.launch_count() == n0 + 2
    leaves = [x, *m.parameters()]
    got = torch.autograd.grad(y, leaves, goal)
    assert basalto.launch_count() >= n0 + 6
    exact = Block(pad=pad, dtype=dtype).double().cuda()
    exact.load_state_dict(m.state_dict())
    xd = x.detach().double().requires_grad_()
    yd = exact(xd)
    want = torch.autograd.grad(yd, [xd, *exact.parameters()], goal.double())
    # Between the two kernels the norm's output (values to 4) is rounded to dtype, and each result once more; the
    # sums run over at most 22 rows: 22 * 4 * (terms to 4) half steps.
    tol = 22 * 16 * torch.finfo(dtype).eps / 2
    for a, b in zip([y, *got], [yd, *want]):
        assert (a.double() - b).abs().max() <= tol


@pytest.mark.gpu
def test_operators_stay_in_compiled_graphs():
    """One graph, no breaks; results and gradients of the eager calls, bit for bit."""
    torch.manual_seed(1)
    c, n = 8, 4
    t = {k: torch.randn(2, L, c, device="cuda", requires_grad=True) for k in ("x", "delta", "z")}
    t["w"], t["b"] = torch.randn(c, 4, device="cuda", requires_grad=True), torch.randn(c, device="cuda",
                                                                                       requires_grad=True)
    t["A"] = (-torch.rand(c, n, device="cuda")).requires_grad_()
    t["B"], t["C"] = (torch.randn(2, L, n, device="cuda", requires_grad=True) for _ in range(2))
    t["h"] = torch.randn(2, c, n, device="cuda", requires_grad=True)
    lens = torch.tensor([L, 5], dtype=torch.int32, device="cuda")

    def f(x, delta, z, w, b, A, B, C, h):
        v = basalto.causal_conv(basalto.layer_norm(x, b, b), w, b, "silu", lengths=lens)
        y, last = basalto.selective_scan(v, delta, A, B, C, D=b, z=z, delta_bias=b, delta_softplus=True,
                                         initial_state=h, lengths=lens, return_state=True)
        return y, last

    args = list(t.values())
    torch._dynamo.reset()
    cf = torch.compile(f, backend="basalto", fullgraph=True, dynamic=False)
    outs = []
    for fn in (f, cf):
        y, last = fn(*args)
        outs.append([y, last, *torch.autograd.grad(y.sum() + (last * last).sum(), args)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_custom_operators_pass_torchs_own_checks():
    x = torch.randn(2, 9, 8, device="cuda", requires_grad=True)
    w = torch.randn(8, 4, device="cuda", requires_grad=True)
    p = torch.randn(8, device="cuda", requires_grad=True)
    A = (-torch.rand(8, 4, device="cuda")).requires_grad_()
    B = torch.randn(2, 9, 1, 4, device="cuda", requires_grad=True)
    check = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.basalto.layer_norm.default, (x, p, p, 1e-5), test_utils=check)
    torch.library.opcheck(torch.ops.basalto.causal_conv.default, (x, w, p, True, None, None), test_utils=check)
    torch.library.opcheck(torch.ops.basalto.selective_scan.default,
                          (x, x, A, B, B, p, x, p, True, None, None, True), test_utils=check)
