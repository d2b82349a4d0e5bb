"""Routing of a graph's own layer norms and convolutions: what stands around them keeps its effects and results.

The routed graphs run here on the CPU, with plain torch in place of the two kernels.
"""
import operator

import pytest
import torch
import torch.nn.functional as F

import basalto
from basalto import fx_layers, layers
from test_layers_compile import as_cuda, graph_of, targets

C, L, TAPS = 6, 11, 4


def plain_conv(x, weight, bias=None, activation=None):
    """As the kernel: the result has its input's layout."""
    y = F.conv1d(x.transpose(1, 2), weight[:, None], bias, padding=weight.shape[1] - 1, groups=x.shape[2])
    y = y[..., :x.shape[1]].transpose(1, 2)
    return torch.empty_like(x).copy_(F.silu(y) if activation else y)


def plain_conv_in(strides, *args):
    y = plain_conv(*args)
    return torch.empty_strided(y.shape, strides).copy_(y)


def plain_norm(x, weight=None, bias=None, eps=1e-5):
    return F.layer_norm(x, x.shape[-1:], weight, bias, eps)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(layers, "causal_conv", plain_conv)
    monkeypatch.setattr(layers, "_causal_conv_in", plain_conv_in, raising=False)
    monkeypatch.setattr(layers, "layer_norm", plain_norm)


def routed(fn, *args):
    """(the routed graph as a function of fn's own argument order, nodes replaced)"""
    gm = as_cuda(graph_of(fn, *[a.clone() for a in args]))
    names = [n.name for n in gm.graph.nodes if n.op == "placeholder"]
    count = fx_layers.route(gm)
    gm.graph.lint()

    def call(**by_name):
        return gm(*[by_name[n] for n in names])

    return gm, call, count


def same_effects(fn, replaced, **args):
    """fn and its routed graph agree on the results and on every argument afterwards."""
    gm, call, n = routed(fn, *args.values())
    assert n == replaced
    a, b = ({k: v.clone() for k, v in args.items()} for _ in range(2))
    want = fn(*a.values())
    got = call(**{f"l_{k}_": v for k, v in b.items()})
    for g, w in zip(got, want if isinstance(want, tuple) else (want,)):
        assert torch.allclose(g, w, rtol=1e-5, atol=1e-6)
    for k in args:
        assert torch.equal(a[k], b[k]), k
    return gm


def x_(channels_first=True):
    torch.manual_seed(0)
    return torch.randn(2, C, L) if channels_first else torch.randn(2, L, C)


def test_in_place_operations_of_the_graph_stay(plain):
    def conv(x, w, buf, count):
        buf.copy_(x[..., -3:])
        count.add_(1)
        torch.relu_(buf)
        F.relu(count, inplace=True)
        torch.add(count, 1, out=count)
        return F.silu(F.conv1d(x, w, padding=TAPS - 1, groups=C)[..., :L])

    same_effects(conv, 1, x=x_(), w=torch.randn(C, 1, TAPS), buf=torch.zeros(2, C, 3), count=torch.zeros(1))

    def norm(x, count):
        count.add_(1)
        return F.layer_norm(x, (C,))

    gm = same_effects(norm, 1, x=x_(False), count=torch.zeros(1))
    assert F.layer_norm not in targets(gm)


def test_replaced_nodes_leave_and_shared_ones_stay(plain):
    def shared(x, w):
        p = F.pad(x, (TAPS - 1, 0))
        return F.silu(F.conv1d(p, w, groups=C)), p + 1

    gm = same_effects(shared, 1, x=x_(), w=torch.randn(C, 1, TAPS))
    t = targets(gm)
    assert torch.conv1d not in t and F.silu not in t and sum(f in fx_layers._PAD for f in t) == 1


def test_later_writes_do_not_reach_a_replaced_node(plain):
    w = torch.randn(C, 1, TAPS)
    b = torch.randn(C)

    def input_before_silu(x, w):
        v = F.conv1d(x, w, padding=TAPS - 1, groups=C)[..., :L]
        x = x.mul_(2)
        return F.silu(v) + x

    def weight_before_cut(x, w, b):
        v = F.conv1d(x, w, b, padding=TAPS - 1, groups=C)
        w.mul_(3)
        b.add_(1)
        return F.silu(v[..., :L])

    def input_behind_norm(x):
        y = F.layer_norm(x, (L,))
        x.add_(1)
        return y

    same_effects(input_before_silu, 1, x=x_(), w=w)
    same_effects(weight_before_cut, 1, x=x_(), w=w, b=b)
    same_effects(input_behind_norm, 1, x=x_())


def test_a_pad_is_not_read_through_when_something_writes_in_between(plain):
    w = torch.randn(C, 1, TAPS)

    def source(x, w):
        p = F.pad(x, (TAPS - 1, 0))
        x.mul_(2)
        return F.conv1d(p, w, groups=C)

    def padded(x, w):
        p = F.pad(x, (TAPS - 1, 0))
        p[..., 0] = 1.0
        return F.conv1d(p, w, groups=C)

    def view_of_padded(x, w):
        p = F.pad(x, (TAPS - 1, 0))
        torch.relu_(p[..., 2:])
        return F.conv1d(p, w, groups=C)

    for fn in (source, padded, view_of_padded):
        same_effects(fn, 0, x=x_(), w=w)


def test_several_convolutions_of_one_input(plain):
    def two(x, w):
        p, q = F.pad(x, (TAPS - 1, 0)), F.pad(x, (TAPS - 1, 0))
        return F.conv1d(p, w, groups=C), F.silu(F.conv1d(q, w, groups=C)), F.layer_norm(x, (L,))

    same_effects(two, 3, x=x_(), w=torch.randn(C, 1, TAPS))

    def scaled(x, w):
        p = F.pad(x, (TAPS - 1, 0))
        return F.conv1d(p, (w * 2 + 1).contiguous(), groups=C)

    same_effects(scaled, 1, x=x_(), w=torch.randn(C, 1, TAPS))


@pytest.mark.parametrize("write", [lambda x: x.mul_(2), lambda x: F.relu(x, inplace=True), lambda x: F.relu(x, True),
                                   lambda x: torch.add(x, 1, out=x), lambda x: x[0].zero_(), lambda x: torch.relu_(x),
                                   lambda x: x.__setitem__(0, 1.0), lambda x: x.__iadd__(1),
                                   lambda x: torch.ops.aten.mul_.Tensor(x, x), lambda x: operator.imul(x, 2),
                                   lambda x: torch.ops.aten.add.out(x, x, out=x)])
def test_a_pad_whose_source_is_written_later_stays_for_the_gradients(write):
    """The kernel keeps the source for its gradients, the padded convolution its copy."""
    w = torch.randn(C, 1, TAPS)

    def fn(x, w):
        y = F.conv1d(F.pad(x, (TAPS - 1, 0)), w, groups=C)
        write(x)
        return y

    def pure(x, w):
        y = F.conv1d(F.pad(x, (TAPS - 1, 0)), w, groups=C)
        return y.add_(1), x + 1, F.relu(x), x.mean()

    assert fx_layers.route(as_cuda_sharing(graph_of(fn, x_(), w))) == 0
    assert fx_layers.route(as_cuda_sharing(graph_of(pure, x_(), w))) == 1


def as_cuda_sharing(gm):
    """As as_cuda, with views of one tensor still in one memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    memory = {}
    with FakeTensorMode():
        for n in gm.graph.nodes:
            v = n.meta.get("example_value")
            if isinstance(v, torch.Tensor):
                key = v.untyped_storage()._cdata
                if key not in memory:
                    room = v.untyped_storage().nbytes() // v.element_size()
                    memory[key] = torch.empty(room, dtype=v.dtype, device="cuda")
                n.meta["example_value"] = memory[key].as_strided(v.shape, v.stride(), v.storage_offset())
    return gm


def test_other_forms_are_left_alone_without_an_error(plain):
    """Cuts by something else than a tuple, pads by other ways, inputs without strides."""
    w = torch.randn(C, 1, TAPS)

    def conv(x, w):
        return F.conv1d(x, w, padding=TAPS - 1, groups=C)

    cuts = [0, slice(0, L), None, Ellipsis, (Ellipsis,), (), [0, 1], (slice(None), slice(None)),
            (0, Ellipsis, slice(0, L))]
    for idx in cuts:
        same_effects(lambda x, w: conv(x, w)[idx], 0, x=x_(), w=w)
    same_effects(lambda x, w, i: conv(x, w)[i], 0, x=x_(), w=w, i=torch.tensor([1, 0]))
    same_effects(lambda x, w: F.conv1d(F.pad(x, (TAPS - 1, 0), "circular"), w, groups=C), 0, x=x_(), w=w)
    same_effects(lambda x, w: F.conv1d(F.pad(x, [TAPS - 1, 0, 0, 0]), w, groups=C), 0, x=x_(), w=w)

    gm = as_cuda(graph_of(lambda x: F.layer_norm(F.pad(x, (1, 0)), (L + 1,)), x_()))
    norm, pad = (next(n for n in gm.graph.nodes if n.target in t) for t in ({F.layer_norm}, fx_layers._PAD))
    norm.update_arg(1, pad)  # a size that the graph computes
    assert fx_layers.route(gm) == 0
    gm = as_cuda(graph_of(lambda x: F.layer_norm(x, (L,)), x_()))
    source = next(n for n in gm.graph.nodes if n.op == "placeholder")
    source.meta["example_value"] = torch.zeros(2, 3).to_sparse()
    assert fx_layers.route(gm) == 0


def test_results_have_the_layout_that_the_graph_was_traced_with(plain):
    """A convolution answers with the sequence axis contiguous whatever its input's layout, a cut of it with the
    padded length between the rows: code behind it may have been traced for that (views, strides)."""
    w = torch.randn(C, 1, TAPS)

    def padded(x, w):
        return F.conv1d(F.pad(x, (TAPS - 1, 0)), w, groups=C)

    def cut(x, w):
        return F.conv1d(x, w, padding=TAPS - 1, groups=C)[..., :L]

    inputs = {"rows": x_(), "channels": x_(False).transpose(1, 2), "spread": torch.randn(2, C, 2 * L)[..., ::2],
              "one channel": torch.randn(2, 1, L), "one position": torch.randn(2, C, 1)}
    for x in inputs.values():
        c, n = x.shape[1:]
        wx = w[:c]
        fns = [lambda x, w: F.conv1d(F.pad(x, (TAPS - 1, 0)), w, groups=c),
               lambda x, w: F.conv1d(x, w, padding=TAPS - 1, groups=c)[..., :n],
               lambda x, w: F.silu(F.conv1d(x, w, padding=TAPS - 1, groups=c)[..., :n])]
        for fn in fns:
            gm = graph_of(fn, x, wx)
            want = [m.meta["example_value"].stride() for m in gm.graph.nodes if m.op != "output"][-1]
            assert fx_layers.route(as_cuda(gm)) == 1
            got = gm(*[x if m.name == "l_x_" else wx for m in gm.graph.nodes if m.op == "placeholder"])[0]
            assert got.stride() == want and torch.allclose(got, fn(x, wx), rtol=1e-5, atol=1e-6)

    def viewed(x, w):
        y = padded(x, w)
        return y.view(x.shape[0], -1), y.as_strided((2, 3), (C * L, 1))

    same_effects(viewed, 1, x=inputs["channels"], w=w)
    same_effects(lambda x, w: (cut(x, w).as_strided((2, C), (C * (L + TAPS - 1), L + TAPS - 1)),), 1,
                 x=inputs["channels"], w=w)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "channels"])
@pytest.mark.parametrize("form", ["pad", "cut", "silu"])
def test_compiled_layouts_on_the_kernels(monkeypatch, layout, form):
    """The same through the backend, with gradients, against conv1d in 64 bits."""
    monkeypatch.setenv("BASALTO_MODEL_OPS", "1")
    n = 37
    x = torch.randn(2, C, n, device="cuda") if layout == "rows" else torch.randn(2, n, C, device="cuda").transpose(1, 2)
    w = torch.randn(C, 1, TAPS, device="cuda")

    def fn(x, w):
        if form == "pad":
            y = F.conv1d(F.pad(x, (TAPS - 1, 0)), w, groups=C)
            return y.view(x.shape[0], -1)
        y = F.conv1d(x, w, padding=TAPS - 1, groups=C)[..., :x.shape[2]]
        return F.silu(y).view(x.shape[0], -1) if form == "silu" else y

    torch._dynamo.reset()
    cf = torch.compile(fn, backend="basalto", dynamic=False)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    n0 = basalto.launch_count()
    y = cf(*leaves)
    assert basalto.launch_count() == n0 + 1
    if form == "cut":
        assert y.stride() == (C * (n + TAPS - 1), n + TAPS - 1, 1)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = fn(*exact)
    dy = torch.randn_like(want)
    got = [y, *torch.autograd.grad(y, leaves, dy.float())]
    # Values and weights to 5, sums over 4 taps, or 74 positions for the weights: 74 * 25 * 8 half steps of 2^-24.
    for a, b in zip(got, [want, *torch.autograd.grad(want, exact, dy)]):
        assert (a.double() - b).abs().max() <= 74 * 25 * 8 * 2.0 ** -24


def test_what_the_kernels_refuse_is_left_alone():
    """More sequences than a launch can hold, a negative eps: eager torch runs them."""
    w, meta = torch.randn(C, 1, TAPS), torch.device("meta")

    def conv(x, w):
        return F.conv1d(x, w, padding=TAPS - 1, groups=C)[..., :2]

    for batch, want in ((65535, 1), (65536, 0)):
        assert fx_layers.route(as_cuda(graph_of(conv, torch.empty(batch, C, 2, device=meta), w.to(meta)))) == want
    for eps, want in ((0.0, 1), (-1e-3, 0), (float("nan"), 0)):
        gm = as_cuda(graph_of(lambda x: F.layer_norm(x, (C,), eps=eps), x_(False)))
        assert fx_layers.route(gm) == want
