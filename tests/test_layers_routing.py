"""Routing of a graph's own layer norms and convolutions: what stands around them keeps its effects and results.

The routed graphs run here on the CPU, with plain torch in place of the two kernels.
"""
import pytest
import torch
import torch.nn.functional as F

from basalto import fx_layers, layers
from test_layers_compile import as_cuda, graph_of, targets

C, L, TAPS = 6, 11, 4


def plain_conv(x, weight, bias=None, activation=None, **_):
    y = F.conv1d(x.transpose(1, 2), weight[:, None], bias, padding=weight.shape[1] - 1, groups=x.shape[2])
    y = y[..., :x.shape[1]].transpose(1, 2)
    return F.silu(y) if activation else y


def plain_norm(x, weight=None, bias=None, eps=1e-5):
    return F.layer_norm(x, x.shape[-1:], weight, bias, eps)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(layers, "causal_conv", plain_conv)
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
