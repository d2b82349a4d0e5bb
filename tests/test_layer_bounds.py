"""The bounded 64-bit scan against the plain 64-bit one, and against the same computation in float32 (CPU)."""
import pytest
import torch

import layer_bounds
import layer_reference as R


@pytest.mark.parametrize("gate,softplus,groups", [(True, True, 1), (False, False, 2)])
def test_values_are_those_of_the_plain_reference(gate, softplus, groups):
    torch.manual_seed(0)
    b, l, c, n = 3, 7, 6, 4
    f = torch.float64
    t = {"u": torch.randn(b, l, c, dtype=f), "delta": torch.rand(b, l, c, dtype=f), "A": -torch.rand(c, n, dtype=f),
         "B": torch.randn(b, l, groups, n, dtype=f), "C": torch.randn(b, l, groups, n, dtype=f),
         "D": torch.randn(c, dtype=f), "z": torch.randn(b, l, c, dtype=f) if gate else None,
         "delta_bias": torch.randn(c, dtype=f), "initial": torch.randn(b, c, n, dtype=f)}
    dy, dfinal, lens = torch.randn(b, l, c, dtype=f), torch.randn(b, c, n, dtype=f), torch.tensor([7, 0, 3])
    got = layer_bounds.scan(**t, softplus=softplus, lengths=lens, dy=dy, dfinal=dfinal)
    v = {k: None if x is None else x.numpy() for k, x in t.items()}
    want, _, _ = R.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["delta_bias"], softplus,
                                  v["initial"], lens.tolist(), dy.numpy(), dfinal.numpy())
    for k, (x, _) in got.items():
        assert (x - torch.from_numpy(want[k])).abs().max() <= 1e-13, k  # 64-bit values of order ten
    assert set(got) >= {"y", "final", "u", "delta", "A", "B", "C", "D", "delta_bias", "initial"}


def test_a_decay_that_loses_a_digit_is_out_of_bounds():
    """States with a memory of 1000 positions: decays off by 8 half steps are caught, rounded ones are not."""
    torch.manual_seed(1)
    l, c, n = 2000, 8, 4
    u, delta = torch.rand(1, l, c) + 0.5, torch.full((1, l, c), 2.0 ** -6)
    A, one = -torch.full((c, n), 2.0 ** -4), torch.ones(1, l, 1, n)
    want = layer_bounds.scan(u, delta, A, one, one)["final"]
    a = torch.exp(2.0 ** -6 * A.double())
    for off, ok in ((0.0, True), (8 * layer_bounds.U, False)):
        decay, h = (a * (1 + off)).float(), torch.zeros(c, n)
        for t in range(l):
            h = torch.addcmul(2.0 ** -6 * u[0, t][:, None].expand(c, n), decay, h)
        assert (layer_bounds.worst(h[None], *want) <= 1) == ok
