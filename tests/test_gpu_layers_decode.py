"""Token by token: thousands of single steps against one scan and against the recurrence in 64 bits."""
import numpy as np
import pytest
import torch

import basalto

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels,states,groups", [(40, 16, 1), (6, 5, 2)])
def test_tokens_leave_the_state_of_a_scan(dtype, channels, states, groups):
    """Bit for bit: both forms round at the same places."""
    torch.manual_seed(channels)
    b, n = 2, 500
    u, delta = (torch.randn(b, n, channels, device="cuda").to(dtype) for _ in range(2))
    B, C = (torch.randn(b, n, groups, states, device="cuda").to(dtype) for _ in range(2))
    A = -torch.exp(torch.empty(channels, states, device="cuda").uniform_(-4, 1))
    bias = torch.empty(channels, device="cuda").uniform_(-6, -2)
    state = torch.randn(b, channels, states, device="cuda")
    _, want = basalto.selective_scan(u, delta, A, B, C, delta_bias=bias, delta_softplus=True, initial_state=state,
                                     return_state=True)
    for t in range(n):
        basalto.selective_scan_step(u[:, t], delta[:, t], A, B[:, t], C[:, t], state, delta_bias=bias,
                                    delta_softplus=True)
    assert torch.equal(state, want)


@pytest.mark.parametrize("form", ["tokens", "scan"])
def test_states_with_a_long_memory(form):
    """Decays from 1 - 2^-10 to 1 - 2^-4, 4000 positions, inputs of one sign.  Per step the state gathers the decay's
    error (its last rounding, 2^-25 below 1, and x = d A log2(e), whose constant, product and second product are each
    off by 2^-24: with the series' other roundings below 6 |d A| 2^-24), the fused operation's (2^-24) and the
    input's (d u, times B: 2 of 2^-24), and passes them on with the decay: the bound follows the same recurrence,
    so it grows with the memory, not with the length."""
    c, n, steps = 64, 16, 4000
    rng = np.random.default_rng(0)
    d = (2.0 ** rng.uniform(-6, -4, c)).astype(np.float32)
    A = -(2.0 ** rng.uniform(-4, 0, (c, n))).astype(np.float32)
    u = rng.uniform(0.5, 1.5, (steps, c)).astype(np.float32)
    one = torch.ones(1, 1, n, device="cuda")
    dt, At = torch.from_numpy(d).cuda()[None], torch.from_numpy(A).cuda()
    ut = torch.from_numpy(u).cuda()[None]
    if form == "tokens":
        h = torch.zeros(1, c, n, device="cuda")
        for t in range(steps):
            basalto.selective_scan_step(ut[:, t], dt, At, one[:, 0], one[:, 0], h)
    else:
        wide = one.expand(1, steps, n)
        _, h = basalto.selective_scan(ut, dt.expand(1, steps, c), At, wide, wide, return_state=True)
    d, A, u = d.astype(float)[:, None], A.astype(float), u.astype(float)
    a = np.exp(d * A)
    want, bound = np.zeros((c, n)), np.zeros((c, n))
    for t in range(steps):
        add = d * u[t][:, None]
        want = a * want + add
        bound = a * bound + EPS * ((0.5 + 6 * np.abs(d * A)) * (want - add) + want + 2 * add)
    off = np.abs(h[0].double().cpu().numpy() - want)
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,channels,states,groups", [
    (149, 4096, 16, 1), (150, 4090, 12, 2), (151, 4096, 16, 1),  # 4 lanes a channel
    (301, 4094, 8, 1),                                           # 2 lanes
    (77, 4096, 32, 2), (78, 4096, 64, 1),                        # 8 lanes, one and two accesses each
])
def test_steps_of_many_sequences(dtype, batch, channels, states, groups):
    """Batches whose threads have four sequences each, with one to three of them left over."""
    g = torch.Generator(device="cuda").manual_seed(batch)

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    u, delta, z = (normal(batch, channels) for _ in range(3))
    B, C = (normal(batch, groups, states) for _ in range(2))
    h = normal(batch, channels, states, dtype=torch.float32)
    A = -torch.exp(torch.empty(channels, states, device="cuda").uniform_(-3, 1, generator=g))
    D, bias = (normal(channels, dtype=torch.float32) for _ in range(2))
    u64, r64, z64, B64, C64, h64, A64, D64 = (t.double() for t in (u, delta, z, B, C, h, A, D))
    d = torch.nn.functional.softplus(r64 + bias.double(), threshold=1000)[..., None]
    B64, C64 = (t.repeat_interleave(channels // groups, 1) for t in (B64, C64))
    keep, add = torch.exp(d * A64) * h64, d * u64[..., None] * B64
    # The step size is good to 12 half steps (its 2^x, its sum, a division and a polynomial) and 4 |delta| of e^-|x|;
    # the decay to 2 and the argument's error times |d A|; d u B two products more; the sum of both one.
    eps_d = 16 + 4 * float((r64 + bias).abs().max())
    err = EPS * ((3 + (eps_d + 3) * (d * A64).abs()) * keep.abs() + (eps_d + 3) * add.abs())
    # y: at most `states` roundings on a sum, the skip's two; the gate's e^-z (4 |z|) and ten more operations.
    gate = z64 * torch.sigmoid(z64)
    y = ((keep + add) * C64).sum(-1) + D64 * u64
    big = ((keep + add) * C64).abs().sum(-1) + (D64 * u64).abs()
    tol = (err * C64.abs()).sum(-1) + EPS * (states + 2) * big
    tol = tol * gate.abs() + EPS * (10 + 4 * z64.abs()) * (y * gate).abs()
    want, new = y * gate, keep + add
    half = EPS if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tol = tol + half * (want.abs() + tol) + torch.finfo(dtype).tiny * half
    for out in (torch.full_like(h, 7.0), None):
        before = h.clone()
        got, state = basalto.selective_scan_step(u, delta, A, B, C, h, D, z, bias, True, out_state=out)
        assert ((got.double() - want).abs() <= tol).all()
        assert ((state.double() - new).abs() <= err + EPS * new.abs()).all()
        assert out is None or torch.equal(h, before)
