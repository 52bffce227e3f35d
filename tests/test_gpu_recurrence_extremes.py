"""The gated linear recurrence with closed and open gates beside states, candidates and gradients near the
end of FP32, against the formulas in 64 bits.

Bounds.  With E = 2^-24, sigmoid(g) and sigmoid(-g) are within 12 E of themselves, a step u h + k c adds 14 E of
its terms, and the maps of the stretches that are joined two roundings more for each step: 64 E of the terms
covers them.  Beneath 2^-126 a gate, or a product of gates, is a multiple of 2^-149 and off by at most one:
2^-147 of the largest state and candidate so far (M) covers a step's gate, candidate and stretch.  So
E_t = u_t E_{t-1} + 64 E (u_t |h_{t-1}| + k_t |c_t|) + 2^-147 M_t, the gradient's bound is the same recurrence
backwards, and dg = G (h - c) u k and dv = G k follow by the product rule, where (h - c) u k beneath 2^-126 is itself
a multiple of 2^-149, rounded to one before G multiplies it: 2^-150 |G| more.  A 16-bit result is off by half a
step more.
"""

import math

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E, TINY = 64 * 2.0**-24, 2.0**-147


def reference(x, state, dy, dlast):
    """y, last, dx and dstate for ``x`` [T, B, 2H] and activation None in 64 bits on the CPU, with their bounds."""
    x, h, dy, G = (t.double().cpu() for t in (x, state, dy, dlast))
    steps, width = x.shape[0], h.shape[1]
    g, c = x[..., :width], x[..., width:]
    u, k = torch.sigmoid(g), torch.sigmoid(-g)
    err, most = torch.zeros_like(h), h.abs()
    rows, before = [], []
    for t in range(steps):
        before.append((h, err))
        most = torch.maximum(most, c[t].abs())
        err = u[t] * err + E * (u[t] * h.abs() + k[t] * c[t].abs()) + TINY * most
        h = u[t] * h + k[t] * c[t]
        rows.append((h, err))
    out = dict(y=tuple(map(torch.stack, zip(*rows))), last=(h, err))
    F, most = torch.zeros_like(G), G.abs()
    dx, dxe = torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(range(steps)):
        G, F = G + dy[t], F + E * (dy[t].abs() + G.abs())
        most = torch.maximum(most, G.abs())
        far, far_e = before[t][0] - c[t], before[t][1]
        gate = u[t] * k[t]
        far_e = far_e + E * (before[t][0].abs() + c[t].abs())
        dx[t, :, :width], dx[t, :, width:] = G * far * gate, G * k[t]
        dxe[t, :, :width] = F * far.abs() * gate + G.abs() * far_e * gate + \
            (E * gate + TINY) * (G * far).abs() + 2.0**-150 * G.abs()
        dxe[t, :, width:] = F * k[t] + (E * k[t] + TINY) * G.abs()
        G, F = u[t] * G, u[t] * F + E * u[t] * G.abs() + TINY * most
    return out | dict(dx=(dx, dxe), dstate=(G, F))


def near(got, pair, label):
    value, bound = pair
    info = torch.finfo(got.dtype)
    if got.dtype != torch.float32:
        bound = bound + info.eps / 2 * (value.abs() + bound) + info.smallest_normal * info.eps
    got = got.detach().double().cpu()
    inside = value.abs() + bound < info.max             # beyond it a result of the type is infinite
    off = torch.where(inside, (got - value).abs(), 0.0)
    assert bool((off <= bound + 2.0**-148).all()), (label, float((off / (bound + 2.0**-148)).max()))


def run(x, state, dy, dlast):
    leaf, start = x.detach().requires_grad_(True), state.detach().requires_grad_(True)
    y, last = memfast.gated_recurrence(leaf, start, activation=None)
    dx, dstate = torch.autograd.grad((y, last), (leaf, start), (dy, dlast))
    return dict(y=y, last=last, dx=dx, dstate=dstate)


GATES = [-math.inf, -3e38, -200.0, -110.0, -104.0, -103.0, -100.0, -95.0, -90.0, -88.0, -87.5, -87.0, -86.0,
         -40.0, 40.0, 86.0, 87.0, 87.5, 88.0, 90.0, 95.0, 100.0, 103.0, 104.0, 110.0, 200.0, 3e38, math.inf]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,at", [(1, 0), (2, 1), (20, 13), (150, 140), (400, 3), (400, 200), (400, 399)])
def test_closed_and_open_gates(hip_device, kind, steps, at):
    """A state that is kept until step ``at`` meets a gate at the ends there; what a closed gate drops is
    gone, however large, and so is what an open one does not take."""
    huge = 1e38 if kind != "fp16" else 6e4
    grid = torch.meshgrid(torch.tensor(GATES), torch.tensor([0.0, 1.0, huge, -huge]),
                          torch.tensor([0.0, 1.0, -1.0, 1e30, 1e38, -1e38]), indexing="ij")
    gate, candidate, state = (t.reshape(-1) for t in grid)
    gen = torch.Generator().manual_seed(steps + at)
    width = len(gate)
    x = torch.randn(steps, 1, 2 * width, generator=gen)
    x[:at, 0, :width] = 40.0
    x[at, 0, :width], x[at, 0, width:] = gate, candidate
    dy = torch.randn(steps, 1, width, generator=gen).to(TYPES[kind])
    given = (x.to(TYPES[kind]), state[None], dy, torch.randn(1, width, generator=gen))
    got = run(*(t.to(hip_device) for t in given))
    for label, pair in reference(*given).items():
        near(got[label], pair, label)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,at", [(1, 0), (20, 13), (150, 10), (400, 200)])
def test_closed_and_open_gates_of_a_large_gradient(hip_device, kind, steps, at):
    """The same backwards: a gradient of the last state that is kept until step ``at``."""
    gate, dlast = (t.reshape(-1) for t in torch.meshgrid(
        torch.tensor(GATES), torch.tensor([0.0, 1.0, 1e30, 1e38, -1e38]), indexing="ij"))
    gen = torch.Generator().manual_seed(steps + at)
    width = len(gate)
    x = torch.randn(steps, 1, 2 * width, generator=gen)
    x[at + 1:, 0, :width] = 40.0
    x[at, 0, :width] = gate
    dy = torch.randn(steps, 1, width, generator=gen).to(TYPES[kind])
    given = (x.to(TYPES[kind]), torch.randn(1, width, generator=gen), dy, dlast[None])
    got = run(*(t.to(hip_device) for t in given))
    for label, pair in reference(*given).items():
        near(got[label], pair, label)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("steps", [3, 16, 40, 300, 700, 9000])
def test_infinite_states_stay(hip_device, kind, reverse, steps):
    """Gates of -10 take a state's share beneath FP32 within a stretch of nine steps; an infinite one is
    infinite after every step all the same, as u h is for every u above 0, and so are gradients."""
    gen = torch.Generator().manual_seed(steps)
    x = torch.randn(steps, 2, 8, generator=gen)
    x[..., :4] = -10.0
    state = torch.tensor([math.inf, -math.inf, 1.0, 0.0]).expand(2, 4).contiguous()
    x, state = x.to(TYPES[kind]).to(hip_device), state.to(hip_device)
    leaf, start = x.clone().requires_grad_(True), state.clone().requires_grad_(True)
    y, last = memfast.gated_recurrence(leaf, start, activation=None, reverse=reverse)
    for channel, sign in ((0, 1), (1, -1)):
        assert bool((y[..., channel] == sign * math.inf).all())
        assert bool((last[..., channel] == sign * math.inf).all())
    assert bool(y[..., 2:].isfinite().all()) and bool(last[..., 2:].isfinite().all())
    # The gradients of a last state, and of one step's state, in steps where the state is finite.
    at = steps // 2
    dlast = torch.zeros_like(last)
    dlast[:, 2], dlast[:, 3] = math.inf, 1.0
    dx, dstate = torch.autograd.grad((y, last), (leaf, start), (torch.zeros_like(y), dlast), retain_graph=True)
    assert bool((dx[..., 6] == math.inf).all()) and bool((dstate[:, 2] == math.inf).all())
    assert bool(dx[..., 2].isinf().all()) and bool(dx[..., 7].isfinite().all())
    dy = torch.zeros_like(y)
    dy[at, :, 2] = -math.inf
    dx, dstate = torch.autograd.grad((y, last), (leaf, start), (dy, torch.zeros_like(last)))
    reached = torch.arange(steps, device=hip_device) >= at if reverse else \
        torch.arange(steps, device=hip_device) <= at
    assert bool((dx[reached][..., 6] == -math.inf).all()) and bool((dx[~reached][..., 6] == 0).all())
    assert bool((dstate[:, 2] == -math.inf).all()) and bool((dstate[:, 3] == 0).all())
    # A candidate, from its step on.
    x[at, :, 4 + 3] = math.inf
    y, last = memfast.gated_recurrence(x, state, activation=None, reverse=reverse)
    after = ~reached if reverse else torch.arange(steps, device=hip_device) >= at
    after[at] = True
    assert bool((y[after][..., 3] == math.inf).all()) and bool((last[:, 3] == math.inf).all())
    assert bool(y[~after][..., 3].isfinite().all()) and bool(y[..., 2].isfinite().all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,batch,width", [(1, 1, 70), (20, 3, 33), (600, 1, 40), (700, 2, 5), (600, 256, 5)])
@pytest.mark.parametrize("activation", ["tanh", None])
def test_far_gates_leave_other_channels_alone(hip_device, kind, steps, batch, width, activation):
    """A closed gate, an open one and a NaN in some channels of a wave: the others' bits are the same."""
    gen = torch.Generator().manual_seed(steps + width)
    x = torch.randn(steps, batch, 2 * width, generator=gen).to(TYPES[kind]).to(hip_device)
    state, dlast = (torch.randn(batch, width, generator=gen).to(hip_device) for _ in range(2))
    dy = torch.randn(steps, batch, width, generator=gen).to(TYPES[kind]).to(hip_device)

    def call(x):
        leaf, start = x.detach().requires_grad_(True), state.clone().requires_grad_(True)
        y, last = memfast.gated_recurrence(leaf, start, activation=activation)
        dx, dstate = torch.autograd.grad((y, last), (leaf, start), (dy, dlast))
        return y, last, dx[..., :width], dx[..., width:], dstate

    expected = call(x)
    x[steps // 2, :, 0], x[steps // 3, :, 1], x[steps - 1, 0, 2] = -200.0, 300.0, math.nan
    got = call(x)
    for a, b in zip(got, expected):
        assert torch.equal(a[..., 3:], b[..., 3:])
    assert not bool(got[1][:, :2].isnan().any()) and bool(got[1][0, 2].isnan())
    assert bool(got[4][0, 2].isnan()) and not bool(got[4][1:].isnan().any())
