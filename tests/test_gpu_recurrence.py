"""The gated linear recurrence and its gradients against the formulas in 64 bits.

Bounds.  With e = 2^-24: sigmoid(g) and its complement come from exp2 and rcp (each within an ulp, 2 e), an
argument whose rounding is made good but for log2(e)'s own (e |g| / 4), a sum and a product, so within 12 e
for |g| below 20, beyond which the smaller of them is nothing beside the other's term; tanh above 1/4 is
1 - 2 r with r = 1 / (1 + x) and x = exp(2 v): r is below 0.63 beside 1/4 and within 5 e, so the difference
within 2 * 0.63 * 5 e / 0.245 < 27 e, and the series below 1/4 within less.  A step u h + k c adds at most
(12 + 2) e u|h| + (12 + 27 + 2) e k|c|, and the joined maps of sixteen steps, eight waves and the segments
one rounding of A and one of S more for each step that they stand for: 2 C = 64 covers both, where C stands
in the recurrences of the bounds and near() takes them twice.  The bound of h is therefore itself a recurrence, E_t = u_t E_{t-1} + C e (u_t|h_{t-1}| + k_t|c_t|), that of
G is F_t = |dy| C e + u_{t+1} F_{t+1} + C e u_{t+1}|G_{t+1}|, and the gradients' bounds follow by the product
rule.  A result of a 16-bit type is off by half a step more.
"""

import math

import pytest
import torch

import memfast_amd as memfast
from memfast_amd.nn import GatedRecurrence, Int4Linear

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0**-24
C = 32.0


def reference(x, state, lengths, reverse, tanh, dy=None, dlast=None):
    """Everything for ``x`` [T, B, 2H] on the CPU in 64 bits, with bounds: y, last, and with ``dy`` dx and
    dstate."""
    x = x.double().cpu()
    steps, batch, width = x.shape[0], x.shape[1], x.shape[2] // 2
    g, v = x[..., :width], x[..., width:]
    lengths = torch.full((batch,), steps) if lengths is None else lengths.cpu().clamp(0, steps)
    u, k, c = torch.sigmoid(g), torch.sigmoid(-g), torch.tanh(v) if tanh else v
    h = torch.zeros(batch, width, dtype=torch.float64) if state is None else state.double().cpu()
    err = torch.zeros_like(h)
    y, ye = torch.zeros(steps, batch, width, dtype=torch.float64), None
    ye = torch.zeros_like(y)
    before, before_e = torch.zeros_like(y), torch.zeros_like(y)
    live = torch.arange(steps)[:, None] < lengths
    order = range(steps - 1, -1, -1) if reverse else range(steps)
    for t in order:
        on = live[t][:, None]
        before[t], before_e[t] = h, err
        err = torch.where(on, u[t] * err + C * E * (u[t] * h.abs() + k[t] * c[t].abs()), err)
        h = torch.where(on, u[t] * h + k[t] * torch.where(on, c[t], 0.0), h)
        y[t], ye[t] = torch.where(on, h, 0.0), torch.where(on, err, 0.0)
    out = dict(y=(y, ye), last=(h, err))
    if dy is None and dlast is None:
        return out
    G = torch.zeros_like(h) if dlast is None else dlast.double().cpu()
    F = torch.zeros_like(G)
    dy = torch.zeros_like(y) if dy is None else dy.double().cpu()
    dx, dxe = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for t in reversed(order):
        on = live[t][:, None]
        G = torch.where(on, G + dy[t], G)
        F = torch.where(on, F + C * E * dy[t].abs() + C * E * G.abs(), F)
        far = before[t] - c[t]
        far_e = before_e[t] + 13 * E * c[t].abs() + E * far.abs()
        gate = u[t] * k[t]
        slope = k[t] * (1 - c[t] * c[t]) if tanh else k[t]
        slope_e = C * E * slope.abs() + (k[t] * 32 * E * c[t] * c[t] if tanh else 0)
        dx[t, :, :width] = torch.where(on, G * far * gate, 0.0)
        dxe[t, :, :width] = torch.where(
            on, F * far.abs() * gate + G.abs() * far_e * gate + C * E * (G * far * gate).abs(), 0.0)
        dx[t, :, width:] = torch.where(on, G * slope, 0.0)
        dxe[t, :, width:] = torch.where(on, F * slope.abs() + G.abs() * slope_e, 0.0)
        G, F = torch.where(on, u[t] * G, G), torch.where(on, u[t] * F + C * E * u[t] * G.abs(), F)
    return out | dict(dx=(dx, dxe), dstate=(G, F))


def near(got, pair, label):
    value, bound = pair
    info = torch.finfo(got.dtype)
    tiny = 0.0 if got.dtype == torch.float32 else info.smallest_normal * info.eps   # steps of subnormals
    slack = 2 * bound + (info.eps / 2) * value.abs() * (got.dtype != torch.float32) + tiny + 1e-37
    got = got.detach().double().cpu()
    assert got.shape == value.shape, label
    off = (got - value).abs()
    assert bool((off <= slack).all()), (label, float((off / slack).max()), int((off > slack).sum()))


def case(device, steps, batch, width, kind, seed=0):
    gen = torch.Generator().manual_seed(1000 * seed + steps + 7 * batch + 13 * width)
    x = torch.randn(steps, batch, 2 * width, generator=gen)
    x[..., :width] += 1.5 + 1.5 * torch.randn(width, generator=gen)
    dtype = TYPES[kind]
    state = torch.randn(batch, width, generator=gen)
    dy = torch.randn(steps, batch, width, generator=gen).to(dtype)
    dlast = torch.randn(batch, width, generator=gen)
    return tuple(t.to(device) for t in (x.to(dtype), state, dy, dlast))


def check(x, state, dy, dlast, **options):
    """Forward, forward without gradients and gradients of one call against the reference."""
    lengths, reverse = options.get("lengths"), options.get("reverse", False)
    first = options.get("batch_first", False)
    tanh = options.get("activation", "tanh") == "tanh"
    leaf = x.detach().requires_grad_(True)
    start = None if state is None else state.detach().requires_grad_(True)
    y, last = memfast.gated_recurrence(leaf, start, **options)
    assert y.dtype == x.dtype and last.dtype == torch.float32 and y.is_contiguous()
    with torch.no_grad():
        again = memfast.gated_recurrence(x, state, **options)
    assert torch.equal(again[0], y) and torch.equal(again[1], last)
    outputs, grads = [], []
    if dy is not None:
        outputs.append(y), grads.append(dy)
    if dlast is not None:
        outputs.append(last), grads.append(dlast)
    got = torch.autograd.grad(outputs, [leaf] + ([] if start is None else [start]), grads)

    def turn(v):
        return v.transpose(0, 1) if first else v

    expected = reference(turn(x), state, lengths, reverse, tanh, None if dy is None else turn(dy), dlast)
    near(turn(y), expected["y"], "y")
    near(last, expected["last"], "last")
    near(turn(got[0]), expected["dx"], "dx")
    if start is not None:
        near(got[1], expected["dstate"], "dstate")
    return y, last, got


SIZES = [(1, 1, 1), (1, 3, 70), (2, 2, 5), (7, 2, 64), (8, 1, 65), (9, 2, 129), (16, 1, 130), (63, 3, 33),
         (127, 2, 20), (128, 1, 64), (129, 2, 7), (255, 1, 128), (257, 2, 40), (384, 1, 6), (511, 1, 12),
         (513, 3, 66), (640, 1, 3), (1025, 2, 34), (2100, 1, 257)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,batch,width", SIZES)
def test_sizes(hip_device, kind, steps, batch, width):
    x, state, dy, dlast = case(hip_device, steps, batch, width, kind)
    check(x, state, dy, dlast)
    check(x, None, dy, dlast, reverse=True, activation=None)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("steps,width", [(5, 6), (130, 33), (700, 10)])
def test_lengths(hip_device, kind, reverse, first, steps, width):
    """Sequences of no step, one, whole spans, all steps, and lengths outside 0 .. T; what lies behind a
    sequence is not read."""
    lengths = torch.tensor([0, 1, steps, steps - 1, min(128, steps), 4, steps + 9, -3, 129])
    x, state, dy, dlast = case(hip_device, steps, len(lengths), width, kind)
    for b, length in enumerate(lengths.clamp(0, steps).tolist()):
        x[length:, b] = math.nan if b % 2 else math.inf
        dy[length:, b] = math.nan
    if first:
        x, dy = x.transpose(0, 1).contiguous(), dy.transpose(0, 1).contiguous()
    for dtype in (torch.int64, torch.int32):
        y, last, (dx, dstate) = check(x, state, dy, dlast, lengths=lengths.to(hip_device, dtype),
                                      reverse=reverse, batch_first=first)
    for b, length in enumerate(lengths.clamp(0, steps).tolist()):
        rows, grads = (y[b], dx[b]) if first else (y[:, b], dx[:, b])
        assert bool((rows[length:] == 0).all()) and bool((grads[length:] == 0).all())
        if length == 0:
            assert torch.equal(last[b], state[b]) and torch.equal(dstate[b], dlast[b])


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_only_one_output_is_differentiated(hip_device, kind):
    for steps in (20, 700):
        x, state, dy, dlast = case(hip_device, steps, 2, 10, kind)
        check(x, state, dy, None)
        check(x, state, None, dlast)
        y, _ = memfast.gated_recurrence(x.requires_grad_(True), state)
        dx, = torch.autograd.grad(y.sum(), x)                  # an expanded gradient
        near(dx, reference(x.detach(), state, None, False, True, torch.ones_like(dy))["dx"], "dx")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps", [9, 600])
def test_layouts(hip_device, kind, steps):
    """Views with any distances of steps and sequences, odd ones and 0 among them, and a state and
    gradients that are not contiguous, give the bits of their copies."""
    batch, width = 3, 22
    wide = torch.randn(2 * steps, batch, 2 * width + 9, device=hip_device).to(TYPES[kind])
    state = torch.randn(width, batch, device=hip_device).T
    dy = torch.randn(steps, width, batch, device=hip_device).to(TYPES[kind]).transpose(1, 2)
    one = wide[:steps, :1, :2 * width]
    views = (wide[::2, :, 1:2 * width + 1], wide[steps:, :, 3:2 * width + 3], wide[:steps, :, :2 * width],
             one.expand(steps, batch, 2 * width), wide[:steps, :, :4 * width:2],
             wide.transpose(0, 1)[:, :steps, :2 * width].transpose(0, 1))
    for view in views:
        view = view[..., :2 * (view.shape[-1] // 2)]
        w = view.shape[-1] // 2
        results = []
        for x in (view, view.contiguous()):
            leaf = x.detach().requires_grad_(True)
            y, last = memfast.gated_recurrence(leaf, state[:, :w])
            grads = torch.autograd.grad((y, last), leaf, (dy[..., :w], state[:, :w]))
            results.append((y, last, *grads))
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_edges_without_values(hip_device):
    state = torch.randn(2, 3, device=hip_device)
    y, last = memfast.gated_recurrence(torch.zeros(0, 2, 6, device=hip_device), state)
    assert y.shape == (0, 2, 3) and torch.equal(last, state) and last.data_ptr() != state.data_ptr()
    y, last = memfast.gated_recurrence(torch.zeros(2, 0, 6, device=hip_device, requires_grad=True),
                                       batch_first=True)
    assert y.shape == (2, 0, 3) and bool((last == 0).all())
    y.sum().backward()
    for shape in ((4, 0, 6), (4, 2, 0)):
        y, last = memfast.gated_recurrence(torch.zeros(shape, device=hip_device))
        assert y.shape == (*shape[:2], shape[2] // 2) and last.shape == y.shape[1:]


def test_extreme_gates_and_values(hip_device):
    """Gates at the ends of FP32, candidates of every size, NaN and infinities only where they are."""
    gates = torch.tensor([-math.inf, -3e38, -200.0, -88.0, -20.0, -1e-3, 0.0, 1e-30, 5.0, 17.0, 90.0, 200.0,
                          3e38, math.inf])
    values = torch.tensor([1e-30, -1e-4, 0.2499, 0.2501, -0.3, 1.0, -9.0, 30.0, 3e38, -3e38])
    g, v = torch.meshgrid(gates, values, indexing="ij")
    x = torch.cat((g.reshape(1, 1, -1), v.reshape(1, 1, -1)), -1).to(hip_device)
    x = x.expand(3, 1, -1).contiguous()
    width = x.shape[-1] // 2
    state = torch.randn(1, width, device=hip_device)
    near(memfast.gated_recurrence(x, state)[0], reference(x, state, None, False, True)["y"], "y")
    leaf = x.requires_grad_(True)
    y, _ = memfast.gated_recurrence(leaf, state)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    near(dx, reference(x.detach(), state, None, False, True, torch.ones_like(y))["dx"], "dx")
    x = torch.zeros(300, 2, 8, device=hip_device)
    x[150, 0, 1] = math.nan       # a gate
    x[10, 1, 6] = math.inf        # a candidate, bounded by tanh
    x[20, 1, 7] = math.nan
    y, last = memfast.gated_recurrence(x)
    bad = torch.zeros(300, 2, 4, dtype=torch.bool, device=hip_device)
    bad[150:, 0, 1] = True
    bad[20:, 1, 3] = True
    assert torch.equal(y.isnan(), bad) and torch.equal(last.isnan(), bad[-1])


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_parts_are_the_sequence(hip_device, kind):
    """A sequence taken in parts, down to single steps, passes its FP32 state on."""
    x, state, _, _ = case(hip_device, 300, 2, 20, kind)
    expected = reference(x, state, None, False, True)
    for cut in ((100, 200), (1, 2, 3, 130)):
        h, parts = state, []
        for part in torch.tensor_split(x, cut):
            y, h = memfast.gated_recurrence(part, h)
            parts.append(y)
        near(torch.cat(parts), expected["y"], "y")
        near(h, expected["last"], "last")
    h = state
    for t in range(40):
        y, h = memfast.gated_recurrence(x[t:t + 1], h)
        near(y[0], (expected["y"][0][t], expected["y"][1][t]), "step")
    if kind == "bf16":          # a state of the input's type
        short = reference(x, state.bfloat16(), None, False, True)
        near(memfast.gated_recurrence(x, state.bfloat16())[0], short["y"], "y")


def test_a_sequence_without_batch(hip_device):
    x, state, dy, _ = case(hip_device, 40, 1, 6, "fp32")
    lengths = torch.tensor([30], device=hip_device)
    for options in ({}, dict(reverse=True)):
        for first in (False, True):
            y, last = memfast.gated_recurrence(x[:, 0], state[0], lengths=lengths[0], batch_first=first,
                                               **options)
            expected = memfast.gated_recurrence(x, state, lengths=lengths, **options)
            assert torch.equal(y, expected[0][:, 0]) and torch.equal(last, expected[1][0])


def test_gradients_against_differences(hip_device):
    """Central differences of the kernel's own outputs. Their error: what the 64-bit formula's own
    difference has (truncation), and the outputs' bounds over the step."""
    x, state, dy, dlast = case(hip_device, 40, 1, 3, "fp32")
    gen = torch.Generator().manual_seed(5)
    step = 2.0**-7
    expected = reference(x, state, None, False, True, dy, dlast)

    def value(y, last):
        return float((y.double().cpu() * dy.double().cpu()).sum() + (last.double().cpu() *
                                                                     dlast.double().cpu()).sum())

    leaf = x.clone().requires_grad_(True)
    y, last = memfast.gated_recurrence(leaf, state)
    dx, = torch.autograd.grad((y, last), leaf, (dy, dlast))
    for _ in range(6):
        d = torch.randint(-1, 2, x.shape, generator=gen).float().to(hip_device)     # exact sums
        up, down = (x + step * d), (x - step * d)
        slope = (value(*memfast.gated_recurrence(up, state)) -
                 value(*memfast.gated_recurrence(down, state))) / (2 * step)
        exact, noise = [], 0.0
        for at in (up, down):
            ref = reference(at, state, None, False, True)
            exact.append(value(ref["y"][0], ref["last"][0]))
            noise += float((ref["y"][1] * dy.double().cpu().abs()).sum() +
                           (ref["last"][1] * dlast.double().cpu().abs()).sum())
        along = float((expected["dx"][0] * d.double().cpu()).sum())
        truncation = abs((exact[0] - exact[1]) / (2 * step) - along)
        got = float((dx.double() * d.double()).sum())
        allowed = truncation + noise / step + float((2 * expected["dx"][1]).sum())
        assert abs(got - slope) <= allowed, (got, slope, allowed)


# ---------------------------------------------------------------------------
# Streams, graphs, autograd
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("steps", [1, 50, 700])
def test_captured_and_replayed(hip_device, steps):
    x, state, dy, dlast = case(hip_device, steps, 2, 24, "bf16")
    inputs = [case(hip_device, steps, 2, 24, "bf16", seed=s) for s in range(3)]

    def call(x, state, dy, dlast):
        leaf, start = x.detach().requires_grad_(True), state.detach().requires_grad_(True)
        y, last = memfast.gated_recurrence(leaf, start)
        return (y.detach(), last.detach(), *torch.autograd.grad((y, last), (leaf, start), (dy, dlast)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(x, state, dy, dlast)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    held = [t.clone() for t in (x, state, dy, dlast)]
    with torch.cuda.graph(graph):
        outputs = call(*held)
    for given in inputs * 2:
        for a, b in zip(held, given):
            a.copy_(b)
        graph.replay()
        expected = call(*given)                               # eager work between replays
        torch.cuda.synchronize()
        for a, b in zip(outputs, expected):
            assert torch.equal(a, b)


def test_another_stream(hip_device):
    x, state, _, _ = case(hip_device, 700, 2, 24, "fp32")
    expected = memfast.gated_recurrence(x, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device=hip_device)
        for _ in range(20):
            big = big @ big * 1e-3                             # x is ready only behind this
        late = x + 0 * big[0, 0].clamp(-1, 1).nan_to_num()
        results = [memfast.gated_recurrence(late, state) for _ in range(2)]   # two calls at once
    torch.cuda.current_stream().wait_stream(side)
    for result in results:
        assert torch.equal(result[0], expected[0]) and torch.equal(result[1], expected[1])


def test_autograd_keeps_its_promises(hip_device):
    x, state, dy, dlast = case(hip_device, 200, 2, 8, "fp32")
    leaf = x.clone().requires_grad_(True)
    y, last = memfast.gated_recurrence(leaf, state)
    first = torch.autograd.grad((y, last), leaf, (dy, dlast), retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad((y, last), leaf, (dy, dlast))[0])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaf, dy)
    leaf = x.clone().requires_grad_(True)
    moved = leaf * 1
    y, _ = memfast.gated_recurrence(moved, state)
    moved.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, dy)
    y, _ = memfast.gated_recurrence(leaf, state)
    y.mul_(2)                                                 # the states are not what is kept
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0],
                       torch.autograd.grad(memfast.gated_recurrence(leaf, state)[0], leaf, 2 * dy)[0])
    y, _ = memfast.gated_recurrence(leaf, state)
    dx, = torch.autograd.grad(y, leaf, dy, create_graph=True)
    assert torch.equal(dx, torch.autograd.grad(memfast.gated_recurrence(leaf, state)[0], leaf, dy)[0])
    with pytest.raises(NotImplementedError, match="no second derivative"):
        torch.autograd.grad(dx.sum() + leaf.sum(), leaf)


def test_many_sequences_and_wide_rows(hip_device):
    """More workgroups than one launch takes, and steps and sequences more than 2^31 values apart."""
    batch = (1 << 21) + 5
    x = torch.randn(1, batch, 2, device=hip_device)
    y, last = memfast.gated_recurrence(x, activation=None)
    expected = torch.sigmoid(-x[..., :1].double()) * x[..., 1:].double()
    assert bool(((y.double() - expected).abs() <= 32 * E * expected.abs() + 1e-37).all())
    assert torch.equal(last, y[0])
    far = torch.zeros((1 << 31) + 64, dtype=torch.bfloat16, device=hip_device)
    small = torch.randn(2, 2, 8, device=hip_device).bfloat16()
    for strides in ((1 << 31, 16), (16, 1 << 31)):
        view = far.as_strided((2, 2, 8), (strides[0], strides[1], 1))
        view.copy_(small)
        assert torch.equal(memfast.gated_recurrence(view)[0], memfast.gated_recurrence(small)[0])


# ---------------------------------------------------------------------------
# The layer
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_layer(hip_device, first, both):
    """Projections, recurrences and dropout of a stacked layer, written out."""
    torch.manual_seed(1)
    layer = GatedRecurrence(12, 10, 2, dropout=0.25, bidirectional=both, batch_first=first).to(hip_device)
    ways = 2 if both else 1
    x = torch.randn(4, 30, 12, device=hip_device) if first else torch.randn(30, 4, 12, device=hip_device)
    lengths = torch.tensor([30, 7, 0, 12], device=hip_device)
    hx = torch.randn(2 * ways, 4, 10, device=hip_device)
    torch.manual_seed(4)
    y, last = layer(x, hx, lengths)
    torch.manual_seed(4)
    seed = int(torch.randint(1 << 62, ()))
    h, finals = x, []
    for n in range(2):
        outputs = []
        for d in range(ways):
            projected = torch.nn.functional.linear(h, layer.projections[n * ways + d].weight,
                                                   layer.projections[n * ways + d].bias)
            states, final = memfast.gated_recurrence(projected, hx[n * ways + d], lengths=lengths,
                                                     reverse=d == 1, batch_first=first)
            outputs.append(states)
            finals.append(final)
        h = torch.cat(outputs, -1)
        if n == 0:
            h = memfast.dropout(h, 0.25, seed=seed)
    assert torch.equal(y, h) and torch.equal(last, torch.stack(finals))
    y.sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in layer.parameters())
    layer.eval()
    assert torch.equal(layer(x, hx, lengths)[0], layer(x, hx, lengths)[0])


def test_trained_held_and_stepped(hip_device):
    """The operators as they are used together: a training step with dropout, then the projections held
    in 4 bits and the layer run token by token, which is the layer on the whole sequence."""
    torch.manual_seed(2)
    layer = GatedRecurrence(64, 48, 2, dropout=0.1).to(hip_device)
    x = torch.randn(20, 3, 64, device=hip_device)
    optimizer = torch.optim.SGD(layer.parameters(), lr=0.01)
    layer(x)[0].square().mean().backward()
    optimizer.step()
    layer.eval()
    with torch.no_grad():
        for n, projection in enumerate(layer.projections):
            held = memfast.int4_quantize(projection.weight)
            near_weight = held.dequantize()
            assert float((near_weight - projection.weight).abs().max()) <= float(
                held.scales.max()) * 0.5001
            layer.projections[n] = Int4Linear(projection)
        whole, last = layer(x)
        hx, rows = None, []
        for t in range(len(x)):
            y, hx = layer(x[t:t + 1], hx)
            rows.append(y)
    # Sums over 64 and 48 inputs are split in the same way for 3 rows and 60, up to FP32 rounding: values of
    # order 1 and 20 steps of it.
    assert float((torch.cat(rows) - whole).abs().max()) < 1e-4
    assert float((hx - last).abs().max()) < 1e-4


@pytest.mark.parametrize("training", [False, True])
def test_converted_projections(hip_device, training):
    """convert_model makes the projections analog; one read of a sequence a layer."""
    torch.manual_seed(3)
    config = memfast.Config(activation_bits=8, weight_bits=8, input_slice=(1, 1, 2, 2, 2),
                            weight_slice=(1, 1, 2, 2, 2), array_size=(128, 128), rows_per_read=32,
                            weight_quant_gran=(32, 1), input_quant_gran=(1, 32),
                            nonidealities=memfast.Nonidealities(write_variation=0.0))
    simulator = memfast.Simulator(config, device=hip_device)
    layer = GatedRecurrence(32, 16, 2).to(hip_device)
    model = memfast.convert_model(layer, simulator, training=training)
    x = torch.randn(9, 2, 32, device=hip_device)
    if training:
        model.train()
        y, _ = model(x)
        y.sum().backward()
        assert all(p.grad is not None for p in model.parameters())
    else:
        with torch.no_grad():
            y, _ = model(x)
        assert all(p._event == 1 for p in model.projections)
    # 8-bit operands: steps of 1/127 of a group's peak, sums of 32, two layers.
    digital = layer(x)[0].detach()
    assert float((y.detach() - digital).abs().max()) < 0.15
