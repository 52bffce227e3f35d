"""The largest logits and the distillation loss against their definitions in 64 bits.

Tolerances.  Values and indices of the largest logits are compared exactly.  The exponents are
formed in FP32 as powers of two: with M the largest magnitude of a row's logits in that scale,
one carries an error of at most D = (4 M + 64) * 2**-24 (the scaling factor and the scaled value
are each rounded, the exponential and the logarithm are good to about an ulp, and a sum of
nonnegative terms in a tree or in runs of up to 2**10 adds a few 2**-24 of itself, 2**-19 at most).
So a probability is within E = D + 2**-18 of itself, the logarithm of a quotient of two within
2 E, and the loss within T**2 * sum |p - q| * 2 E plus E of each of its terms.
"""

import math

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def say(*args):
    print("[distillation]", *args, flush=True)


def logits(n, v, dtype, device, seed=0, scale=3.0):
    gen = torch.Generator().manual_seed(seed + 7919 * n + v)
    return (scale * torch.randn(n, v, generator=gen)).to(dtype).to(device)


def exponent_error(s, temperature):
    finite = torch.where(torch.isfinite(s), s, 0.0)
    m = finite.abs().amax(-1) * (1.4427 / temperature)
    return (4 * m + 64) * 2.0**-24 + 2.0**-18


# ---------------------------------------------------------------------------
# The largest logits
# ---------------------------------------------------------------------------
def check_top(s, k, temperature):
    values, indices, tail = memfast.top_logits(s, k, temperature=temperature)
    rows = s.detach().cpu().reshape(-1, s.shape[-1]).double() + 0.0
    ordered, at = torch.sort(rows, dim=1, descending=True, stable=True)
    # torch sorts a NaN as the largest value too.
    assert values.dtype == s.dtype and indices.dtype == torch.int64 and tail.dtype == torch.float32
    assert values.shape == indices.shape == s.shape[:-1] + (k,) and tail.shape == s.shape[:-1]
    assert torch.equal(indices.cpu().reshape(-1, k), at[:, :k])
    got = values.cpu().reshape(-1, k).double()
    assert torch.equal(torch.nan_to_num(got, nan=777.0), torch.nan_to_num(ordered[:, :k], nan=777.0))
    expected = torch.logsumexp(ordered[:, k:] / temperature, 1)
    got = tail.cpu().reshape(-1).double()
    fine = torch.isfinite(expected)
    assert torch.equal(got[~fine].isnan(), expected[~fine].isnan())
    minus = expected == -math.inf
    assert torch.equal(got[minus], expected[minus])
    bound = exponent_error(rows, temperature) + 2.0**-22 * expected.abs()
    assert bool(((got - expected).abs() <= bound)[fine].all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 64), (4, 1000, 10),
                                   (1, 50001, 20), (3, 4096, 1024), (2, 1500, 1024), (9, 32000, 64),
                                   (2, 131072, 256), (300, 129, 5), (1, 1 << 20, 33)])
def test_top(hip_device, kind, n, v, k):
    say("top", kind, n, v, k)
    check_top(logits(n, v, TYPES[kind], hip_device), k, 2.0)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v,k", [(1000, 10), (40000, 100), (131072, 1024)])
def test_top_of_equal_and_ordered_rows(hip_device, kind, v, k):
    """Ties across the cut, rows in either order, rows of few distinct values, all in one stretch."""
    dtype = TYPES[kind]
    ramp = torch.linspace(-8, 8, v)
    s = torch.stack((torch.zeros(v), ramp, ramp.flip(0), (torch.arange(v) % 3).float(),
                     torch.where(torch.arange(v) < 2 * k, 5.0, -5.0),
                     torch.where(torch.arange(v) >= v - 2 * k, 5.0, -5.0),
                     torch.where(torch.arange(v) % 64 == 5, 5.0, -5.0),
                     -torch.zeros(v)))
    s[7, ::2] = 0.0
    check_top(s.to(dtype).to(hip_device), k, 1.0)


def test_top_of_rows_with_infinities_and_nan(hip_device):
    s = logits(6, 3001, torch.float32, hip_device)
    s[0, 5:] = -math.inf                  # fewer finite values than entries
    s[1] = -math.inf
    s[2, 17] = math.inf
    s[3, 100] = float("nan")
    s[3, 200] = -float("nan")
    s[4, ::2] = -math.inf
    s[5, 3:] = torch.finfo(torch.float32).min
    check_top(s, 20, 1.0)


@pytest.mark.parametrize("kind", list(TYPES))
def test_top_of_strided_rows(hip_device, kind):
    base = logits(7, 4103, TYPES[kind], hip_device)
    for s in (base[:, 1:], base[:, 5:4000], base[::2], base.T[:4000].T, base[3], base[:6].reshape(2, 3, -1),
              base[:1].expand(4, 4103), base[:, :1].expand(7, 50)):
        check_top(s, 9, 0.5)
    assert memfast.top_logits(base[:0], 3)[0].shape == (0, 3)


# ---------------------------------------------------------------------------
# The loss
# ---------------------------------------------------------------------------
def oracle(s, values, indices, tail, temperature, weight, reduction, incoming=None):
    """(loss, gradient, bound of the loss's rows, bound of the gradient) in 64 bits on the CPU."""
    s = s.detach().cpu().double().requires_grad_(True)
    n, v = s.shape
    kept = indices.cpu() >= 0
    t = (values.cpu().double() / temperature).masked_fill(~kept, -math.inf)
    rest = torch.full((n, 1), -math.inf, dtype=torch.float64) if tail is None else \
        tail.cpu().double()[:, None]
    t = torch.cat((t, rest), 1)
    empty = (t == -math.inf).all(1)
    t = torch.where(empty[:, None], 0.0, t)
    log_p = torch.log_softmax(t, 1)
    z = s / temperature
    log_all = torch.log_softmax(z, 1)
    at = indices.cpu().clamp(min=0).long()
    inside = torch.zeros(n, v, dtype=torch.int64).scatter_add_(1, at, kept.long()) > 0
    others = log_all.masked_fill(inside, -math.inf)
    none = (others == -math.inf).all(1, keepdim=True)     # torch's logsumexp has no gradient there
    bucket = torch.logsumexp(torch.where(none, 0.0, others), 1, keepdim=True)
    bucket = torch.where(none, -math.inf, bucket)
    log_q = torch.cat((log_all.gather(1, at), bucket), 1)
    present = log_p > -math.inf
    terms = torch.where(present, log_p.exp() * (log_p.clamp(min=-1e300) -
                                                torch.where(present, log_q, 0.0)), 0.0)
    rows = torch.where(empty, 0.0, terms.sum(1) * temperature**2)
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.cpu().double()
    weighted = torch.where(w == 0, 0.0, w * rows)
    loss = {"none": weighted, "sum": weighted.sum(),
            "mean": weighted.sum() / w.sum() if float(w.sum()) else weighted.sum() * 0}[reduction]
    grad, = torch.autograd.grad(loss, s, torch.ones_like(loss) if incoming is None
                                else incoming.cpu().double())
    error = exponent_error(s.detach(), temperature) + exponent_error(t * temperature, temperature)
    p, q = log_p.exp(), torch.where(torch.cat((kept, torch.ones(n, 1, dtype=torch.bool)), 1),
                                    log_q.exp(), 0.0).detach()
    spread = (p - q).abs().sum(1)
    row_bound = temperature**2 * error * (2 * spread + 2 * error) + 4 * error * rows.detach().abs()
    share = {"none": w, "sum": w, "mean": w / w.sum() if float(w.sum()) else w * 0}[reduction].abs()
    if incoming is not None:
        share = share * incoming.cpu().double().abs()
    # q and p_c (or p_r q / q_r) are each within 2 E of themselves.
    most = log_all.exp().detach()
    most = most + torch.where(inside, 0.0, (p[:, -1:] * torch.exp(log_all - bucket)).nan_to_num(0)).detach()
    most = most.scatter_add(1, at, torch.where(kept, p[:, :-1], 0.0))
    grad_bound = (temperature * share * 2 * error)[:, None] * most
    return loss.detach(), grad, row_bound * share, grad_bound


def check_loss(s, values, indices, tail=None, *, temperature=1.0, weight=None, reduction="mean",
               incoming=None):
    s = s.detach().requires_grad_(True)
    loss = memfast.distillation_loss(s, values, indices, tail, temperature=temperature,
                                     weight=weight, reduction=reduction)
    given = incoming if incoming is not None else torch.ones_like(loss)
    grad, = torch.autograd.grad(loss, s, given)
    expected, slope, row_bound, grad_bound = oracle(s, values, indices, tail, temperature, weight,
                                                    reduction, incoming)
    assert loss.dtype == torch.float32 and grad.dtype == s.dtype and grad.shape == s.shape
    bound = row_bound if reduction == "none" else row_bound.sum()
    if incoming is not None and reduction == "none":
        bound = bound / incoming.cpu().double().abs().clamp(min=1e-30)
    off = (loss.detach().cpu().double() - expected).abs()
    assert bool((off <= bound + 2.0**-22 * expected.abs() + 2.0**-126).all()), (loss, expected, bound)
    off = (grad.cpu().double() - slope).abs()
    allowed = grad_bound + UNIT[s.dtype] * slope.abs() * (1 + 2.0**-7) + TINY[s.dtype]
    assert bool((off <= allowed).all()), float((off / allowed).max())
    return loss.detach(), grad


def teacher_of(s, k, temperature, noise=1.0, seed=3):
    gen = torch.Generator().manual_seed(seed)
    t = s.detach().float().cpu() + noise * torch.randn(s.shape, generator=gen)
    return memfast.top_logits(t.to(s.device), k, temperature=temperature)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (2, 2, 1), (3, 5, 5), (4, 33, 7), (32, 1000, 10),
                                   (5, 4097, 64), (3, 32000, 256), (2, 50001, 100),
                                   (2, 131072, 64), (2, 70000, 1024), (200, 100, 3),
                                   (2, 140001, 20), (1, 1 << 20, 40)])
@pytest.mark.parametrize("tail", [False, True])
def test_loss_and_gradient(hip_device, kind, n, v, k, tail):
    say("loss", kind, n, v, k, tail)
    s = logits(n, v, TYPES[kind], hip_device)
    for temperature in (1.0, 3.0):
        values, indices, rest = teacher_of(s, k, temperature)
        check_loss(s, values, indices, rest if tail else None, temperature=temperature)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [257, 20000, 140001])
def test_weights_reductions_and_incoming_gradients(hip_device, kind, v):
    n = 6
    s = logits(n, v, TYPES[kind], hip_device)
    values, indices, rest = teacher_of(s, 12, 2.0)
    weight = torch.tensor([1.0, 0.0, 0.25, 2.0, 0.0, 1.0], device=hip_device)
    for w in (None, weight, weight > 0, weight * 0, weight.half()):
        for reduction in ("mean", "sum", "none"):
            shape = (n,) if reduction == "none" else ()
            scale = torch.linspace(0.5, 2.0, n, device=hip_device) if shape else \
                torch.tensor(1.7, device=hip_device)
            loss, grad = check_loss(s, values, indices, rest, temperature=2.0, weight=w,
                                    reduction=reduction, incoming=scale)
            if w is not None:
                assert not grad[w == 0].any()
    # Unit and other incoming gradients, and a second backward through one graph.
    leaf = s.clone().requires_grad_(True)
    loss = memfast.distillation_loss(leaf, values, indices, rest, temperature=2.0)
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = one.clone()
    one.zero_()                                     # the caller's own tensor
    two, = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device=hip_device), retain_graph=True)
    again, = torch.autograd.grad(loss, leaf)
    assert torch.equal(again, kept)
    assert bool(((two.double() - 2 * kept.double()).abs() <=
                 2 * UNIT[s.dtype] * 2 * kept.double().abs() + 2 * TINY[s.dtype]).all())


@pytest.mark.parametrize("v", [50, 5000, 140001])
def test_absent_entries_and_rows_without_any(hip_device, v):
    n, k = 8, 6
    s = logits(n, v, torch.float32, hip_device)
    values, indices, rest = teacher_of(s, k, 1.0)
    gen = torch.Generator().manual_seed(1)
    lost = (torch.rand(n, k, generator=gen) < 0.5).to(hip_device)
    lost[0], lost[1] = True, False
    indices = indices.masked_fill(lost, -1)
    values = values.masked_fill(lost, float("nan"))           # never looked at
    loss, grad = check_loss(s, torch.where(lost, 0.0, values), indices, rest, reduction="none")
    again = memfast.distillation_loss(s, values, indices, rest, reduction="none")
    assert torch.equal(loss, again)
    loss, grad = check_loss(s, torch.where(lost, 0.0, values), indices, reduction="none")
    assert float(loss[0]) == 0.0 and not grad[0].any()
    only = torch.full_like(indices, -1)
    loss, grad = check_loss(s, torch.zeros_like(values), only, reduction="sum")
    assert float(loss) == 0.0 and not grad.any()


@pytest.mark.parametrize("v", [40, 9000, 140001])
def test_wrong_indices_make_their_row_nan(hip_device, v):
    n, k = 6, 5
    s = logits(n, v, torch.float32, hip_device).requires_grad_(True)
    values, indices, rest = teacher_of(s, k, 1.0)
    clean, = torch.autograd.grad(memfast.distillation_loss(s, values, indices, rest, reduction="sum"), s)
    bad = indices.clone()
    bad[0, 1], bad[1, 2], bad[2, 0] = v, -2, 1 << 40
    bad[3, 4] = bad[3, 0]                                     # twice the same class
    loss = memfast.distillation_loss(s, values, bad, rest, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), s)
    assert loss[:4].isnan().all() and torch.isfinite(loss[4:]).all()
    assert grad[:4].isnan().all() and torch.equal(grad[4:], clean[4:])
    weight = torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0, 1.0], device=hip_device)
    loss = memfast.distillation_loss(s, values, bad, rest, weight=weight)
    grad, = torch.autograd.grad(loss, s)
    assert torch.isfinite(loss) and not grad[:4].any()


@pytest.mark.parametrize("v", [60, 6000, 140001])
def test_non_finite_logits(hip_device, v):
    n, k = 8, 4
    s = logits(n, v, torch.float32, hip_device)
    values, indices, rest = teacher_of(s, k, 1.0)
    low = torch.ones_like(s, dtype=torch.bool).scatter_(1, indices, False)
    s[0] = torch.where(low[0] & (torch.arange(v, device=hip_device) % 2 == 0), -math.inf, s[0])
    s[1] = torch.where(low[1], torch.finfo(torch.float32).min, s[1])
    s[2] = torch.where(low[2], -math.inf, s[2])               # no mass outside the entries
    check_loss(s[:2], values[:2], indices[:2], rest[:2], reduction="none")
    check_loss(s[:3], values[:3], indices[:3], reduction="none")
    minus = rest.clone()
    minus[:] = -math.inf
    check_loss(s[:3], values[:3], indices[:3], minus[:3], reduction="none")
    # An entry of the teacher that the student excludes, a NaN, an infinity.
    s[3, indices[3, 0]] = -math.inf
    s[4, v // 2] = float("nan")
    s[5, v // 3] = math.inf
    s[6] = -math.inf
    leaf = s.clone().requires_grad_(True)
    loss = memfast.distillation_loss(leaf, values, indices, rest, reduction="none")
    assert float(loss[3]) == math.inf and loss[4:7].isnan().all() and torch.isfinite(loss[7])
    # Rows that do not count do not show.
    weight = (torch.arange(n, device=hip_device) == 7).float()
    total = memfast.distillation_loss(leaf, values, indices, rest, weight=weight)
    assert float(total) == float(loss[7])
    grad, = torch.autograd.grad(total, leaf)
    assert not grad[:7].any() and torch.isfinite(grad[7]).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [501, 4103, 33333])
def test_strided_operands(hip_device, kind, v):
    dtype = TYPES[kind]
    base = logits(6, v, dtype, hip_device)
    for s in (base[:, 1:], base[:, 3:v - 4], base[::2], base.T.contiguous().T):
        values, indices, rest = teacher_of(s, 8, 1.0)
        wide = torch.zeros(len(s), 20, device=hip_device)
        wide[:, 3:11] = values
        loss, grad = check_loss(s, values, indices, rest)
        check_loss(s.clone(memory_format=torch.contiguous_format), values, indices, rest)
        other = s.detach().requires_grad_(True)
        again = memfast.distillation_loss(other, wide[:, 3:11], indices.int().T.contiguous().T,
                                          rest.double())
        assert torch.equal(again.detach(), loss)
        same, = torch.autograd.grad(again, other)
        assert torch.equal(same, grad)
    s = base.reshape(2, 3, v)
    values, indices, rest = memfast.top_logits(s, 4)
    loss = memfast.distillation_loss(s, values, indices, rest, reduction="none")
    assert loss.shape == (2, 3)
    empty = memfast.distillation_loss(base[:0], values.reshape(-1, 4)[:0], indices.reshape(-1, 4)[:0])
    assert empty.shape == () and float(empty) == 0.0


def test_values_of_another_type(hip_device):
    s = logits(5, 700, torch.bfloat16, hip_device)
    values, indices, rest = teacher_of(s, 6, 1.0)             # FP32 teacher, BF16 student
    assert values.dtype == torch.float32
    check_loss(s, values, indices, rest)
    check_loss(s.float(), values.bfloat16(), indices, rest)
    check_loss(s.half(), values.half(), indices, rest)


def test_a_student_near_its_teacher(hip_device):
    """A loss far below the rounding of its logarithms keeps its leading digits."""
    s = logits(64, 1000, torch.float32, hip_device)
    for noise in (1e-1, 1e-2):
        values, indices, rest = teacher_of(s, 10, 4.0, noise=noise)
        loss = memfast.distillation_loss(s, values, indices, rest, temperature=4.0)
        expected = oracle(s, values, indices, rest, 4.0, None, "mean")[0]
        assert abs(float(loss) - float(expected)) <= 2e-3 * float(expected)
    values, indices, rest = memfast.top_logits(s, 10)
    loss, grad = check_loss(s, values, indices, rest)
    assert float(loss) < 1e-9


def test_gradient_against_differences(hip_device):
    """Central differences of the FP32 loss along random directions.  With steps of h = 2**-4 the
    cubic term is below h**2 / 6 of the third derivative's size (at most 1 here, as the direction's
    entries are signs), and the loss's own error below 1e-5 is divided by 2 h."""
    s = logits(4, 300, torch.float32, hip_device, scale=1.0)
    values, indices, rest = teacher_of(s, 8, 1.0)
    leaf = s.clone().requires_grad_(True)
    loss = memfast.distillation_loss(leaf, values, indices, rest, reduction="sum")
    grad, = torch.autograd.grad(loss, leaf)
    gen = torch.Generator().manual_seed(2)
    h = 2.0**-4
    for _ in range(8):
        u = (2.0 * torch.randint(2, s.shape, generator=gen) - 1).to(hip_device)
        up, down = (memfast.distillation_loss(s + d * u, values, indices, rest, reduction="sum")
                    for d in (h, -h))
        quotient = (float(up) - float(down)) / (2 * h)
        slope = float((grad.double() * u.double()).sum())
        assert abs(quotient - slope) <= 4 * h**2 / 6 + 1e-5 / (2 * h)


def test_streams_and_repeated_results(hip_device):
    s = logits(40, 9000, torch.bfloat16, hip_device).requires_grad_(True)
    values, indices, rest = teacher_of(s, 16, 1.0)

    def step():
        loss = memfast.distillation_loss(s, values, indices, rest)
        return (loss.detach(), *torch.autograd.grad(loss, s), *memfast.top_logits(s, 16))

    first = step()
    side = torch.cuda.Stream(hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream(hip_device).wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)
