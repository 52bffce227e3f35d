"""The distillation operators at the edges of their ranges: rows with nothing outside their entries,
losses changed in place, infinite tails, the smallest temperature and more rows than one launch takes.

Bounds are those that tests/test_gpu_distillation.py derives; everything else is compared bit for bit.
"""

import math

import pytest
import torch
from test_gpu_distillation import TYPES, check_loss, logits, say, teacher_of

import memfast_amd as memfast

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Nothing outside the entries
# ---------------------------------------------------------------------------
def loss_and_gradient(s, values, indices, tail, **options):
    leaf = s.detach().requires_grad_(True)
    loss = memfast.distillation_loss(leaf, values, indices, tail, **options)
    return loss.detach(), torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [10, 1000, 20000])
def test_low_entries_with_nothing_outside_them(hip_device, kind, v):
    """Every other class is -inf (or there is none): the loss depends on differences of the entries
    alone. Steps and shifts are whole multiples of 32, exact in every type, so a shift, also to
    below exp's range at this temperature, changes no bit."""
    n, k, temperature = 4, 10, 5.0
    gen = torch.Generator().manual_seed(v)
    indices = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(n)]).to(hip_device)
    step = (32.0 * torch.randint(0, 9, (n, k), generator=gen)).to(hip_device)
    teacher = (step + 32.0 * torch.randint(0, 2, (n, k), generator=gen).to(hip_device)).to(TYPES[kind])
    no_tail = torch.full((n,), -math.inf, device=hip_device)
    for reduction in ("none", "mean"):
        for tail in (None, no_tail):
            results = []
            for shift in (0.0, -4096.0, 4096.0):
                s = torch.full((n, v), -math.inf, device=hip_device)
                s = s.scatter(1, indices, step + shift).to(TYPES[kind])
                results.append(loss_and_gradient(s, teacher, indices, tail, temperature=temperature,
                                                 reduction=reduction))
                check_loss(s, teacher, indices, tail, temperature=temperature, reduction=reduction)
            for loss, grad in results[1:]:
                assert torch.equal(loss, results[0][0]) and torch.equal(grad, results[0][1])


@pytest.mark.parametrize("shift,temperature", [(-40.0, 0.05), (-72.0, 0.1), (-800.0, 1.0), (-1e5, 3.0)])
def test_all_classes_are_entries(hip_device, shift, temperature):
    s = logits(6, 10, torch.float32, hip_device, scale=temperature) + shift
    values, indices, rest = teacher_of(s, 10, temperature, noise=temperature)
    assert bool((rest == -math.inf).all())
    for tail in (None, rest):
        loss, grad = check_loss(s, values, indices, tail, temperature=temperature)
        assert bool(torch.isfinite(loss)) and bool(torch.isfinite(grad).all())


# ---------------------------------------------------------------------------
# A loss that is changed in place or kept
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("weighted", [False, True])
def test_losses_can_be_changed_in_place(hip_device, reduction, weighted):
    """Divided by a number of accumulation steps and joined by another loss, as training loops do."""
    n = 5
    s = logits(n, 700, torch.float32, hip_device)
    values, indices, rest = teacher_of(s, 6, 1.0)
    options = dict(reduction=reduction)
    if weighted:
        options["weight"] = torch.tensor([1.0, 0.0, 2.0, 0.5, 1.0], device=hip_device)

    def gradient(in_place):
        leaf = s.clone().requires_grad_(True)
        loss = memfast.distillation_loss(leaf, values, indices, rest, **options)
        other = 0.1 * leaf.square().mean()
        if in_place:
            loss /= 4
            loss += other
        else:
            loss = loss / 4 + other
        loss.sum().backward()
        return loss.detach(), leaf.grad

    for here, there in zip(gradient(True), gradient(False)):
        assert torch.equal(here, there)
    # Without a gradient too; what a caller does to a loss reaches no other result.
    loss = memfast.distillation_loss(s, values, indices, rest, **options)
    kept = loss.clone()
    loss.zero_()
    assert torch.equal(memfast.distillation_loss(s, values, indices, rest, **options), kept)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_kept_losses_hold_no_other_memory(hip_device, reduction):
    s = logits(40, 300, torch.float32, hip_device)
    values, indices, rest = teacher_of(s, 20, 1.0)
    for leaf in (s, s.clone().requires_grad_(True)):
        loss = memfast.distillation_loss(leaf, values, indices, rest, reduction=reduction).detach()
        assert loss.untyped_storage().nbytes() == 4 * loss.numel()


# ---------------------------------------------------------------------------
# Infinities among the others
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v,k", [(2, 1), (9, 2), (3001, 2), (3001, 64), (40000, 1), (70003, 129)])
@pytest.mark.parametrize("repeats", [1, 200])
def test_the_tail_of_infinite_logits(hip_device, kind, v, k, repeats):
    """log(sum(exp)) of others with +inf among them is +inf, with NaN it is NaN, and beside
    an infinity that is selected, or -inf, it is as finite as without."""
    s = torch.zeros(6, v)
    at = torch.arange(v)
    s[0] = torch.where(at >= v - (k + 1), math.inf, 0.0)      # one more than is selected
    s[1] = torch.where(at < k + 1, math.inf, -math.inf)
    s[2] = math.inf
    s[3] = torch.where(at % 2 == 0, math.nan, math.inf) if 2 * k < v else math.nan
    s[4] = torch.where(at < k, math.inf, 0.0)                 # all of them are selected
    s[5] = torch.where(at < k, math.nan, math.inf)            # every NaN is
    s = s.to(TYPES[kind]).to(hip_device).repeat(repeats, 1)
    values, indices, tail = memfast.top_logits(s, k, temperature=2.0)
    rows = s[:6].cpu().double()
    ordered, order = torch.sort(rows, dim=1, descending=True, stable=True)
    assert torch.equal(indices.cpu(), order[:, :k].repeat(repeats, 1))
    expected = torch.logsumexp(ordered[:, k:] / 2.0, 1)
    assert torch.equal(expected[:3], torch.full((3,), math.inf, dtype=torch.float64))
    got = tail.cpu().double().reshape(repeats, 6)
    assert torch.equal(got[:, [0, 1, 2, 5]], expected[[0, 1, 2, 5]].expand(repeats, 4))
    assert bool(expected[3].isnan()) and bool(got[:, 3].isnan().all())
    assert bool(((got[:, 4] - expected[4]).abs() <= 2.0**-17 + 2.0**-22 * expected[4].abs()).all())


def test_the_smallest_temperature(hip_device):
    """At 2**-126 the largest class has all the mass, and exponents stay finite."""
    temperature = 2.0**-126
    s = torch.arange(8.0, device=hip_device)[None] / 4
    values, indices, tail = memfast.top_logits(s, 2, temperature=temperature)
    assert indices.tolist() == [[7, 6]] and float(tail) == 1.25 * 2.0**126
    s = s * 2.0**-126
    values, indices, tail = memfast.top_logits(s, 2, temperature=temperature)
    check_loss(s, values, indices, temperature=temperature)


# ---------------------------------------------------------------------------
# More rows than one launch takes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_rows_past_a_launch(hip_device, reduction):
    """2**24 + 7 rows, one workgroup each: their threads pass 2**32. Every row has the bits of the
    same row among a few."""
    n, v, k, period = (1 << 24) + 7, 3, 1, 16
    say("rows", n, reduction)
    few = logits(period, v, torch.bfloat16, hip_device)
    many = few.repeat(-(-n // period), 1)[:n]

    def equal_rows(got, expected):
        whole = n // period * period
        assert torch.equal(got[:whole].reshape(-1, period, *got.shape[1:]),
                           expected.expand(n // period, *expected.shape))
        assert torch.equal(got[whole:], expected[:n - whole])

    top = memfast.top_logits(many, k)
    expected = memfast.top_logits(few, k)
    for a, b in zip(top, expected):
        equal_rows(a, b)
    teacher = [t.roll(1, 0) for t in expected]
    teachers = [t.repeat(-(-n // period), *[1] * (t.ndim - 1))[:n] for t in teacher]
    results = [loss_and_gradient(rows, *t, reduction=reduction)
               for rows, t in ((many, teachers), (few, teacher))]
    equal_rows(results[0][1], results[1][1])
    if reduction == "none":
        equal_rows(results[0][0], results[1][0])
    else:
        rows = memfast.distillation_loss(few, *teacher, reduction="none").double()
        total = rows.sum() * (n // period) + rows[:n % period].sum()
        # FP64 sums, rounded once.
        assert abs(float(results[0][0]) - float(total)) <= 2.0**-23 * float(total)
