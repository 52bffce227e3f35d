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
