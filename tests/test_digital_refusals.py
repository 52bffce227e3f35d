"""What the digital operators refuse before any device is asked, and say so."""

import pytest
import torch
from torch.autograd import forward_ad

import memfast_amd as memfast
from memfast_amd import hip


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("grads", [False, True])
def test_forward_mode_is_refused(grads):
    """A tangent is not dropped, with gradients recorded beside it or not."""
    x, w, b = torch.ones(2, 32), torch.ones(3, 32, requires_grad=grads), torch.ones(3)
    s, values, indices = torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64)
    s.requires_grad_(grads)
    with forward_ad.dual_level():
        for call in (lambda: memfast.mx_linear(dual(x), w, b), lambda: memfast.mx_linear(x, dual(w)),
                     lambda: memfast.mx_linear(x, w, dual(b)),
                     lambda: memfast.distillation_loss(dual(s), values, indices),
                     lambda: memfast.distillation_loss(s, dual(values), indices),
                     lambda: memfast.distillation_loss(s, values, indices, dual(torch.zeros(2))),
                     lambda: memfast.distillation_loss(s, values, indices, weight=dual(torch.ones(2)))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        # Without a tangent the device is asked for, as outside.
        with pytest.raises(hip.BackendError, match="HIP devices only"):
            memfast.mx_linear(x, w, b)
        with pytest.raises(hip.BackendError, match="HIP devices only"):
            memfast.distillation_loss(s, values, indices)


def test_temperatures_whose_reciprocal_is_infinite():
    """1 / T is formed in FP32."""
    s, values, indices = torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64)
    for temperature in (1e-40, 1e-46, 2.0**-127, 1e39, 2.0**128, 10**400):
        with pytest.raises(ValueError, match="temperature"):
            memfast.top_logits(s, 1, temperature=temperature)
        with pytest.raises(ValueError, match="temperature"):
            memfast.distillation_loss(s, values, indices, temperature=temperature)
    for temperature in (2.0**-126, 1, 3.4e38):
        with pytest.raises(hip.BackendError, match="HIP devices only"):
            memfast.top_logits(s, 1, temperature=temperature)
    # The library itself, on host memory that it refuses before it launches anything.
    top = hip.library().mf_top_logits
    at = s.data_ptr()
    for temperature in (1e-40, 0.0, -1.0, float("nan"), float("inf")):
        assert top(at, 0, 2, 8, 8, 1, temperature, at, at, at, None) == hip.E_INVALID
