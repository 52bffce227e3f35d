"""What the 4-bit operands and the distillation loss refuse before any device is asked."""

import pytest
import torch

import memfast_amd as memfast
from memfast_amd import hip


def test_tensor_parts():
    codes, scales = torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8)
    assert memfast.MXTensor(codes, scales, (2, 200)).shape == (2, 200)
    assert memfast.MXTensor(codes, scales, (2, 1, 256)).shape == (2, 1, 256)
    for bad, error in (((codes, scales, (2, 257)), ValueError), ((codes, scales, (3, 200)), ValueError),
                       ((codes.int(), scales, (2, 200)), TypeError), ((codes, None, (2, 200)), TypeError),
                       ((codes, scales, ()), ValueError)):
        with pytest.raises(error):
            memfast.MXTensor(*bad)


def test_quantize_and_linear():
    x = torch.zeros(2, 32)
    for bad in (x.double(), x.int(), [1.0], x.to_sparse()):
        with pytest.raises(TypeError):
            memfast.mx_quantize(bad)
        with pytest.raises(TypeError):
            memfast.mx_linear(bad, x)
        with pytest.raises(TypeError):
            memfast.mx_linear(x, x, bad)
    with pytest.raises(ValueError):
        memfast.mx_quantize(torch.tensor(1.0))
    with pytest.raises(ValueError, match="reduction"):
        memfast.mx_linear(x, torch.zeros(4, 31))
    with pytest.raises(ValueError, match="mx_linear takes"):
        memfast.mx_linear(x, torch.zeros(32))
    with pytest.raises(ValueError, match="same dtype"):
        memfast.mx_linear(x, x.bfloat16())
    for call in (lambda: memfast.mx_quantize(x), lambda: memfast.mx_linear(x, x)):
        with pytest.raises(hip.BackendError, match="HIP devices only"):
            call()


def test_top_logits():
    s = torch.zeros(2, 8)
    for k, error in ((0, ValueError), (9, ValueError), (1.0, TypeError), (True, TypeError)):
        with pytest.raises(error):
            memfast.top_logits(s, k)
    for temperature, error in ((0, ValueError), (-1.0, ValueError), (float("nan"), ValueError),
                               (float("inf"), ValueError), ("1", TypeError)):
        with pytest.raises(error):
            memfast.top_logits(s, 1, temperature=temperature)
    with pytest.raises(TypeError):
        memfast.top_logits(s.double(), 1)
    with pytest.raises(ValueError):
        memfast.top_logits(s[:, :0], 1)
    with pytest.raises(NotImplementedError):
        memfast.top_logits(torch.zeros(1, 2000), 1025)
    with pytest.raises(NotImplementedError):
        memfast.top_logits(torch.zeros(1, (1 << 20) + 1), 1)
    with pytest.raises(hip.BackendError, match="HIP devices only"):
        memfast.top_logits(s, 1)


def test_distillation_loss():
    s, values, indices = torch.zeros(2, 8), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    loss = memfast.distillation_loss
    for args, options, error in (
            ((s.double(), values, indices), {}, TypeError),
            ((s, values.double(), indices), {}, TypeError),
            ((s, values, indices.float()), {}, TypeError),
            ((s, values, indices[:, :2]), {}, ValueError),
            ((s, values[:1], indices[:1]), {}, ValueError),
            ((s, values[:, :0], indices[:, :0]), {}, ValueError),
            ((s[:, :2], values, indices), {}, ValueError),
            ((s, values, indices, torch.zeros(3)), {}, ValueError),
            ((s, values, indices, torch.zeros(2).int()), {}, TypeError),
            ((s, values, indices), dict(weight=torch.zeros(2, 1)), ValueError),
            ((s, values, indices), dict(weight=torch.zeros(2).int()), TypeError),
            ((s, values, indices), dict(reduction="max"), ValueError),
            ((s, values, indices), dict(temperature=0.0), ValueError),
            ((torch.zeros(1, 2000), torch.zeros(1, 1025), torch.zeros(1, 1025).long()), {},
             NotImplementedError)):
        with pytest.raises(error):
            loss(*args, **options)
    with pytest.raises(hip.BackendError, match="HIP devices only"):
        loss(s, values, indices)
