"""The largest logits where the rows fill the chip, and around the sizes at which the work is split.

Each pattern's row is checked against its definition in 64 bits, and every repetition of it has to be
the same bits.  The logarithm of the others' sum is within the bound that
tests/test_gpu_distillation.py derives: exponents in FP32 within D = (4 M + 64) * 2**-24, M the largest
magnitude of the row's logits as a power of two, the sum within 2**-18 of itself, and the result rounded.
"""

import math

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def patterns(v, k):
    gen = torch.Generator().manual_seed(v + k)
    s = 3.0 * torch.randn(16, v, generator=gen)
    ramp = torch.linspace(-8, 8, v)
    at = torch.arange(v)
    s[4], s[5], s[6] = 0.0, ramp, ramp.flip(0)
    s[7] = (at % 3).float()                             # many ties across the cut
    s[8] = torch.where(at >= v - k, 5.0, -5.0)          # all at the row's end
    s[9] = torch.where(at < k, 5.0, -5.0)               # or at its start
    s[10] = -math.inf
    s[11, : v - max(k // 2, 1)] = -math.inf             # fewer finite values than entries
    s[12, ::2] = -math.inf
    s[13, v // 2] = math.inf
    s[14, v // 3] = math.nan
    s[15, 1:] = -3.0e38 if v > 1 else 0.0
    return s


def check(s, k, temperature, repeats):
    many = s.repeat(repeats, 1)
    values, indices, tail = memfast.top_logits(many, k, temperature=temperature)
    for part in (values, indices, tail):
        rows = part.reshape(repeats, len(s), -1)
        same = (rows == rows[:1]) | (rows != rows) & (rows[:1] != rows[:1])
        assert bool(same.all())
    rows = s.cpu().double() + 0.0
    ordered, at = torch.sort(rows, dim=1, descending=True, stable=True)
    assert torch.equal(indices[:len(s)].cpu(), at[:, :k])
    got = values[:len(s)].cpu().double()
    assert torch.equal(torch.nan_to_num(got, nan=777.0), torch.nan_to_num(ordered[:, :k], nan=777.0))
    expected = torch.logsumexp(ordered[:, k:] / temperature, 1).float().double()    # its type's range
    got = tail[:len(s)].cpu().double()
    fine = torch.isfinite(expected)
    assert torch.equal(got[~fine].isnan(), expected[~fine].isnan())
    assert torch.equal(got[expected == -math.inf], expected[expected == -math.inf])
    # Only what the sum is made of counts: the others' largest and what is near it.
    largest = ordered[:, k].abs() if k < rows.shape[1] else torch.zeros(len(s))
    m = torch.where(torch.isfinite(largest), largest + 128, 0.0) * (1.4427 / temperature)
    bound = (4 * m + 64) * 2.0**-24 + 2.0**-18 + 2.0**-22 * expected.abs()
    off = (got - expected).abs()[fine]
    assert bool((off <= bound[fine]).all()), (off / bound[fine]).max()


def typed(s, dtype, device):
    top = torch.finfo(dtype).max
    return torch.where(torch.isfinite(s), s.clamp(-top, top), s).to(dtype).to(device)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v,k", [(130, 3), (511, 64), (513, 65), (1031, 64), (1031, 200), (2049, 128), (2049, 129),
                                 (4097, 1), (16391, 128), (16391, 256), (33001, 64), (33001, 257),
                                 (70003, 64), (70003, 128), (70003, 129), (70003, 700)])
def test_rows_that_fill_the_chip(hip_device, kind, v, k):
    print("[top-logits]", kind, v, k, flush=True)
    check(typed(patterns(v, k), TYPES[kind], hip_device), k, 2.0, 33)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v,k", [(64, 9), (130, 128), (1031, 129), (4097, 129), (8193, 64), (33001, 1024)])
def test_few_rows(hip_device, kind, v, k):
    print("[top-logits]", kind, v, k, flush=True)
    check(typed(patterns(v, k), TYPES[kind], hip_device), k, 0.5, 2)


@pytest.mark.parametrize("offset", [1, 3, 7])
def test_rows_that_start_inside_a_piece(hip_device, offset):
    base = typed(patterns(20011, 50), torch.bfloat16, hip_device)
    s = base[:, offset:20003]
    check(s.contiguous(), 50, 1.0, 33)
    many = base.repeat(33, 1)[:, offset:20003]
    for here, there in zip(memfast.top_logits(many, 50)[:2], memfast.top_logits(many.contiguous(), 50)[:2]):
        assert torch.equal(torch.nan_to_num(here.double(), nan=777.0),
                           torch.nan_to_num(there.double(), nan=777.0))
