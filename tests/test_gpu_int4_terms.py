"""FP32 inputs of the 4-bit product count with all of their 24 bits.

A row of x has one number that is not 0, with its lowest bit set, and every weight is 1. With codes of 1 and
zero points of 0 the three terms of the number add up to it exactly at every addition (each is the number's
next eight bits), so the result is the number. With zero points of z and codes of z + 1 the sums hold up to
16 |x|: a dozen additions of at most 2^-24 of that each, 192 2^-24 |x| or 2^-16.4; the third term alone, times its
code, is up to 16 2^-16 |x| and, with all bits set, at least (z + 1) 2^-16.1 |x|.
"""

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu

# Few rows, small tiles of 32 and 64 rows, wide tiles.
SIZES = [(1, 40), (5, 40), (16, 8200), (30, 40), (60, 40), (24, 9000), (40, 1100), (100, 1000), (260, 1100),
         (65, 4200), (1030, 300)]


def rows(n, k, device, seed):
    gen = torch.Generator().manual_seed(seed)
    mantissa = torch.randint(1 << 23, 1 << 24, (n,), generator=gen) | 1
    mantissa[::2] = (1 << 24) - 1
    sign = 1 - 2 * torch.randint(0, 2, (n,), generator=gen)
    value = (sign * mantissa).double() * 2.0**torch.randint(-50, 20, (n,), generator=gen).double()
    value = value.float()
    x = torch.zeros(n, k)
    x[torch.arange(n), torch.randint(0, k, (n,), generator=gen)] = value
    return x.to(device), value.to(device)


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("k", [256, 250, 1000, 1024])
@pytest.mark.parametrize("n,o", SIZES)
def test_all_bits_count(hip_device, n, o, k, group):
    groups = -(-k // group)
    x, value = rows(n, k, hip_device, n + k)
    for zero in (0, None, 3, 14):
        z = 8 if zero is None else zero
        codes = torch.full((o, k), z + 1, dtype=torch.uint8, device=hip_device)
        held = memfast.Int4Tensor.pack(
            codes, torch.ones(o, groups, device=hip_device), group=group,
            zeros=None if zero is None else torch.full((o, groups), z, device=hip_device))
        y = memfast.int4_linear(x, held)
        if zero == 0:
            assert torch.equal(y, value[:, None].expand(n, o))
        else:
            off = (y.double() - value.double()[:, None]).abs()
            assert bool((off <= 192 * 2.0**-24 * value.double().abs()[:, None]).all())
