"""Dropout's counter where the number of a block of eight values passes 32 bits."""

import pytest
import torch

import memfast_amd as memfast
from test_gpu_dropout import mask

pytestmark = pytest.mark.gpu


def test_blocks_beyond_32_bits(hip_device):
    """From value 2^35 on the counter's second word is 1."""
    n = (1 << 35) + 8 * 1024 + 3
    if torch.cuda.mem_get_info(hip_device)[0] < 5 * n:
        pytest.skip("needs 160 GiB of device memory")
    x = torch.ones(n, dtype=torch.bfloat16, device=hip_device)
    y = memfast.dropout(x, 0.5, seed=5, event=3)
    for first in (0, (1 << 32) - 16, (1 << 34) - 16, (1 << 35) - 32, (1 << 35), n - 100):
        count = min(64, n - first)
        assert torch.equal(y[first:first + count].cpu() != 0, mask(count, 0.5, 5, 3, first))
    # The second word counts: the first blocks' masks are others.
    assert not torch.equal(y[1 << 35:(1 << 35) + 64], y[:64])
    del x, y
    torch.cuda.empty_cache()
