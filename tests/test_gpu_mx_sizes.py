"""The 4-bit product where its kernels change with the sizes."""

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu


def test_one_row_of_more_outputs_than_a_launch_takes(hip_device):
    """Outputs of 32 threads each would pass 2**32 threads."""
    o = (1 << 27) + 5
    print("[mx-sizes]", o, flush=True)
    w = (torch.arange(o, device=hip_device) % 7 - 3).bfloat16()[:, None]
    x = torch.full((1, 1), 0.5, dtype=torch.bfloat16, device=hip_device)
    y = memfast.mx_linear(x, w)
    assert y.shape == (1, o) and torch.equal(y[0], w[:, 0] / 2)      # whole numbers up to 3 are codes
    del y
    held = memfast.mx_quantize(w)
    assert torch.equal(memfast.mx_linear(x, held)[0], w[:, 0] / 2)
