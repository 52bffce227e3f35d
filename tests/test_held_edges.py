"""4-bit weights without inputs or outputs, packed on any device."""

import pytest
import torch

import memfast_amd as memfast


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("o,k", [(0, 0), (3, 0), (17, 0), (0, 64), (0, 300)])
def test_weights_without_values_are_packed(o, k, zeros):
    """As int4_quantize gives them: no tile for no outputs, no span and no group for no inputs."""
    groups = -(-k // 64)
    held = memfast.Int4Tensor.pack(torch.zeros(o, k, dtype=torch.uint8), torch.ones(o, groups), group=64,
                                   zeros=torch.zeros(o, groups, dtype=torch.uint8) if zeros else None)
    tiles = -(-o // 16)
    assert held.shape == (o, k) and held.codes.shape == (tiles, -(-k // 128), 1024)
    assert held.scales.shape == (tiles, groups, 16)
    assert held.zeros is None or held.zeros.shape == (tiles, groups, 16)


@pytest.mark.parametrize("o,k", [(-1, 64), (16, -1), (-15, -20)])
def test_negative_shapes_are_refused(o, k):
    """Parts without values, as rounding up makes them of such a shape, are no weight."""
    codes = torch.zeros(-(-o // 16), -(-k // 128), 1024, dtype=torch.uint8)
    scales = torch.ones(-(-o // 16), -(-k // 32), 16)
    with pytest.raises(ValueError, match="negative"):
        memfast.Int4Tensor(codes, scales, (o, k), group=32)
