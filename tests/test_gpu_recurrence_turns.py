"""The recurrence where a workgroup goes through many spans, and where many segments are joined.

A workgroup takes 128 steps a turn, and with few channels the steps are split into segments whose number shows
in the workspace (two FP32 values a segment, sequence and channel). The cases are the turns and segments that
they are named by; bounds are those of test_gpu_recurrence.
"""

import pytest
import torch

import memfast_amd as memfast
from memfast_amd import hip
from test_gpu_recurrence import TYPES, case, check

pytestmark = pytest.mark.gpu

# steps, batch, width, segments, spans of 128 steps a segment
SIZES = [(600, 256, 3, 1, 5),           # five turns of one workgroup, the last of 88 steps
         (1030, 300, 2, 1, 9),          # nine, the last of six steps
         (1500, 100, 2, 6, 2),          # segments of two turns
         (3000, 200, 1, 3, 8),          # of eight, and eight rounds of a wave that reduces its share
         (8300, 1, 4, 65, 1)]           # more segments than the eight waves fetch at once


def segments(steps, batch, width):
    work = hip._recurrence_sizes(steps, batch, width)[1]
    return max(1, work // (batch * width * 8))


@pytest.mark.parametrize("steps,batch,width,count,spans", SIZES)
def test_the_cases_are_what_they_are_named(hip_device, steps, batch, width, count, spans):
    assert segments(steps, batch, width) == count
    assert count == -(-steps // (128 * spans))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("steps,batch,width,count,spans", SIZES)
def test_turns(hip_device, kind, steps, batch, width, count, spans):
    x, state, dy, dlast = case(hip_device, steps, batch, width, kind)
    if kind != "bf16":
        check(x, state, dy, dlast)
    if kind != "fp16":
        check(x, None, dy, dlast, reverse=True, activation=None)


@pytest.mark.parametrize("kind,reverse", [("fp32", True), ("bf16", False)])
@pytest.mark.parametrize("steps,batch,width,count,spans", SIZES)
def test_turns_with_lengths(hip_device, kind, reverse, steps, batch, width, count, spans):
    """Sequences that end in every turn and segment, at their borders and within a wave's steps; what lies
    behind them is NaN."""
    gen = torch.Generator().manual_seed(steps)
    lengths = torch.randint(0, steps + 1, (batch,), generator=gen)
    some = [steps, 0, 1, 128, 129, 127, 128 * spans, 128 * spans + 1, 128 * spans - 1, steps - 1, 256, 264]
    lengths[:len(some)] = torch.tensor(some)[:batch].clamp(max=steps)
    if batch == 1:
        lengths[0] = 8291
    x, state, dy, dlast = case(hip_device, steps, batch, width, kind)
    behind = torch.arange(steps)[:, None] >= lengths
    x[behind.to(hip_device)] = torch.nan
    dy[behind.to(hip_device)] = torch.nan
    assert segments(steps, batch, width) == count
    check(x, state, dy, dlast, lengths=lengths.to(hip_device), reverse=reverse)


def test_turns_are_the_sequence_in_parts(hip_device):
    """A last state that is passed on is the state: parts of any turns against the whole."""
    for steps, batch, width, _, _ in SIZES[:3]:
        x, state, _, _ = case(hip_device, steps, batch, width, "fp32")
        whole, last = memfast.gated_recurrence(x, state)
        h, parts = state, []
        for part in torch.tensor_split(x, (100, 357, 485)):
            y, h = memfast.gated_recurrence(part, h)
            parts.append(y)
        # Both within the bound of the 64-bit sequence, whose states are at most 4 here.
        assert float((torch.cat(parts) - whole).abs().max()) < 1e-4
        assert float((h - last).abs().max()) < 1e-4
