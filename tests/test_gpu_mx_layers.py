"""The 4-bit linear layer, the operators together, HIP graphs and sizes past 32 bits."""

import importlib.util
from pathlib import Path

import pytest
import torch
from torch import nn

import memfast_amd as memfast
from memfast_amd.nn import MXLinear

pytestmark = pytest.mark.gpu


def say(*args):
    print("[mx-layers]", *args, flush=True)


def test_layer_holds_its_weight(hip_device):
    torch.manual_seed(0)
    source = nn.Linear(100, 40).to(hip_device)
    layer = MXLinear(source)
    x = torch.randn(3, 5, 100, device=hip_device, requires_grad=True)
    y = layer(x)
    assert torch.equal(y, memfast.mx_linear(x, source.weight, source.bias))
    assert not list(layer.parameters())
    dx, = torch.autograd.grad(y.sum(), x)
    assert dx.shape == x.shape and bool(torch.isfinite(dx).all())
    other = MXLinear(nn.Linear(100, 40).to(hip_device))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    half = MXLinear(nn.Linear(100, 40, bias=False).to(hip_device).bfloat16())
    assert half(x.bfloat16()).dtype == torch.bfloat16
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(layer(x), y)


def test_layer_trains_its_weight(hip_device):
    torch.manual_seed(0)
    source = nn.Linear(96, 33).to(hip_device)
    layer = MXLinear(source, trainable=True)
    assert layer.weight is not source.weight and torch.equal(layer.weight, source.weight)
    x = torch.randn(70, 96, device=hip_device)
    target = torch.randn(70, 33, device=hip_device)
    optimizer = torch.optim.SGD(layer.parameters(), lr=0.05)
    losses = []
    for _ in range(20):
        loss = (layer(x) - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]
    with pytest.raises(TypeError):
        MXLinear(nn.Conv2d(1, 1, 1))


def test_example_distills_an_analog_student(hip_device):
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_student.py"
    spec = importlib.util.spec_from_file_location("distill_student", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.distill(steps=16, batch=32, features=128, hidden=128, classes=300, k=8,
                             device=hip_device)
    say("losses", losses)
    # Batches come round after eight steps.
    assert sum(losses[8:]) < 0.8 * sum(losses[:8])


@pytest.mark.parametrize("n", [3, 40, 300])
def test_operators_replay_in_a_graph(hip_device, n):
    gen = torch.Generator(device=hip_device).manual_seed(n)
    x = torch.randn(n, 512, generator=gen, device=hip_device)
    weight = memfast.mx_quantize(torch.randn(700, 512, generator=gen, device=hip_device))
    student = torch.randn(n, 700, generator=gen, device=hip_device)

    def step():
        logits = memfast.mx_linear(x, weight)
        values, indices, tail = memfast.top_logits(logits, 7)
        loss = memfast.distillation_loss(student, values, indices, tail)
        return logits, values, indices, tail, loss

    side = torch.cuda.Stream(hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(hip_device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        x.copy_(torch.randn(n, 512, generator=gen, device=hip_device))
        student.copy_(torch.randn(n, 700, generator=gen, device=hip_device))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_logits_past_32_bits(hip_device):
    """The last rows of 4.4e9 logits give what they give alone."""
    n, v, k = 33600, 131072, 5
    say("logits", n, v)
    s = torch.zeros(n, v, dtype=torch.bfloat16, device=hip_device)
    gen = torch.Generator(device=hip_device).manual_seed(1)
    s[-3:] = (3 * torch.randn(3, v, generator=gen, device=hip_device)).bfloat16()
    values, indices, tail = memfast.top_logits(s, k)
    alone = memfast.top_logits(s[-3:].clone(), k)
    for a, b in zip((values, indices), alone):
        assert torch.equal(a[-3:], b)
    assert bool(((tail[-3:] - alone[2]).abs() <= 1e-5).all())
    s.requires_grad_(True)
    loss = memfast.distillation_loss(s, values, indices, tail, reduction="sum", temperature=2.0)
    grad, = torch.autograd.grad(loss, s)
    last = s.detach()[-3:].clone().requires_grad_(True)
    part = memfast.distillation_loss(last, values[-3:], indices[-3:], tail[-3:], reduction="sum",
                                     temperature=2.0)
    expected, = torch.autograd.grad(part, last)
    assert torch.equal(grad[-3:], expected)


def test_products_past_32_bits(hip_device):
    """The last tile of an output of 4.4e9 values, and codes past 2**32, against the same rows alone."""
    n, k, o = 40000, 64, 110100
    say("product", n, k, o)
    gen = torch.Generator(device=hip_device).manual_seed(2)
    x = torch.randn(n, k, generator=gen, device=hip_device).bfloat16()
    w = torch.randn(o, k, generator=gen, device=hip_device).bfloat16()
    y = memfast.mx_linear(x, w)
    part = memfast.mx_linear(x[-300:].clone(), w[-300:].clone())
    assert torch.equal(y[-300:, -300:], part)       # one segment: sums of one matrix instruction each
    del y
    wide = torch.zeros(4300, 1 << 20, dtype=torch.bfloat16, device=hip_device)
    wide[-2:] = torch.randn(2, 1 << 20, generator=gen, device=hip_device).bfloat16()
    held, alone = memfast.mx_quantize(wide), memfast.mx_quantize(wide[-2:].clone())
    assert torch.equal(held.codes[-2:], alone.codes) and torch.equal(held.scales[-2:], alone.scales)
    values = held.dequantize(torch.bfloat16)
    assert torch.equal(values[-2:], alone.dequantize(torch.bfloat16)) and not values[:-2].any()
