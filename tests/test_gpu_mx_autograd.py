"""What the 4-bit product keeps for its backward, and what autograd may do with it."""

import gc
import weakref

import pytest
import torch
import torch.utils.checkpoint
from torch import nn

import memfast_amd as memfast
from memfast_amd.nn import MXLinear

pytestmark = pytest.mark.gpu


def operands(device, n=70, k=96, o=40, dtype=torch.float32):
    gen = torch.Generator().manual_seed(n + k + o)
    x, w = (torch.randn(*s, generator=gen).to(dtype).to(device) for s in ((n, k), (o, k)))
    dy = torch.randn(n, o, generator=gen).to(dtype).to(device)
    return x.requires_grad_(True), w.requires_grad_(True), dy


def test_a_held_weight_that_is_rewritten_is_noticed(hip_device):
    """Its gradient would be the new weight's."""
    x, w, dy = operands(hip_device)
    for part in ("codes", "scales"):
        held = memfast.mx_quantize(w)
        y = memfast.mx_linear(x, held)
        getattr(held, part).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, x, dy)
    layer = MXLinear(nn.Linear(96, 40).to(hip_device))
    y = layer(x)
    layer.load_state_dict(MXLinear(nn.Linear(96, 40).to(hip_device)).state_dict())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    torch.autograd.grad(layer(x), x, dy)


@pytest.mark.parametrize("held", [False, True])
def test_saved_tensor_hooks_see_what_is_kept(hip_device, held):
    """Everything that the backward reads goes through the hooks, here to the host and back."""
    x, w, dy = operands(hip_device)
    weight = memfast.mx_quantize(w) if held else w
    wanted = (x,) if held else (x, w)
    expected = torch.autograd.grad(memfast.mx_linear(x, weight), wanted, dy)
    packed = []

    def pack(t):
        packed.append(t.numel())
        return t.to("cpu", copy=True)

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(hip_device)):
        y = memfast.mx_linear(x, weight)
    segments = 1                            # of 256 values, 128 bytes of codes and 8 of scales
    least = segments * (128 + 8) * (40 if held else 40 + 70)
    assert sum(packed) >= least
    for a, b in zip(torch.autograd.grad(y, wanted, dy), expected):
        assert torch.equal(a, b)
    offloaded = torch.autograd.graph.save_on_cpu()
    with offloaded:
        y = memfast.mx_linear(x, weight)
    for a, b in zip(torch.autograd.grad(y, wanted, dy), expected):
        assert torch.equal(a, b)


def test_what_is_kept_is_freed_by_the_backward(hip_device):
    x, w, dy = operands(hip_device, n=2000, k=1000, o=500)
    torch.cuda.synchronize()
    y = memfast.mx_linear(x, w)
    kept = torch.cuda.memory_allocated(hip_device)
    grads = torch.autograd.grad(y, (x, w), dy)
    size = sum(g.untyped_storage().nbytes() for g in grads)
    # 4 segments of 128 bytes of codes a row of either operand.
    assert torch.cuda.memory_allocated(hip_device) - size <= kept - 2500 * 4 * 128
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, (x, w), dy)
    # With the graph retained, both backwards agree.
    y = memfast.mx_linear(x, w)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(y, (x, w), dy)):
        assert torch.equal(a, b)
    node = weakref.ref(y.grad_fn)
    del y
    gc.collect()
    assert node() is None


def test_checkpointed_products(hip_device):
    x, w, dy = operands(hip_device)
    expected = torch.autograd.grad(memfast.mx_linear(x, w), (x, w), dy)
    for reentrant in (False, True):
        y = torch.utils.checkpoint.checkpoint(memfast.mx_linear, x, w, use_reentrant=reentrant)
        x.grad = w.grad = None
        y.backward(dy)
        assert torch.equal(x.grad, expected[0]) and torch.equal(w.grad, expected[1])


def test_sizes_without_a_backward_are_refused_before_the_forward(hip_device):
    """The gradients take fewer rows and outputs than the product."""
    rows, outputs = 1 << 24, (1 << 22) + 1
    many = torch.ones(1, 1, dtype=torch.bfloat16, device=hip_device)
    w = torch.full((1, 1), 2.0, dtype=torch.bfloat16, device=hip_device)
    for x, weight in ((many.expand(rows, 1), w), (many, w.expand(outputs, 1)),
                      (many.expand(rows, 1), memfast.mx_quantize(w))):
        y = memfast.mx_linear(x, weight)
        assert bool((y == 2).all())
        with torch.no_grad():
            assert memfast.mx_linear(x.detach().requires_grad_(True), weight).shape == y.shape
        with pytest.raises(NotImplementedError, match="gradients of more than"):
            memfast.mx_linear(x.detach().requires_grad_(True), weight)
    x = many.expand(rows - 1, 1).contiguous().requires_grad_(True)
    dx, = torch.autograd.grad(memfast.mx_linear(x, w).sum(), x)
    assert bool((dx == 2).all())
    w = w.expand(outputs - 1, 1).contiguous().requires_grad_(True)
    dw, = torch.autograd.grad(memfast.mx_linear(many, w).sum(), w)
    assert bool((dw == 1).all())
