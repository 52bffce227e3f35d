"""Dropout against its definition: the generator in whole numbers, sums in 64 bits.

A kept value is one product by FP32(65536 / (65536 - dropped)), off by 2^-24 relative twice, or one fused
multiply and add, and one rounding to the type: bounds of eps / 2 of the result and 3 * 2^-24 of the terms.
"""

import math

import pytest
import torch
import torch.utils.checkpoint

import memfast_amd as memfast
from memfast_amd.nn import Dropout

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def philox(counter, key):
    """Philox 4x32-10 of whole numbers."""
    c, (k0, k1), low = list(counter), key, 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & low, (p0 >> 32) ^ c[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def mask(count, p, seed, event, first=0):
    """Whether the values ``first`` .. are kept."""
    dropped, kept, low = round(p * 65536), [], 0xFFFFFFFF
    for block in range(first // 8, -(-(first + count) // 8)):
        words = philox((block & low, block >> 32, event & low, event >> 32), (seed & low, seed >> 32))
        for word in words:
            kept += [(word & 0xFFFF) >= dropped, (word >> 16) >= dropped]
    at = first % 8
    return torch.tensor(kept[at:at + count])


def expected(x, p, seed, event, residual=None):
    kept = mask(x.numel(), p, seed, event).view(x.shape)
    dropped = round(p * 65536)
    factor = 65536 / (65536 - dropped) if dropped < 65536 else 0.0
    y = torch.where(kept, x.detach().double().cpu() * factor, 0.0)
    terms = y.abs()
    if residual is not None:
        y, terms = y + residual.detach().double().cpu(), terms + residual.detach().double().cpu().abs()
    return kept, y, terms


def near(got, y, terms):
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * y.abs() + 3 * 2.0**-24 * terms + info.smallest_normal * info.eps
    assert bool(((got.detach().double().cpu() - y).abs() <= bound).all())


def test_known_answers():
    """The generator's published test vectors (the Random123 distribution's kat_vectors)."""
    ones = 0xFFFFFFFF
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (33, 64), (2, 3, 1001), ()])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_values_and_gradients(hip_device, kind, shape, p):
    gen = torch.Generator().manual_seed(11)
    x, residual, dy = (torch.randn(shape, generator=gen).to(TYPES[kind]).to(hip_device) for _ in range(3))
    seed, event = (1 << 63) + 12345678901, (1 << 40) + 3
    for r in (None, residual):
        leaf = x.clone().requires_grad_(True)
        kept, y, terms = expected(x, p, seed, event, r)
        extra = None if r is None else r.clone().requires_grad_(True)
        got = memfast.dropout(leaf, p, seed=seed, event=event, residual=extra)
        near(got, y, terms)
        grads = torch.autograd.grad(got, (leaf,) if r is None else (leaf, extra), dy)
        near(grads[0], *expected(dy, p, seed, event)[1:])
        if r is not None:
            assert torch.equal(grads[1], dy)


def test_strides_and_alignment_do_not_change_the_mask(hip_device):
    wide = torch.randn(40, 77, device=hip_device)
    for view in (wide[:, 1:], wide.T, wide[::2, ::3], wide[3, 5:], wide[:1].expand(9, 77)):
        got = memfast.dropout(view, 0.3, seed=4, event=2)
        assert torch.equal(got, memfast.dropout(view.contiguous(), 0.3, seed=4, event=2))
        assert torch.equal(got != 0, mask(view.numel(), 0.3, 4, 2).view(view.shape).to(hip_device))
    flat = torch.randn(1001, device=hip_device, dtype=torch.bfloat16)
    residual = torch.randn(1003, device=hip_device, dtype=torch.bfloat16)[2:]
    a = memfast.dropout(flat, 0.3, seed=4, residual=residual)
    assert torch.equal(a, memfast.dropout(flat.clone(), 0.3, seed=4, residual=residual.clone()))
    leaf = flat.clone().requires_grad_(True)
    dx, = torch.autograd.grad(memfast.dropout(leaf, 0.3, seed=4).sum(), leaf)      # an expanded gradient
    near(dx, *expected(torch.ones_like(flat), 0.3, 4, 0)[1:])


def test_dropped_values_are_gone(hip_device):
    x = torch.full((64,), math.nan, device=hip_device)
    x[::3], x[1::3] = math.inf, -math.inf
    kept = mask(64, 0.5, 9, 0).to(hip_device)
    y = memfast.dropout(x, 0.5, seed=9)
    assert bool((y[~kept] == 0).all()) and torch.equal(y[kept].isnan(), x[kept].isnan())
    assert torch.equal(y[kept].isinf(), x[kept].isinf())
    r = torch.randn(64, device=hip_device)
    assert torch.equal(memfast.dropout(x, 0.5, seed=9, residual=r)[~kept], r[~kept])
    leaf = torch.ones(64, device=hip_device, requires_grad=True)
    dx, = torch.autograd.grad(memfast.dropout(leaf, 0.5, seed=9), leaf, x)
    assert bool((dx[~kept] == 0).all())


def test_probabilities_at_the_ends(hip_device):
    x, r = torch.randn(5000, device=hip_device), torch.randn(5000, device=hip_device)
    for options in (dict(p=0.0), dict(p=1e-6), dict(p=0.5, training=False)):
        assert torch.equal(memfast.dropout(x, **options, seed=1), x)
        assert torch.equal(memfast.dropout(x, **options, seed=1, residual=r), r + x)
    leaf = x.clone().requires_grad_(True)
    for p in (1.0, 1 - 1e-6):
        y = memfast.dropout(leaf, p, seed=1, residual=r)
        assert torch.equal(y, r) and bool((torch.autograd.grad(y.sum(), leaf)[0] == 0).all())
    for p in (1, 0):
        assert bool((memfast.dropout(x, p, seed=1) == (0 if p else x)).all())
    empty = torch.zeros(3, 0, device=hip_device, requires_grad=True)
    assert memfast.dropout(empty, 0.5, seed=1).shape == (3, 0)
    y = memfast.dropout(x, 65535 / 65536, seed=1)             # one in 65536 is kept, 65536 times as large
    kept = mask(5000, 65535 / 65536, 1, 0).to(hip_device)
    assert torch.equal(y, torch.where(kept, x * 65536, 0.0))


@pytest.mark.parametrize("p", [0.1, 0.5])
def test_masks_are_random(hip_device, p):
    """Shares of kept values, and of values kept in two masks, within 6 standard deviations."""
    n = 1 << 22
    x = torch.ones(n, device=hip_device)
    share = 1 - round(p * 65536) / 65536
    masks = [memfast.dropout(x, p, seed=s, event=e) != 0 for s, e in ((1, 0), (1, 1), (2, 0), (1 << 32, 0))]
    masks += [masks[0].roll(k) for k in (1, 2, 8, 4096)]
    for a in masks:
        assert abs(float(a.double().mean()) - share) < 6 * math.sqrt(share * (1 - share) / n)
    both = share * share
    for b in masks[1:]:
        assert abs(float((masks[0] & b).double().mean()) - both) < 6 * math.sqrt(both * (1 - both) / n)


def test_places_beyond_32_bits(hip_device):
    """A value's number depends on all of its place."""
    n = (1 << 32) + 8 * 1024 + 3
    x = torch.ones(n, dtype=torch.bfloat16, device=hip_device)
    y = memfast.dropout(x, 0.5, seed=5)
    for first in (0, (1 << 31) - 16, (1 << 32) - 16, n - 100):
        count = min(64, n - first)
        assert torch.equal(y[first:first + count].cpu() != 0, mask(count, 0.5, 5, 0, first))
    far = (1 << 35) // 8                                       # the block where the counter's second word is 1
    assert mask(8, 0.5, 5, 0, far * 8).shape == (8,)


def test_event_on_the_device(hip_device):
    """A captured graph makes a new mask where the event's tensor is counted up between replays, and the
    forward and backward of one replay share it."""
    x = torch.randn(3000, device=hip_device)
    event = torch.zeros(1, dtype=torch.int64, device=hip_device)
    leaf = x.clone().requires_grad_(True)

    def call():
        y = memfast.dropout(leaf, 0.5, seed=8, event=event)
        return y.detach(), torch.autograd.grad(y, leaf, torch.ones_like(y))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = call()
        event.add_(1)
    event.zero_()
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, memfast.dropout(x, 0.5, seed=8, event=turn))
        assert torch.equal(dx, memfast.dropout(torch.ones_like(x), 0.5, seed=8, event=turn))
    event.fill_((1 << 62) + 1)
    assert torch.equal(memfast.dropout(x, 0.5, seed=8, event=event),
                       memfast.dropout(x, 0.5, seed=8, event=(1 << 62) + 1))
    y = memfast.dropout(leaf, 0.5, seed=8, event=event)
    event.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), leaf)


def test_second_derivatives_and_checkpoints(hip_device):
    x = torch.randn(200, device=hip_device, requires_grad=True)

    def call(x):
        return memfast.dropout(x * x, 0.4, seed=3, event=1)

    kept = mask(200, 0.4, 3, 1).to(hip_device)
    dx, = torch.autograd.grad(call(x).sum(), x, create_graph=True)
    ddx, = torch.autograd.grad(dx.sum(), x)
    factor = 65536 / (65536 - round(0.4 * 65536))
    assert torch.allclose(ddx, torch.where(kept, 2 * factor, 0.0), rtol=1e-6, atol=0)
    for reentrant in (False, True):
        y = torch.utils.checkpoint.checkpoint(call, x, use_reentrant=reentrant)
        assert torch.equal(torch.autograd.grad(y.sum(), x)[0] if not reentrant else
                           (x.grad if y.sum().backward() is None else None), dx.detach())
        x.grad = None


def test_layer(hip_device):
    """Masks come from torch's default generator, one seed a forward."""
    layer = Dropout(0.3).to(hip_device)
    x = torch.randn(4000, device=hip_device)
    torch.manual_seed(5)
    outputs = [layer(x) for _ in range(3)]
    torch.manual_seed(5)
    for y in outputs:
        seed = int(torch.randint(1 << 62, ()))
        assert torch.equal(y, memfast.dropout(x, 0.3, seed=seed))
    assert not torch.equal(outputs[0], outputs[1])
    r = torch.randn_like(x)
    torch.manual_seed(5)
    assert torch.equal(layer(x, residual=r) == r, outputs[0] == 0)
    layer.eval()
    before = torch.get_rng_state()
    assert layer(x) is x and torch.equal(layer(x, residual=r), r + x)
    assert torch.equal(torch.get_rng_state(), before)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_layer_keeps_its_mask(hip_device, reentrant):
    """The second forward, in the backward, drops what the first one dropped."""
    layer = Dropout(0.5).to(hip_device)
    x = torch.ones(3000, device=hip_device, requires_grad=True)
    for _ in range(2):
        y = torch.utils.checkpoint.checkpoint(lambda v: layer(v * v), x, use_reentrant=reentrant)
        x.grad = None
        y.sum().backward()
        assert torch.equal(x.grad != 0, y != 0)


def test_the_layers_seeds_stay_on_the_cpu(hip_device):
    """A default device moves neither the generator nor the masks, and no draw waits for the GPU."""
    layer = Dropout(0.4)
    x = torch.ones(777, device=hip_device)
    torch.manual_seed(11)
    expected = layer(x)
    torch.manual_seed(11)
    state = torch.cuda.get_rng_state(hip_device)
    with torch.device(hip_device):
        assert torch.equal(layer(x), expected)
    assert torch.equal(torch.cuda.get_rng_state(hip_device), state)
