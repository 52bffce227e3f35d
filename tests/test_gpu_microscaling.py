"""4-bit microscaled tensors and their product against their definition in 64 bits.

Tolerances.  Codes and scales are compared exactly.  Every product of two 4-bit values (and of
one with an eight-bit term of a gradient) is exact in FP32, so a sum of t of them in any order is
within t * 2**-24 of the sum of their magnitudes; the result is then rounded once more (2**-24, 2**-8
and 2**-11 of its size in FP32, BF16 and FP16), and a bias adds one more FP32 rounding.
"""

import pytest
import torch

import memfast_amd as memfast

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TERMS = {torch.float32: 3, torch.bfloat16: 1, torch.float16: 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def say(*args):
    print("[microscaling]", *args, flush=True)


def oracle(x):
    """(codes [n, ceil(k/32), 32], scale bytes [n, ceil(k/32)], values [n, k]) in 64 bits on the CPU."""
    x = x.detach().double().cpu()
    n, k = x.shape
    y = torch.zeros(n, -(-k // 32) * 32, dtype=torch.float64)
    y[:, :k] = x
    y = y.reshape(n, -1, 32)
    bad = ~torch.isfinite(y).all(-1)
    y = torch.where(bad[..., None], 0.0, y)
    peak = y.abs().amax(-1)
    exponent = torch.where(peak > 0, torch.frexp(peak).exponent - 3, -126).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(peak), exponent)
    size = y.abs() / scale[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64)
    near = (size[..., None] - grid).abs()
    least = near.amin(-1, keepdim=True)
    # Among the nearest, the even code: the lower one of a tie unless it is odd.
    first = (near == least).int().argmax(-1)
    tie = (near == least).sum(-1) > 1
    code = torch.where(tie & (first % 2 == 1), first + 1, first)
    values = torch.where(y < 0, -grid[code], grid[code]) * scale[..., None]
    values = torch.where(bad[..., None], float("nan"), values).reshape(n, -1)[:, :k]
    code = code + 8 * torch.signbit(y)
    return (torch.where(bad[..., None], 0, code), torch.where(bad, 255, exponent + 127), values)


def unpacked(t):
    codes = torch.stack((t.codes & 15, t.codes >> 4), -1).reshape(len(t.codes), -1, 32).cpu()
    return codes.long(), t.scales.cpu().long()


def check_codes(x, t):
    code, byte, values = oracle(x.reshape(-1, x.shape[-1]))
    got_code, got_byte = unpacked(t)
    blocks = code.shape[1]
    assert torch.equal(got_byte[:, :blocks], byte)
    assert torch.equal(got_code[:, :blocks], code)
    assert int(got_code[:, blocks:].abs().sum()) == 0      # padding
    for dtype in TYPES.values():
        got = t.dequantize(dtype).cpu().reshape(values.shape)
        assert got.dtype == dtype
        assert torch.equal(torch.nan_to_num(got, nan=777.0),
                           torch.nan_to_num(values.to(dtype), nan=777.0))


def data(n, k, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed + 1000 * n + k)
    x = torch.randn(n, k, generator=gen) * torch.exp(1.5 * torch.randn(n, k, generator=gen))
    return x.clamp(-1000, 1000).to(dtype).to(device)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 255), (1, 256), (4, 257),
                                 (2, 1000), (130, 96), (3, 4096), (1, 11008), (70000, 8)])
def test_codes_and_scales(hip_device, kind, n, k):
    x = data(n, k, TYPES[kind], hip_device)
    check_codes(x, memfast.mx_quantize(x))


def test_ties_signs_and_saturation(hip_device):
    """Every multiple of 1/16 up to the largest a block can hold, of both signs, at several scales."""
    steps = torch.arange(0, 128, dtype=torch.float32) / 16          # 0 .. 7.9375
    rows = []
    for exponent in (-126, -20, -1, 0, 1, 60, 125):
        block = torch.cat((steps, -steps)).reshape(-1, 16)
        # 4 in each block keeps its scale at 2**exponent.
        block = torch.cat((block, torch.full((len(block), 16), 4.0)), 1)
        rows.append(block.reshape(1, -1) * 2.0**exponent)
    x = torch.cat(rows).to(hip_device)
    check_codes(x, memfast.mx_quantize(x))


def test_zeros_subnormals_extremes_and_non_finite_blocks(hip_device):
    x = torch.zeros(8, 96, device=hip_device)
    x[1] = 1e-45
    x[2, :32] = torch.finfo(torch.float32).max
    x[3] = -0.0
    x[4, 40] = float("nan")
    x[5, 95] = float("inf")
    x[6, 0] = float("-inf")
    x[7] = 2.0**-126
    t = memfast.mx_quantize(x)
    check_codes(x, t)
    assert t.dequantize()[4].isnan().sum() == 32


@pytest.mark.parametrize("kind", list(TYPES))
def test_strided_and_unaligned_inputs(hip_device, kind):
    dtype = TYPES[kind]
    base = data(9, 701, dtype, hip_device)
    for x in (base[:, 1:], base[:, 3:300], base.T, base[::2], base[0], base[:1, 5:5].reshape(1, 0),
              base[:, :1].expand(9, 64), base.reshape(3, 3, 701)[:, 1]):
        t = memfast.mx_quantize(x)
        assert t.shape == x.shape
        if x.numel():
            check_codes(x.reshape(-1, x.shape[-1]), t)


SHAPES = [(1, 32, 1), (1, 100, 7), (1, 4096, 130), (2, 256, 64), (5, 257, 33), (16, 512, 100),
          (17, 64, 31), (31, 1500, 65), (33, 300, 129), (64, 96, 64), (65, 784, 10), (100, 784, 512),
          (129, 1000, 257), (300, 33, 260), (260, 2049, 300), (13, 11008, 40)]


def product_bound(x, w, y, bias, dtype):
    k = x.shape[1]
    magnitude = x.abs() @ w.abs().T
    bound = k * 2.0**-24 * magnitude + UNIT[dtype] * y.abs() * (1 + 2.0**-8)
    if bias is not None:
        bound = bound + 2.0**-24 * (magnitude + bias.abs()) * 2
    return bound + 2.0**-133       # results below the smallest normal number


def assert_within(got, expected, bound, label):
    half, got = got.dtype == torch.float16, got.detach().double().cpu()
    assert got.shape == expected.shape, label
    if half:    # subnormal results; those beyond the type are infinite
        bound, inside = bound + 2.0**-25, expected.abs() < 65000
        got, expected, bound = got[inside], expected[inside], bound[inside]
    off = (got - expected).abs()
    assert bool((off <= bound).all()), (label, float((off / bound).nan_to_num(0).max()))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,o", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear(hip_device, kind, n, k, o, bias):
    dtype = TYPES[kind]
    x, w = data(n, k, dtype, hip_device, 1), (0.02 * data(o, k, torch.float32, hip_device, 2)).to(dtype)
    b = data(1, o, dtype, hip_device, 3)[0] if bias else None
    say("linear", kind, n, k, o, bias)
    xq, wq = oracle(x)[2], oracle(w)[2]
    expected = xq @ wq.T
    if bias:
        expected = expected + b.double().cpu()
    bound = product_bound(xq, wq, expected, None if b is None else b.double().cpu(), dtype)
    held = memfast.mx_linear(x, memfast.mx_quantize(w), b)
    assert held.dtype == dtype
    assert_within(held, expected, bound, "held weight")
    assert torch.equal(memfast.mx_linear(x, w, b), held)
    # With gradients wanted the forward is the same.
    again = memfast.mx_linear(x.clone().requires_grad_(True), w.clone().requires_grad_(True), b)
    assert torch.equal(again.detach(), held)


def test_linear_shapes_strides_and_empty_operands(hip_device):
    w = data(48, 64, torch.bfloat16, hip_device)
    x = data(6, 64, torch.bfloat16, hip_device, 4)
    held = memfast.mx_quantize(w)
    flat = memfast.mx_linear(x, held)
    assert torch.equal(memfast.mx_linear(x.reshape(2, 3, 64), held), flat.reshape(2, 3, 48))
    assert torch.equal(memfast.mx_linear(x[2], held), flat[2])
    wide = torch.zeros(6, 130, dtype=x.dtype, device=hip_device)
    wide[:, 3:67] = x
    assert torch.equal(memfast.mx_linear(wide[:, 3:67], held), flat)
    assert torch.equal(memfast.mx_linear(x.T.contiguous().T, held), flat)
    assert memfast.mx_linear(x[:0], held).shape == (0, 48)
    b = data(1, 48, torch.bfloat16, hip_device, 5)[0]
    none = memfast.mx_linear(x[:, :0], w[:, :0], b)
    assert torch.equal(none, b.expand(6, 48))
    assert memfast.mx_linear(x, w[:0]).shape == (6, 0)


def test_linear_rows_do_not_depend_on_their_neighbours_nan(hip_device):
    for n in (3, 40, 200):
        x = data(n, 300, torch.float32, hip_device, 6)
        w = data(70, 300, torch.float32, hip_device, 7)
        clean = memfast.mx_linear(x, w)
        x[1, 50] = float("nan")
        w[5, 7] = float("inf")
        got = memfast.mx_linear(x, w)
        assert got[1].isnan().all() and got[:, 5].isnan().all()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[1], keep[:, 5] = False, False
        assert torch.equal(got[keep], clean[keep])


GRADS = [(1, 32, 1), (3, 100, 7), (64, 256, 64), (65, 257, 33), (100, 784, 512), (128, 64, 128),
         (192, 300, 200), (257, 33, 260), (130, 1000, 10), (64, 2048, 192)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,o", GRADS)
def test_gradients(hip_device, kind, n, k, o):
    dtype = TYPES[kind]
    say("gradients", kind, n, k, o)
    x = data(n, k, dtype, hip_device, 1).requires_grad_(True)
    w = (0.02 * data(o, k, torch.float32, hip_device, 2)).to(dtype).requires_grad_(True)
    b = data(1, o, dtype, hip_device, 3)[0].requires_grad_(True)
    dy = (0.1 * data(n, o, torch.float32, hip_device, 4)).clamp(-1e4, 1e4).to(dtype)
    dx, dw, db = torch.autograd.grad(memfast.mx_linear(x, w, b), (x, w, b), dy)
    xq, wq, d = oracle(x)[2], oracle(w)[2], dy.double().cpu()
    terms = TERMS[dtype]
    for got, left, right, label in ((dx, d, wq, "dx"), (dw, d.T, xq, "dw")):
        assert got.dtype == dtype
        expected = left @ right
        bound = (terms * left.shape[1] * 2.0**-24 * (left.abs() @ right.abs())
                 + UNIT[dtype] * expected.abs() * (1 + 2.0**-8) + 2.0**-133)
        assert_within(got, expected, bound, label)
    expected = d.sum(0)
    assert_within(db, expected, n * 2.0**-24 * d.abs().sum(0) + UNIT[dtype] * expected.abs() * (1 + 2.0**-8)
                  + 2.0**-133, "db")
    # The weight alone, the input alone (also of a held weight).
    alone, = torch.autograd.grad(memfast.mx_linear(x.detach(), w, b), w, dy)
    assert torch.equal(alone, dw)
    alone, = torch.autograd.grad(memfast.mx_linear(x, memfast.mx_quantize(w)), x, dy)
    assert torch.equal(alone, dx)


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_of_strided_and_broadcast_incoming_gradients(hip_device, kind):
    dtype = TYPES[kind]
    n, k, o = 64, 96, 128
    x = data(n, k, dtype, hip_device, 1).requires_grad_(True)
    w = data(o, k, dtype, hip_device, 2).requires_grad_(True)
    wide = data(n, o + 9, dtype, hip_device, 4).clamp(-10, 10)
    y = memfast.mx_linear(x, w)
    for dy in (wide[:, :o], wide[:, 1:o + 1], wide.T.contiguous().T[:, :o],
               wide[:1, :o].expand(n, o), wide[:1, :1].expand(n, o)):
        got = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        expected = torch.autograd.grad(y, (x, w), dy.clone(memory_format=torch.contiguous_format),
                                       retain_graph=True)
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])


def test_gradients_against_differences(hip_device):
    """On operands whose values are codes already, a step to a neighbouring code is a real change
    of the product: its difference quotient is the gradient, exactly (small whole numbers)."""
    gen = torch.Generator().manual_seed(5)
    grid = torch.tensor((0.0, 1.0, 2.0, 3.0))
    x, w = (grid[torch.randint(4, s, generator=gen)] for s in ((70, 64), (40, 64)))
    x[:, ::32] = w[:, ::32] = 4.0           # keeps every block's scale at 1
    dy = torch.randint(-3, 4, (70, 40), generator=gen).float()
    x, w, dy = (t.to(hip_device) for t in (x, w, dy))
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(memfast.mx_linear(x, w), (x, w), dy)
    with torch.no_grad():
        base = (memfast.mx_linear(x, w) * dy).sum()
        for t, grad in ((x, dx), (w, dw)):
            for i, j in ((0, 1), (13, 40), (39, 63)):
                moved = t.detach().clone()
                moved[i, j] = 1.0 if moved[i, j] == 0 else moved[i, j] - 1.0
                pair = (moved, w) if t is x else (x, moved)
                quotient = ((memfast.mx_linear(*pair) * dy).sum() - base) / (moved[i, j] - t[i, j])
                assert float(quotient) == float(grad[i, j])


def test_non_finite_gradients_stay_in_their_rows(hip_device):
    for kind, dtype in TYPES.items():
        x = data(70, 64, dtype, hip_device, 1).requires_grad_(True)
        w = data(40, 64, dtype, hip_device, 2).clamp(-100, 100).requires_grad_(True)
        dy = torch.ones(70, 40, dtype=dtype, device=hip_device)
        dy[69, 39] = float("nan")
        dx, dw = torch.autograd.grad(memfast.mx_linear(x, w), (x, w), dy)
        assert dx[69].isnan().all() and not dx[:69].isnan().any(), kind
        assert dw[39].isnan().all() and not dw[:39].isnan().any(), kind
    big = torch.full((70, 40), torch.finfo(torch.float32).max, device=hip_device)
    w = torch.zeros(40, 64, device=hip_device)
    w[0, 0] = 0.5
    x = data(70, 64, torch.float32, hip_device, 1).requires_grad_(True)
    dx, = torch.autograd.grad(memfast.mx_linear(x, w), x, big)
    assert torch.equal(dx[:, 0], big[:, 0] / 2) and not dx[:, 1:].any()


def test_results_repeat_and_streams(hip_device):
    x, w = (data(200, 512, torch.bfloat16, hip_device, s).requires_grad_(True) for s in (1, 2))
    dy = data(200, 200, torch.bfloat16, hip_device, 3).clamp(-4, 4)

    def step():
        y = memfast.mx_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    first = step()
    side = torch.cuda.Stream(hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream(hip_device).wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_held_weight_from_its_parts(hip_device):
    w = data(40, 100, torch.float32, hip_device)
    t = memfast.mx_quantize(w)
    store = torch.empty(t.codes.numel() + 3, dtype=torch.uint8, device=hip_device)
    shifted = store[3:].view_as(t.codes).copy_(t.codes)       # unaligned
    again = memfast.MXTensor(shifted, t.scales.T.contiguous().T, (40, 100))
    x = data(5, 100, torch.float32, hip_device, 2)
    assert torch.equal(memfast.mx_linear(x, again), memfast.mx_linear(x, t))
    with pytest.raises(ValueError, match="shape"):
        memfast.MXTensor(t.codes[:, :64], t.scales, (40, 100))
    with pytest.raises(ValueError, match="same device"):
        memfast.MXTensor(t.codes, t.scales.cpu(), (40, 100))
    with pytest.raises(ValueError, match="reduction"):
        memfast.mx_linear(x[:, :64], t)
    with pytest.raises(ValueError, match="same dtype"):
        memfast.mx_linear(x, w.half())
    with pytest.raises(ValueError, match="same device"):
        memfast.mx_linear(x.cpu(), t)
    with pytest.raises(ValueError, match="per output"):
        memfast.mx_linear(x, t, x[0])


def test_gradients_are_not_differentiable(hip_device):
    x, w = (data(64, 64, torch.float32, hip_device, s).requires_grad_(True) for s in (1, 2))
    dx, = torch.autograd.grad(memfast.mx_linear(x, w).square().sum(), x, create_graph=True)
    assert dx.shape == x.shape
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
