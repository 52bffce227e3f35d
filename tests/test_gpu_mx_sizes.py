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


# ---------------------------------------------------------------------------
# Every tile, on ragged sizes
# ---------------------------------------------------------------------------
# The bounds are those of tests/test_gpu_microscaling.py: products of two 4-bit values, or of one with an
# eight-bit term of a gradient, are exact in FP32, a sum of t of them in any order is within t * 2**-24 of the sum of
# their magnitudes, a bias adds one more rounding, and the result is rounded once to its type.
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TERMS = {torch.float32: 3, torch.bfloat16: 1, torch.float16: 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def data(n, k, dtype, device, seed, scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed + 1000 * n + k)
    x = torch.randn(n, k, generator=gen, device=device)
    return (scale * (x * torch.exp(torch.randn(n, k, generator=gen, device=device))).clamp(-50, 50)).to(dtype)


def quantized(x):
    """The values of x's codes in 64 bits: to the nearest of the grid, a tie to the even code."""
    n, k = x.shape
    y = torch.zeros(n, -(-k // 32) * 32, dtype=torch.float64, device=x.device)
    y[:, :k] = x.detach().double()
    y = y.reshape(n, -1, 32)
    exponent = (torch.frexp(y.abs().amax(-1, keepdim=True)).exponent - 3).clamp(min=-126)
    size = torch.ldexp(y.abs(), -exponent)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(size, middle)                    # a tie to the lower code
    for odd in (0.75, 1.75, 3.5):                           # whose lower neighbour is odd
        code = code + (size == odd)
    return torch.ldexp(torch.copysign(grid[code], y), exponent).reshape(n, -1)[:, :k].contiguous()


def assert_within(got, expected, bound, label):
    half, got = got.dtype == torch.float16, got.detach().double()
    assert got.shape == expected.shape, label
    bound = bound + 2.0**-133
    if half:    # subnormal results; those beyond the type are infinite
        inside = expected.abs() < 65000
        off, bound = torch.where(inside, (got - expected).abs(), 0.0), bound + 2.0**-25
    else:
        off = (got - expected).abs()
    assert bool((off <= bound).all()), (label, float((off / bound).nan_to_num(0).max()),
                                        (off > bound).nonzero()[:4].tolist())


# Sizes of x's rows and outputs that take each tile.
PRODUCTS = {"256x256": (3100, 4000), "128x256": (1030, 8200), "128x128": (1030, 3700),
            "64x64, two stages": (1030, 1111), "64x64, four stages": (129, 1100), "few rows, wide": (40, 8200),
            "few rows, 4 x 16": (50, 1100), "few rows, 2 x 16": (30, 1100), "few rows": (9, 8200)}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("tile", list(PRODUCTS))
@pytest.mark.parametrize("k", [100, 300, 1100])         # one, two and five segments of 256
def test_products_of_every_tile(hip_device, kind, tile, k):
    (n, o), dtype = PRODUCTS[tile], TYPES[kind]
    print("[mx-sizes] product", kind, tile, n, k, o, flush=True)
    x, w = data(n, k, dtype, hip_device, 1), data(o, k, dtype, hip_device, 2, 0.02)
    b = data(1, o, dtype, hip_device, 3)[0]
    xq, wt = quantized(x), quantized(w).T.contiguous()
    expected, magnitude = xq @ wt, xq.abs() @ wt.abs()
    for bias in (None, b):
        y = expected if bias is None else expected + bias.double()
        bound = k * 2.0**-24 * magnitude + UNIT[dtype] * y.abs() * (1 + 2.0**-8)
        if bias is not None:
            bound = bound + 2.0**-23 * (magnitude + bias.double().abs())
        got = memfast.mx_linear(x, memfast.mx_quantize(w), bias)
        assert got.dtype == dtype
        assert_within(got, y, bound, "held weight")
        assert torch.equal(memfast.mx_linear(x, w, bias), got)


# Rows and columns of a gradient that take each tile, and depths: in whole steps of 64 and not, where
# BF16 gradients are read in place and where not.
GRADIENTS = {"128x128": (2060, 2100, 72), "128x128, whole": (2064, 2100, 128),
             "192x256": (2996, 3990, 72), "192x256, whole": (3000, 4000, 128),
             "256x256": (3996, 3990, 200), "256x256, whole": (4000, 4000, 64),
             "64x64": (700, 1000, 200), "64x64, whole": (704, 1000, 192)}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("tile", list(GRADIENTS))
@pytest.mark.parametrize("wide", ["input", "weight"])
def test_gradients_of_every_tile(hip_device, kind, tile, wide):
    """The input's gradient has the tile's rows, or the weight's; the other one is small."""
    (rows, k, depth), dtype = GRADIENTS[tile], TYPES[kind]
    n, o = (rows, depth) if wide == "input" else (depth, rows)
    print("[mx-sizes] gradients", kind, tile, n, k, o, flush=True)
    x = data(n, k, dtype, hip_device, 1).requires_grad_(True)
    w = data(o, k, dtype, hip_device, 2, 0.02).requires_grad_(True)
    b = data(1, o, dtype, hip_device, 3)[0].requires_grad_(True)
    dy = data(n, o, dtype, hip_device, 4, 0.1)
    dx, dw, db = torch.autograd.grad(memfast.mx_linear(x, w, b), (x, w, b), dy)
    d, xq, wq = dy.double(), quantized(x), quantized(w)
    for got, left, right, label in ((dx, d, wq, "dx"), (dw, d.T.contiguous(), xq, "dw")):
        assert got.dtype == dtype
        expected = left @ right
        bound = (TERMS[dtype] * left.shape[1] * 2.0**-24 * (left.abs() @ right.abs())
                 + UNIT[dtype] * expected.abs() * (1 + 2.0**-8))
        assert_within(got, expected, bound, label)
    expected = d.sum(0)
    assert_within(db, expected, n * 2.0**-24 * d.abs().sum(0) + UNIT[dtype] * expected.abs() * (1 + 2.0**-8), "db")
    # Alone, the large one is the same kernel's.
    alone, = torch.autograd.grad(memfast.mx_linear(x, w, b), x if wide == "input" else w, dy)
    assert torch.equal(alone, dx if wide == "input" else dw)


# ---------------------------------------------------------------------------
# Codes and scales from elsewhere
# ---------------------------------------------------------------------------
def test_every_scale_byte_means_the_same_everywhere(hip_device):
    """Byte b is 2**(b - 127) from 0 on, in what is restored, in both products and in the gradient."""
    bytes_ = torch.arange(253)
    codes, scales = torch.zeros(253, 128, dtype=torch.uint8), torch.zeros(253, 8, dtype=torch.uint8)
    codes[:, :16] = torch.tensor([2 * i | (2 * i + 1) << 4 for i in range(8)] * 2, dtype=torch.uint8)
    scales[:, 0] = bytes_.to(torch.uint8)
    held = memfast.MXTensor(codes.to(hip_device), scales.to(hip_device), (253, 32))
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64).repeat(2)
    values = torch.ldexp(grid.expand(253, 32), (bytes_ - 127)[:, None])
    for dtype in TYPES.values():
        assert torch.equal(held.dequantize(dtype).cpu(), values.to(dtype))
    exponent = (127 - bytes_).clamp(-100, 100)          # brings the products near 1
    expected = torch.ldexp(values, exponent[:, None])
    for i in (0, 1, 2, 127, 252):
        for n in (3, 100):
            x = torch.eye(32).repeat(4, 1)[:n] * 2.0**float(exponent[i])
            y = memfast.mx_linear(x.to(hip_device), held)[:, i].double().cpu()
            assert torch.equal(y, expected[i].repeat(4)[:n])
    x = torch.ones(253, 32, device=hip_device, requires_grad=True)
    dy = torch.diag(torch.ldexp(torch.ones(253), exponent)).to(hip_device)
    dx, = torch.autograd.grad(memfast.mx_linear(x, held), x, dy)
    assert torch.equal(dx.double().cpu(), expected)
