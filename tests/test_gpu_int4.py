"""Products with weights in 4-bit whole numbers against the formula in 64 bits.

Bounds.  Products of a code (0 .. 15) and an input are exact, their sum over a group and that of the inputs are
FP32 sums in the order of the matrix cores: with m terms off by at most m 2^-24 of the terms' sizes (the
cores may drop bits below 2^-24 of the largest term too, so twice that), then joined over groups, waves
and the bias by FP32 additions.  With |q| + |z| in the place of |q - z|, K = k + groups + 16 additions bound
the error by 2 K 2^-24 sum |x| s (q + z).  Results of 16-bit types are off by half a step more.
"""

import math

import pytest
import torch
from torch import nn

import memfast_amd as memfast
from memfast_amd.nn import Int4Linear

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def weight(device, o, k, group, dtype, zeros, seed=0):
    """Whole numbers, tables and the tensor that holds them."""
    gen = torch.Generator().manual_seed(seed + 3 * o + 5 * k)
    q = torch.randint(0, 16, (o, k), generator=gen)
    groups = -(-k // group)
    s = (0.01 * (0.2 + torch.rand(o, groups, generator=gen))).to(dtype)
    z = torch.randint(0, 16, (o, groups), generator=gen) if zeros else None
    held = memfast.Int4Tensor.pack(q.to(device), s.to(device), group=group,
                                   zeros=None if z is None else z.to(device))
    return q, s, z, held


def expected(x, q, s, z, group, bias):
    """y and the bound's sum in 64 bits."""
    k = q.shape[1]

    def spread(table):
        return table.double()[:, torch.arange(k) // group]

    zero = torch.full_like(q, 8).double() if z is None else spread(z)
    x = x.double().cpu()
    y = x @ (spread(s) * (q.double() - zero)).T
    terms = x.abs() @ (spread(s) * (q.double() + zero)).T
    if bias is not None:
        y, terms = y + bias.double().cpu(), terms + bias.double().cpu().abs()
    return y, terms


def near(got, y, terms, k, group):
    info = torch.finfo(got.dtype)
    bound = 2 * (k + k // group + 16) * 2.0**-24 * terms
    if got.dtype != torch.float32:
        bound = bound + info.eps / 2 * (y.abs() + bound) + info.smallest_normal * info.eps
    off = (got.double().cpu() - y).abs()
    assert got.shape == y.shape
    assert bool((off <= bound + 1e-37).all()), float((off / bound).max())


def check(device, n, k, o, group, kind, zeros=False, bias=True, scales=None, seed=0):
    dtype = TYPES[kind]
    q, s, z, held = weight(device, o, k, group, scales or dtype, zeros, seed)
    gen = torch.Generator().manual_seed(seed + n)
    x = torch.randn(n, k, generator=gen).to(dtype).to(device)
    b = torch.randn(o, generator=gen).to(dtype).to(device) if bias else None
    y = memfast.int4_linear(x, held, b)
    near(y, *expected(x, q, s, z, group, b), k, group)
    return x, held, b, y


ROWS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 48, 49, 64, 65, 100, 128, 129, 200]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", ROWS)
def test_rows(hip_device, kind, n):
    check(hip_device, n, 384, 80, 32, kind)
    check(hip_device, n, 1000, 50, 128, kind, zeros=True, bias=False)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("k,o", [(1, 1), (31, 15), (32, 16), (33, 17), (127, 100), (128, 256), (129, 300),
                                 (255, 31), (511, 33), (640, 257), (1028, 513), (4096, 7)])
def test_sizes(hip_device, kind, k, o):
    for n in (1, 6, 40, 130):
        check(hip_device, n, k, o, 32, kind, zeros=n == 6)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,o", [(65, 300, 17000), (200, 1024, 4200), (129, 130, 5600), (300, 1000, 4096),
                                   (1000, 96, 1100), (8200, 40, 300), (8193, 256, 140), (9000, 33, 100)])
def test_large_tiles_and_many_rows(hip_device, kind, n, k, o):
    """Tiles of 64 by 256 with their spans split or not, and rows taken 8192 at a time."""
    for group, zeros in ((32, False), (128, True), (64, True), (256, False)):
        check(hip_device, n, k, o, group, kind, zeros=zeros, bias=zeros)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_scalings_of_a_span(hip_device, kind, group, zeros):
    """One, two and four in the wide tiles and in both of the small ones, scales of either type."""
    for n, k, o in ((260, 1000, 4100), (70, 900, 300), (30, 3000, 600), (48, 4000, 4100)):
        check(hip_device, n, k, o, group, kind, zeros=zeros)
        if kind != "fp32":
            check(hip_device, n, k, o, group, kind, zeros=zeros, scales=torch.float32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,k,o", [(17, 600, 8200), (6, 300, 8193), (32, 264, 8192), (64, 1032, 500),
                                   (40, 8, 33), (24, 11008, 400), (48, 4096, 300)])
def test_between_few_rows_and_tiles(hip_device, kind, n, k, o):
    """Both sides of the rules that choose a kernel."""
    for group, zeros in ((32, True), (128, False)):
        check(hip_device, n, k, o, group, kind, zeros=zeros)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("group", [32, 64, 128, 256, 1024, 1 << 24])
@pytest.mark.parametrize("zeros", [False, True])
def test_groups(hip_device, kind, group, zeros):
    for n in (1, 20, 150):
        for k in (100, 700, 1500):
            check(hip_device, n, k, 70, group, kind, zeros=zeros)
            if kind != "fp32":
                check(hip_device, n, k, 70, group, kind, zeros=zeros, scales=torch.float32)


@pytest.mark.parametrize("kind", list(TYPES))
def test_strides_and_alignment(hip_device, kind):
    """Views of x give what their copies give, to the bit where both are summed alike."""
    for n in (1, 7, 150):
        for k in (256, 200):
            q, s, z, held = weight(hip_device, 90, k, 64, TYPES[kind], True)
            wide = torch.randn(2 * n, k + 24, device=hip_device).to(TYPES[kind])
            for view in (wide[::2, :k], wide[n:, 3:k + 3], wide[:n, 8:k + 8], wide[:1, :k].expand(n, k),
                         wide.T[:k, :n].T, wide[:n, :k].unsqueeze(0)):
                y = memfast.int4_linear(view, held)
                assert torch.equal(y, memfast.int4_linear(view.contiguous(), held))
                near(y.reshape(-1, 90), *expected(view.reshape(-1, k), q, s, z, 64, None), k, 64)
    # A misplaced bias and tables.
    q, s, z, held = weight(hip_device, 90, 256, 64, TYPES[kind], True)
    moved = memfast.Int4Tensor(*(torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)
                                 for t in (held.codes, held.scales)), (90, 256), group=64,
                               zeros=held.zeros)
    x = torch.randn(3, 256, device=hip_device).to(TYPES[kind])
    bias = torch.randn(181, device=hip_device).to(TYPES[kind])[1::2]
    assert torch.equal(memfast.int4_linear(x, held, bias), memfast.int4_linear(x, moved, bias.contiguous()))
    assert memfast.int4_linear(x[0], held).shape == (90,)


def test_codes_past_the_edges_may_be_any(hip_device):
    for kind in TYPES:
        for n in (1, 30, 140):
            x, held, b, y = check(hip_device, n, 77, 21, 32, kind)
            full = torch.full_like(held.codes, 255)
            inside = memfast.Int4Tensor.pack(torch.full((21, 77), 15, device=hip_device),
                                             torch.zeros(21, 3, device=hip_device), group=32).codes != 0
            codes = torch.where(inside, held.codes, full)
            # Bytes whose lower half alone lies within k keep that half.
            low = memfast.Int4Tensor.pack(torch.full((21, 77), 15, device=hip_device),
                                          torch.zeros(21, 3, device=hip_device), group=32).codes == 15
            codes = torch.where(low, held.codes | 0xF0, codes)
            other = memfast.Int4Tensor(codes, held.scales, (21, 77), group=32)
            assert torch.equal(memfast.int4_linear(x, other, b), y)


def test_values_that_are_not_finite(hip_device):
    """They stay in their rows of x, and in the outputs of their scale."""
    for kind in TYPES:
        for n in (3, 20, 140):
            q, s, z, held = weight(hip_device, 40, 300, 32, TYPES[kind], False)
            x = torch.randn(n, 300, device=hip_device).to(TYPES[kind])
            fine = memfast.int4_linear(x, held)
            x[0, 17], x[2, 250] = math.inf, math.nan
            y = memfast.int4_linear(x, held)
            assert not bool(y[[0, 2]].isfinite().any())
            rest = [r for r in range(n) if r not in (0, 2)]
            assert torch.equal(y[rest], fine[rest])
            scales = held.scales.clone()
            scales[1, 4, 3] = math.nan                       # output 19
            y = memfast.int4_linear(x, memfast.Int4Tensor(held.codes, scales, (40, 300), group=32))
            assert bool(y[:, 19].isnan().all())
            others = [c for c in range(40) if c != 19]
            assert torch.equal(y[rest][:, others], fine[rest][:, others])


def test_one_row_of_any_distance(hip_device):
    flat = torch.randn(64, device=hip_device)
    q, s, z, held = weight(hip_device, 20, 64, 32, torch.float32, False)
    one = flat.as_strided((1, 64), (1, 1))
    assert torch.equal(memfast.int4_linear(one, held), memfast.int4_linear(flat, held)[None])
    assert torch.equal(memfast.int4_quantize(one).codes, memfast.int4_quantize(flat[None]).codes)


def test_subnormal_inputs(hip_device):
    """FP16's subnormal numbers, and FP32 numbers whose lower terms are far below, count."""
    for n in (1, 40, 150):
        for o in (40, 6000):
            q, s, z, held = weight(hip_device, o, 256, 32, torch.float32, False)
            x = (torch.randint(-8, 9, (n, 256)).float() * 2.0**-24).half().to(hip_device)
            y, terms = expected(x, q, s, z, 32, None)
            got = memfast.int4_linear(x, held)
            assert bool(((got.double().cpu() - y).abs() <= 2.0**-25 + 2.0**-12 * terms).all())
            assert float(y.abs().max()) > 2.0**-22
            x = torch.randn(n, 256, device=hip_device) * 2.0**-90
            near(memfast.int4_linear(x, held), *expected(x, q, s, z, 32, None), 256, 32)


def test_exact_sums(hip_device):
    """Whole numbers whose sums fit FP32 come out exactly, in every type, whatever is split."""
    for kind in TYPES:
        for n in (1, 5, 16, 40, 64, 150):
            q, _, z, _ = weight(hip_device, 100, 900, 64, torch.float32, True)
            s = torch.full((100, 15), 0.5)
            held = memfast.Int4Tensor.pack(q.to(hip_device), s.to(hip_device), group=64,
                                           zeros=z.to(hip_device))
            x = torch.randint(-8, 9, (n, 900)).to(TYPES[kind]).to(hip_device)
            y, _ = expected(x, q, s, z, 64, None)
            assert torch.equal(memfast.int4_linear(x, held).double().cpu(), y.to(TYPES[kind]).double())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("o,k,group", [(1, 1, 32), (17, 100, 32), (33, 300, 64), (16, 128, 128),
                                       (40, 1000, 256), (20, 700, 512), (5, 3000, 1024),
                                       (3, 5001, 4096)])
def test_quantization(hip_device, kind, o, k, group):
    """Scales max|w| / 7 in their type, nearest codes, and the values that they stand for."""
    dtype = TYPES[kind]
    gen = torch.Generator().manual_seed(o)
    w = torch.randn(o, k, generator=gen).to(dtype)
    w[0, :min(32, k)] = 0
    for scale_dtype in {dtype, torch.float32}:
        held = memfast.int4_quantize(w.to(hip_device), group=group, scale_dtype=scale_dtype)
        groups = -(-k // group)
        spans = nn.functional.pad(w.float(), (0, -k % group)).view(o, groups, group)
        peak = spans.abs().amax(-1)
        s = torch.where(peak > 0, peak / 7, 1.0).to(scale_dtype)
        q = torch.round(spans / s.float()[..., None]).clamp(-8, 7).view(o, -1)[:, :k] + 8
        same = memfast.Int4Tensor.pack(q.to(torch.uint8).to(hip_device), s.to(hip_device), group=group)
        assert torch.equal(held.scales, same.scales) and held.zeros is None
        values = s.float()[:, torch.arange(k) // group] * (q - 8)
        for out in TYPES.values():
            assert torch.equal(held.dequantize(out).cpu(), values.to(out))
        # The product does not look at codes past the edges, but they are the code of 0.
        assert torch.equal(held.dequantize(), same.dequantize())
    view = torch.randn(o, 2 * k + 1, generator=gen).to(dtype).to(hip_device)[:, 1:k + 1]
    assert torch.equal(memfast.int4_quantize(view, group=group).codes,
                       memfast.int4_quantize(view.contiguous(), group=group).codes)


def test_quantization_at_the_edges(hip_device):
    w = torch.randn(20, 96, device=hip_device)
    w[3, 40], w[5, 0], w[7, 95] = math.nan, math.inf, -math.inf
    values = memfast.int4_quantize(w).dequantize()
    bad = torch.zeros(20, 96, dtype=torch.bool, device=hip_device)
    bad[3, 32:64] = bad[5, :32] = bad[7, 64:] = True
    assert torch.equal(values.isnan(), bad)
    tiny = torch.full((1, 32), 1e-44, device=hip_device)      # scales beneath their type
    assert bool(memfast.int4_quantize(tiny).dequantize().isfinite().all())
    tiny = torch.full((1, 32), 6e-8, device=hip_device).half()
    assert bool(memfast.int4_quantize(tiny).dequantize().isfinite().all())
    for shape in ((0, 64), (3, 0)):
        held = memfast.int4_quantize(torch.zeros(shape, device=hip_device))
        assert held.dequantize().shape == shape
        y = memfast.int4_linear(torch.zeros(2, shape[1], device=hip_device), held)
        assert y.shape == (2, shape[0]) and bool((y == 0).all())
    held = memfast.int4_quantize(torch.zeros(3, 0, device=hip_device))
    bias = torch.randn(3, device=hip_device)
    assert torch.equal(memfast.int4_linear(torch.zeros(2, 0, device=hip_device), held, bias),
                       bias.expand(2, 3))
    held = memfast.int4_quantize(torch.zeros(3, 64, device=hip_device))
    assert memfast.int4_linear(torch.zeros(0, 64, device=hip_device), held).shape == (0, 3)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,o", [(1, 300), (24, 300), (150, 300), (200, 4200)])
def test_captured_streams_and_repeats(hip_device, kind, n, o):
    x, held, b, y = check(hip_device, n, 1100, o, 64, kind, zeros=True)
    for _ in range(5):
        assert torch.equal(memfast.int4_linear(x, held, b), y)
    graph = torch.cuda.CUDAGraph()
    inside = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        elsewhere = [memfast.int4_linear(x, held, b) for _ in range(2)]
    torch.cuda.current_stream().wait_stream(side)
    for e in elsewhere:
        assert torch.equal(e, y)
    with torch.cuda.graph(graph):
        first = memfast.int4_linear(inside, held, b)
        second = memfast.int4_linear(inside * 2, held, b)
    for factor in (1, -1, 3):
        inside.copy_(x * factor)
        graph.replay()
        a, c = memfast.int4_linear(x * factor, held, b), memfast.int4_linear(x * factor * 2, held, b)
        torch.cuda.synchronize()
        assert torch.equal(first, a) and torch.equal(second, c)


def test_more_outputs_than_tiles_of_a_launch(hip_device):
    """Many outputs of one group: codes beyond 2^31 bytes from each other are not needed for that."""
    o = (1 << 20) + 7
    q = torch.randint(0, 16, (o, 32), device=hip_device)
    held = memfast.Int4Tensor.pack(q, torch.ones(o, 1, device=hip_device), group=32)
    x = torch.randint(-4, 5, (2, 32), device=hip_device).float()
    assert torch.equal(memfast.int4_linear(x, held), x @ (q.float() - 8).T)


def test_codes_beyond_32_bits(hip_device):
    """A weight of more than 2^32 bytes of codes; its last tile is where it should be."""
    o, k = 33000, 1 << 18
    codes = torch.full((-(-o // 16), k // 128, 1024), 0x88, dtype=torch.uint8, device=hip_device)
    codes[-1] = 0x99
    scales = torch.ones(-(-o // 16), 1, 16, device=hip_device)
    held = memfast.Int4Tensor(codes, scales, (o, k), group=1 << 18)
    for n in (1, 80):
        y = memfast.int4_linear(torch.ones(n, k, device=hip_device), held)
        tail = o - (o - 1) // 16 * 16
        assert bool((y[:, :-tail] == 0).all()) and bool((y[:, -tail:] == k).all())


def test_models_with_held_layers_are_converted(hip_device):
    """convert_model copies and keeps them; moving the model moves codes and tables."""
    torch.manual_seed(1)
    config = memfast.Config(activation_bits=8, weight_bits=8, input_slice=(1, 1, 2, 2, 2),
                            weight_slice=(1, 1, 2, 2, 2), array_size=(128, 128), rows_per_read=32,
                            nonidealities=memfast.Nonidealities(write_variation=0.0))
    head = Int4Linear(nn.Linear(24, 10).to(hip_device))
    model = nn.Sequential(nn.Linear(40, 24).to(hip_device), head)
    analog = memfast.convert_model(model, memfast.Simulator(config, device=hip_device))
    assert isinstance(analog[0], memfast.AnalogLinear) and isinstance(analog[1], Int4Linear)
    x = torch.randn(5, 40, device=hip_device)
    with torch.no_grad():
        assert torch.equal(analog(x), head(analog[0](x)))
        short = Int4Linear(nn.Linear(24, 10).to(hip_device)).bfloat16()
        y = short(x[:, :24].bfloat16())
        assert y.dtype == torch.bfloat16 and short.codes.dtype == torch.uint8
    assert analog[1].cpu().codes.device.type == "cpu"


def test_layer(hip_device):
    torch.manual_seed(0)
    linear = nn.Linear(200, 70).to(hip_device)
    layer = Int4Linear(linear, group=64)
    x = torch.randn(3, 4, 200, device=hip_device)
    with torch.no_grad():
        y = layer(x)
        held = memfast.int4_quantize(linear.weight, group=64)
        assert torch.equal(y, memfast.int4_linear(x, held, linear.bias))
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(layer(x), y)
        other = Int4Linear(nn.Linear(200, 70).to(hip_device), group=64)
        other.load_state_dict(layer.state_dict())
        assert torch.equal(other(x), y)
        imported = Int4Linear.from_tensor(held)
        assert torch.equal(imported(x), memfast.int4_linear(x, held)) and imported.bias is None
    with pytest.raises(NotImplementedError, match="no gradient"):
        layer(x.requires_grad_(True))


def test_imported_weights_agree_with_the_analog_import(hip_device):
    """Codes, scales and zero points as Simulator.map_quantized takes them stand for the same weight."""
    q = torch.randint(0, 16, (24, 64), device=hip_device)
    s = torch.rand(24, 2, device=hip_device) + 0.5
    z = torch.randint(0, 16, (24, 2), device=hip_device)
    held = memfast.Int4Tensor.pack(q, s, group=32, zeros=z)
    assert torch.equal(held.dequantize(), s.repeat_interleave(32, 1) * (q - z.repeat_interleave(32, 1)))
