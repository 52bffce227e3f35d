"""What the gated recurrence, dropout and 4-bit weights refuse before any device is asked."""

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

import memfast_amd as memfast
from memfast_amd import hip
from memfast_amd.nn import Dropout, GatedRecurrence, Int4Linear


def raises_on_cpu(call):
    with pytest.raises(hip.BackendError, match="HIP devices only"):
        call()


def test_recurrence():
    x, state, run = torch.zeros(4, 2, 6), torch.zeros(2, 3), memfast.gated_recurrence
    for bad in (x.double(), x.int(), [1.0], x.to_sparse()):
        with pytest.raises(TypeError):
            run(bad)
    for args, options, error in (
            ((x[..., :5],), {}, ValueError), ((x[0, 0],), {}, ValueError), ((x[None],), {}, ValueError),
            ((x, state[:1]), {}, ValueError), ((x, state[:, :2]), {}, ValueError),
            ((x, state.bfloat16()), {}, ValueError), ((x, state.double()), {}, TypeError),
            ((x[:, 0], state), {}, ValueError), ((x, state), dict(batch_first=True), ValueError),
            ((x,), dict(activation="relu"), ValueError),
            ((x,), dict(lengths=torch.zeros(2)), TypeError), ((x,), dict(lengths=[4, 4]), TypeError),
            ((x,), dict(lengths=torch.zeros(3).long()), ValueError),
            ((x[:, 0],), dict(lengths=torch.zeros(1).long()), ValueError)):
        with pytest.raises(error):
            run(*args, **options)
    with pytest.raises(NotImplementedError, match="channels"):
        run(torch.empty(1, 1, 1).expand(1, 1, (1 << 25) + 2))
    with pytest.raises(NotImplementedError, match="steps"):
        run(torch.empty(1, 1, 2).expand(1 << 31, 1, 2))
    raises_on_cpu(lambda: run(x, state))
    raises_on_cpu(lambda: run(x.bfloat16(), state, lengths=torch.tensor([1, 2])))
    raises_on_cpu(lambda: run(x[:, 0], state[0], lengths=torch.tensor(2)))


def test_dropout():
    x, run = torch.zeros(4, 6), memfast.dropout
    for bad in (x.double(), x.int(), [1.0]):
        with pytest.raises(TypeError):
            run(bad, 0.5, seed=1)
    with pytest.raises(TypeError):
        run(x, 0.5)
    for options, error in ((dict(seed=1.0), TypeError), (dict(seed=True), TypeError),
                           (dict(seed=-1), ValueError), (dict(seed=1 << 64), ValueError),
                           (dict(seed=1, event=-1), ValueError), (dict(seed=1, event=1.5), TypeError),
                           (dict(seed=1, event=torch.zeros(1)), TypeError),
                           (dict(seed=1, event=torch.zeros(2).long()), TypeError),
                           (dict(seed=1, residual=x[:1]), ValueError),
                           (dict(seed=1, residual=x.bfloat16()), ValueError)):
        with pytest.raises(error):
            run(x, 0.5, **options)
    for p, error in ((-0.1, ValueError), (1.1, ValueError), (float("nan"), ValueError), ("1", TypeError),
                     (True, TypeError)):
        with pytest.raises(error):
            run(x, p, seed=1)
        with pytest.raises(error):
            Dropout(p)
    for call in (lambda: run(x, 0.5, seed=1), lambda: run(x, 0.0, seed=1),
                 lambda: run(x, 0.5, seed=1, training=False)):
        raises_on_cpu(call)


def weight(o=20, k=200, group=32, dtype=torch.float32):
    return memfast.Int4Tensor.pack(torch.zeros(o, k, dtype=torch.int32),
                                   torch.ones(o, -(-k // group), dtype=dtype), group=group)


def test_held_parts():
    codes, scales = torch.zeros(2, 2, 1024, dtype=torch.uint8), torch.ones(2, 7, 16)
    make = memfast.Int4Tensor
    assert make(codes, scales, (20, 200), group=32).shape == (20, 200)
    zeros = torch.zeros(2, 7, 16, dtype=torch.uint8)
    for args, options, error in (
            ((codes, scales, (40, 200)), {}, ValueError), ((codes, scales, (20, 300)), {}, ValueError),
            ((codes, scales, (20,)), {}, ValueError), ((codes.int(), scales, (20, 200)), {}, TypeError),
            ((codes, scales.double(), (20, 200)), {}, TypeError),
            ((codes, scales, (20, 200)), dict(zeros=zeros.int()), TypeError),
            ((codes, scales, (20, 200)), dict(zeros=zeros[:1]), ValueError)):
        with pytest.raises(error):
            make(*args, group=32, **options)
    for group, error in ((16, ValueError), (48, ValueError), (0, ValueError), (32.0, TypeError),
                         (True, TypeError), (1 << 25, ValueError)):
        with pytest.raises(error):
            make(codes, scales, (20, 200), group=group)
        with pytest.raises(error):
            memfast.int4_quantize(torch.zeros(20, 200), group=group)
    q, s = torch.zeros(20, 200, dtype=torch.int32), torch.ones(20, 7)
    for args, options, error in (
            ((q - 1, s), {}, ValueError), ((q + 16, s), {}, ValueError), ((q.float(), s), {}, TypeError),
            ((q[0], s), {}, ValueError), ((q, s[:, :6]), {}, ValueError), ((q, s.int()), {}, TypeError),
            ((q, s), dict(zeros=torch.full((20, 7), 16)), ValueError),
            ((q, s), dict(zeros=torch.zeros(20, 6).int()), ValueError)):
        with pytest.raises(error):
            make.pack(*args, group=32, **options)


def test_codes_are_laid_out_as_documented():
    q = torch.randint(0, 16, (37, 300), generator=torch.Generator().manual_seed(0))
    s = torch.rand(37, 5)
    held = memfast.Int4Tensor.pack(q, s, group=64, zeros=q[:, :5])
    for o, k in ((0, 0), (36, 299), (16, 128), (15, 127), (20, 77), (31, 260)):
        i = k % 128
        byte = int(held.codes[o // 16, k // 128, (i // 8 % 4) * 256 + o % 16 * 16 + i // 32 * 4 + i % 4])
        assert (byte >> (4 if i % 8 >= 4 else 0)) & 15 == int(q[o, k])
        assert held.scales[o // 16, k // 64, o % 16] == s[o, k // 64]
        assert held.zeros[o // 16, k // 64, o % 16] == q[o, k // 64]


def test_held_products():
    x, held, run = torch.zeros(3, 200), weight(), memfast.int4_linear
    for bad in (x.double(), x.int(), [1.0]):
        with pytest.raises(TypeError):
            run(bad, held)
        with pytest.raises(TypeError):
            run(x, held, bad)
        with pytest.raises(TypeError):
            memfast.int4_quantize(bad)
    for args, error in (((x, x), TypeError), ((x[:, :199], held), ValueError),
                        ((x, held, torch.zeros(19)), ValueError),
                        ((x, held, torch.zeros(20).bfloat16()), ValueError),
                        ((x, weight(dtype=torch.bfloat16)), ValueError),
                        ((x.half(), weight(dtype=torch.bfloat16)), ValueError)):
        with pytest.raises(error):
            run(*args)
    with pytest.raises(ValueError):
        memfast.int4_quantize(x[0])
    with pytest.raises(ValueError):
        memfast.int4_quantize(x, scale_dtype=torch.float16)
    with pytest.raises(NotImplementedError, match="no gradient"):
        run(x.requires_grad_(True), held)
    with pytest.raises(NotImplementedError, match="no gradient"):
        run(x.detach(), held, torch.zeros(20, requires_grad=True))
    learned = memfast.Int4Tensor(held.codes, held.scales.clone().requires_grad_(True), held.shape, group=32)
    with pytest.raises(NotImplementedError, match="no gradient"):
        run(x.detach(), learned)
    with torch.no_grad():
        raises_on_cpu(lambda: run(x, held))
        raises_on_cpu(lambda: run(x, learned))
    raises_on_cpu(lambda: run(x.detach(), held))
    raises_on_cpu(lambda: memfast.int4_quantize(x))
    raises_on_cpu(held.dequantize)
    with pytest.raises(TypeError):
        held.dequantize(torch.float64)
    with pytest.raises(TypeError):
        Int4Linear(nn.Conv2d(1, 1, 1))
    with pytest.raises(TypeError):
        Int4Linear.from_tensor(x)


def test_forward_mode_is_refused():
    def dual(x):
        return forward_ad.make_dual(x, torch.ones_like(x))

    x, state, held = torch.zeros(4, 2, 6), torch.zeros(2, 3), weight(k=6)
    with forward_ad.dual_level():
        for call in (lambda: memfast.gated_recurrence(dual(x)),
                     lambda: memfast.gated_recurrence(x, dual(state)),
                     lambda: memfast.dropout(dual(x), seed=1),
                     lambda: memfast.dropout(x, seed=1, residual=dual(x)),
                     lambda: memfast.int4_linear(dual(x), held),
                     lambda: memfast.int4_linear(x, held, dual(torch.zeros(20))),
                     lambda: memfast.int4_linear(x, memfast.Int4Tensor(
                         held.codes, dual(held.scales), held.shape, group=32))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()


def test_library_arguments():
    """The library itself, on host memory that it refuses before it launches anything."""
    lib, at = hip.library(), torch.zeros(64).data_ptr()
    def run(**changed):
        a = dict(x=at, type=0, steps=2, batch=1, width=3, xt=6, xb=6, state=None, lengths=None, reverse=0,
                 tanh=1, y=at, yt=3, yb=3, last=at, marks=None, work=None, bytes=0, stream=None)
        return lib.mf_recurrence(*(a | changed).values())

    for changed in (dict(state=at + 2), dict(lengths=at + 4), dict(last=at + 1), dict(marks=at + 2),
                    dict(x=None), dict(type=3), dict(steps=0), dict(batch=0), dict(width=0), dict(xt=-1),
                    dict(xb=-1), dict(y=None), dict(last=None), dict(yt=-1), dict(x=at + 1),
                    dict(y=at + 2), dict(steps=100000)):     # split over workgroups: it needs a workspace
        assert run(**changed) == hip.E_INVALID, changed
    assert run(steps=1 << 31) == hip.E_UNSUPPORTED
    assert lib.mf_dropout(at, 0, 0, None, 1, 0, 0, None, at, None) == hip.E_INVALID
    assert lib.mf_dropout(at, 0, 4, None, 65537, 0, 0, None, at, None) == hip.E_INVALID
    assert lib.mf_dropout(at + 1, 0, 4, None, 1, 0, 0, None, at, None) == hip.E_INVALID
    for group in (0, 16, 33, 1 << 25):
        assert lib.mf_int4_dequantize(at, at, 0, None, 1, 1, group, at, 0, None) == hip.E_INVALID
    assert lib.mf_int4_linear(at, 0, 0, 1, 1, at, at, 0, None, 1, 32, None, at, None, 0, None) == hip.E_INVALID
    assert lib.mf_int4_linear(at, 0, 2, 2, 1, at, at, 0, None, 1, 32, None, at, None, 0, None) == hip.E_INVALID
    assert lib.mf_int4_linear(at, 1, 1, 1, 1, at, at, 2, None, 1, 32, None, at, None, 0, None) == hip.E_INVALID
    assert lib.mf_int4_quantize(at, 0, 2, 32, 31, 32, at, at, 0, None) == hip.E_INVALID


def test_layers():
    layer = GatedRecurrence(5, 4, 2, dropout=0.1, bidirectional=True)
    assert [tuple(p.weight.shape) for p in layer.projections] == [(8, 5), (8, 5), (8, 8), (8, 8)]
    for bad in (torch.zeros(3, 2, 4), torch.zeros(5), torch.zeros(0, 2, 5)):
        with pytest.raises(ValueError):
            layer(bad)
    with pytest.raises(ValueError, match="hidden state"):
        layer(torch.zeros(3, 2, 5), torch.zeros(2, 2, 4))
    with pytest.raises(ValueError):
        GatedRecurrence(5, 4, activation="relu")
    with pytest.raises(ValueError):
        GatedRecurrence(5, 0)
    raises_on_cpu(lambda: layer(torch.zeros(3, 2, 5)))
