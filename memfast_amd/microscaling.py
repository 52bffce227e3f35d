"""4-bit microscaled floating point: quantized tensors and their linear product.

The digital number format that an analog layer is compared with, and that the layers which
stay digital (a classifier head, a distillation teacher) are held in.  Blocks of 32
consecutive values along the last dimension share a power-of-two scale 2**e with
``e = max(floor(log2(max|x|)) - 2, -126)``; a value's code is ``x / 2**e`` rounded to nearest even
on {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign, saturating at 6.  A block that holds a NaN or an
infinity stands for NaN.

``mx_quantize`` makes an ``MXTensor`` of codes and scales, ``mx_linear`` multiplies two such
operands on the matrix cores with FP32 sums.  Its backward passes gradients straight through
both quantizers: ``dx = dy Q(W)``, ``dw = dy^T Q(x)``, as the surrogate of the hardware-aware layers
does (memfast_amd/nn/training.py).  Nothing is read back to the host, so a non-finite operand
shows as NaN in the result and raises nothing.
"""

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import hip


def _check_floating(label, value):
    if not isinstance(value, torch.Tensor):
        raise TypeError(f"{label} must be a torch.Tensor")
    if value.layout != torch.strided or value.dtype not in hip.FLOAT_TYPES:
        raise TypeError(f"{label} must be a dense float32, bfloat16 or float16 tensor")


class MXTensor:
    """Codes and scales of a 4-bit tensor of ``shape``, whose last dimension k is blocked.

    ``codes`` is uint8 [rows, 128 * S] with S = ceil(k / 256), two codes a byte, the even value in
    the lower half, codes past k zero; ``scales`` is uint8 [rows, 8 * S], e + 127 of each block (255:
    NaN; not in blocks past k).  rows is the product of the other dimensions.  Codes from elsewhere
    may have any e from -127 on; a value beyond FP32's range (e of 126 and 127) is infinite in
    ``dequantize`` and in gradients."""

    def __init__(self, codes, scales, shape):
        self.shape = shape = torch.Size(shape)
        if not shape:
            raise ValueError("an MXTensor has at least one dimension")
        rows, segments = math.prod(shape[:-1]), -(-shape[-1] // hip.MX_SEGMENT)
        self.codes = _part("codes", codes, (rows, hip.MX_SEGMENT_BYTES * segments))
        self.scales = _part("scales", scales, (rows, hip.MX_SEGMENT_SCALES * segments))
        if codes.device != scales.device:
            raise ValueError("codes and scales must use the same device")

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """The values that the codes stand for, rounded to ``dtype``."""
        if dtype not in hip.FLOAT_TYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        return hip.mx_dequantize(self.codes, self.scales, self.shape[-1], dtype).reshape(self.shape)

    def __repr__(self):
        return f"MXTensor(shape={tuple(self.shape)}, device={self.device})"


def _refuse_tangents(name, *operands):
    """The operators have no forward-mode derivative: an operand with a tangent is refused, as the
    autograd functions do where some operand wants a gradient."""
    if getattr(forward_ad, "_current_level", 0) < 0:     # outside forward mode, the usual case
        return
    for value in operands:
        if isinstance(value, torch.Tensor) and forward_ad.unpack_dual(value).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


def _part(label, value, shape):
    """``value``, checked, contiguous and at a 16-byte address, as the kernels load it."""
    if not isinstance(value, torch.Tensor) or value.dtype != torch.uint8:
        raise TypeError(f"{label} must be a uint8 tensor")
    if value.shape != shape:
        raise ValueError(f"{label} must have shape {shape}")
    if not value.is_contiguous():
        value = value.contiguous()
    return value if value.data_ptr() % 16 == 0 else value.clone()


def mx_quantize(x):
    """``x`` (float32, bfloat16 or float16, blocked along its last dimension) as an MXTensor.  It has
    fewer than 2**28 rows of fewer than 2**24 values; no gradient flows through it."""
    _check_floating("x", x)
    if x.ndim == 0:
        raise ValueError("x must have at least one dimension")
    hip.require_device(x)
    if x.numel() == 0:
        codes, scales = hip.mx_empty(math.prod(x.shape[:-1]), x.shape[-1], x.device)
        return MXTensor(codes, scales, x.shape)
    codes, scales = hip.mx_quantize(hip.rows_of(x.detach()))
    return MXTensor(codes, scales, x.shape)


class _MXLinear(torch.autograd.Function):
    """Product of Q(x) and Q(weight), or of a weight held in ``codes`` and ``scales``."""

    @staticmethod
    def forward(ctx, x, weight, bias, codes, scales):
        y, block = hip.mx_linear(x, weight, codes, scales, bias, ctx.needs_input_grad[1])
        ctx.width = x.shape[1]
        # A held weight's gradients need none of what the call quantized.
        ctx.save_for_backward(codes, scales, block if codes is None else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():     # create_graph: the gradients are not differentiable
            return once_differentiable(_MXLinear._grads)(ctx, dy)
        return _MXLinear._grads(ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        codes, scales, block = ctx.saved_tensors
        return (*hip.mx_grads(hip.rows_of(dy), ctx.width, codes, scales, block,
                              ctx.needs_input_grad[:3]), None, None)


def mx_linear(x, weight, bias=None):
    """``Q(x) Q(weight)^T + bias`` for ``x`` [..., k] and ``weight`` [o, k], in x's dtype.

    ``weight`` is an MXTensor, or a tensor of x's dtype that is quantized in the call and gets a
    gradient.  ``bias`` [o] has x's dtype.  Rows of x and o are below 2**28 and k below 2**24; where a
    gradient is wanted, x has at most 2**24 - 1 rows and o is at most 2**22.  An operand with a
    tangent of forward mode is refused."""
    _check_floating("x", x)
    held = isinstance(weight, MXTensor)
    if not held:
        _check_floating("weight", weight)
    if bias is not None:
        _check_floating("bias", bias)
    if not held and weight.dtype != x.dtype:
        raise ValueError("x and weight must have the same dtype")
    if bias is not None and bias.dtype != x.dtype:
        raise ValueError("x and bias must have the same dtype")
    if weight.device != x.device:
        raise ValueError("x and weight must use the same device")
    if bias is not None and bias.device != x.device:
        raise ValueError("x and bias must use the same device")
    if x.ndim == 0 or len(weight.shape) != 2:
        raise ValueError("mx_linear takes x [..., k] and weight [o, k]")
    (o, k) = weight.shape
    if x.shape[-1] != k:
        raise ValueError("x and weight have incompatible reduction dimensions")
    if bias is not None and bias.shape != (o,):
        raise ValueError("bias must have one value per output")
    _refuse_tangents("mx_linear", x, weight, bias)
    hip.require_device(x)
    shape = x.shape[:-1] + (o,)
    if x.numel() == 0 or o == 0:
        # Nothing to sum: zeros, or the bias, tied to the operands for autograd.
        y = x.sum(-1, keepdim=True).expand(shape) * 0
        if not held:
            y = y + weight.sum(-1) * 0
        return y if bias is None else y + bias
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    recorded = torch.is_grad_enabled() and (x.requires_grad or not held and weight.requires_grad or
                                            bias is not None and bias.requires_grad)
    if recorded and (x.numel() // k > hip.MX_GRAD_ROWS or o > hip.MX_GRAD_OUTPUTS):
        raise NotImplementedError(f"gradients of more than {hip.MX_GRAD_ROWS} rows or "
                                  f"{hip.MX_GRAD_OUTPUTS} outputs")
    codes, scales = (weight.codes, weight.scales) if held else (None, None)
    weight = None if held else hip.rows_of(weight)
    rows = hip.rows_of(x)
    if recorded:
        y = _MXLinear.apply(rows, weight, bias, codes, scales)
    else:
        y = hip.mx_linear(rows, weight, codes, scales, bias, False)[0]
    return y if y.shape == shape else y.reshape(shape)


__all__ = ["MXTensor", "mx_quantize", "mx_linear"]
