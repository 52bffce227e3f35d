"""Weights held as 4-bit whole numbers with a scale for each group of inputs, and their product.

The digital form of the integer weights that ``Simulator.map_quantized`` imports: ``scales * (codes -
zero_points)``, here with codes of 0 .. 15 and one scale (and zero point) for ``group`` consecutive inputs of
an output.  ``int4_linear`` multiplies them with an input that is not quantized: products of codes and
inputs are summed in FP32 by group and only then scaled, so no weight is rounded.

Codes lie as the matrix instructions take them: tiles of 16 outputs by 128 inputs, 1024 bytes each, and
tables of scales and zero points by tiles of 16 outputs.  ``Int4Tensor.pack`` lays out whole numbers that
come from elsewhere.
"""

import torch

from . import hip
from .microscaling import _check_floating, _refuse_tangents

MOST_OUTPUTS, MOST_INPUTS, MOST_ROWS = (1 << 25) - 1, (1 << 24) - 1, (1 << 27) - 1


def _check_group(group):
    if isinstance(group, bool) or not isinstance(group, int):
        raise TypeError("group must be an integer")
    if group < 32 or group & group - 1 or group > 1 << 24:
        raise ValueError("group must be a power of two between 32 and 2**24")
    return group


def _check_sizes(o, k):
    if o > MOST_OUTPUTS or k > MOST_INPUTS:
        raise NotImplementedError(f"more than {MOST_OUTPUTS} outputs or {MOST_INPUTS} inputs")


_WHOLE, _FLOATING = (torch.uint8,), tuple(hip.FLOAT_TYPES)


def _part(label, value, dtypes, shape, device):
    if not isinstance(value, torch.Tensor) or value.dtype not in dtypes:
        raise TypeError(f"{label} must be a tensor of {' or '.join(str(d)[6:] for d in dtypes)}")
    if value.shape != shape:
        raise ValueError(f"{label} must have shape {shape}")
    if value.device != device:
        raise ValueError(f"codes and {label} must use the same device")
    if not value.is_contiguous():
        value = value.contiguous()
    return value if value.data_ptr() % 16 == 0 else value.clone()


def _by_tile(table):
    """[tiles, groups, 16] of a table [o, groups], with zeros past o."""
    o, groups = table.shape
    table = torch.nn.functional.pad(table, (0, 0, 0, -o % hip.INT4_TILE))
    return table.view(len(table) // hip.INT4_TILE, hip.INT4_TILE, groups).transpose(1, 2).contiguous()


class Int4Tensor:
    """A weight of ``shape`` [o, k] in 4-bit codes with groups of ``group`` inputs (a power of two from
    32 on).

    With T = ceil(o / 16) tiles, P = ceil(k / 128) and G = ceil(k / group): ``codes`` is uint8 [T, P, 1024]
    (input i of 128 and output r of 16 in byte ``(i // 8 % 4) * 256 + r * 16 + i // 32 * 4 + i % 4``, in
    its lower half if ``i % 8 < 4``), ``scales`` [T, G, 16] of float32, bfloat16 or float16, and ``zeros``
    uint8 [T, G, 16] in 0 .. 15, or None for 8 throughout.  Codes past o and k may be any."""

    def __init__(self, codes, scales, shape, *, group, zeros=None):
        self.shape = shape = torch.Size(shape)
        if len(shape) != 2:
            raise ValueError("an Int4Tensor has two dimensions")
        o, k = shape
        if o < 0 or k < 0:
            raise ValueError("an Int4Tensor has no negative dimension")
        self.group = _check_group(group)
        _check_sizes(o, k)
        if not isinstance(codes, torch.Tensor):
            raise TypeError("codes must be a tensor of uint8")
        tiles, device = -(-o // hip.INT4_TILE), codes.device
        table = (tiles, -(-k // group), hip.INT4_TILE)
        self.codes = _part("codes", codes, _WHOLE, (tiles, -(-k // hip.INT4_SPAN), hip.INT4_TILE_BYTES),
                           device)
        self.scales = _part("scales", scales, _FLOATING, table, device)
        self.zeros = None if zeros is None else _part("zeros", zeros, _WHOLE, table, device)

    @classmethod
    def pack(cls, codes, scales, *, group, zeros=None):
        """The tensor of whole numbers ``codes`` [o, k] in 0 .. 15, ``scales`` [o, ceil(k / group)] and
        ``zeros`` of the same shape in 0 .. 15 (None: 8), which is ``scales * (codes - zeros)``.  Their
        values are looked at, so this waits for the device."""
        _check_group(group)
        for label, value in (("codes", codes), ("zeros", zeros)):
            if value is None and label == "zeros":
                continue
            if not isinstance(value, torch.Tensor) or value.is_floating_point() or value.is_complex():
                raise TypeError(f"{label} must be a tensor of whole numbers")
            if value.ndim != 2:
                raise ValueError(f"{label} must have two dimensions")
            if value.numel() and not 0 <= int(value.min()) <= int(value.max()) <= 15:
                raise ValueError(f"{label} must be between 0 and 15")
        o, k = codes.shape
        if not isinstance(scales, torch.Tensor) or scales.dtype not in hip.FLOAT_TYPES:
            raise TypeError("scales must be a float32, bfloat16 or float16 tensor")
        for label, value in (("scales", scales), ("zeros", zeros)):
            if value is not None and value.shape != (o, -(-k // group)):
                raise ValueError(f"{label} must have one value per output and group")
        tiles, spans = -(-o // hip.INT4_TILE), -(-k // hip.INT4_SPAN)
        q = torch.nn.functional.pad(codes.to(torch.uint8), (0, -k % hip.INT4_SPAN, 0, -o % hip.INT4_TILE))
        # [tile, r, span, word, quarter, half, place] -> [tile, span, quarter, r, word, place, half]
        q = q.view(tiles, hip.INT4_TILE, spans, 4, 4, 2, 4).permute(0, 2, 4, 1, 3, 6, 5)
        q = (q[..., 0] | q[..., 1] << 4).reshape(tiles, spans, hip.INT4_TILE_BYTES)
        return cls(q, _by_tile(scales), (o, k), group=group,
                   zeros=None if zeros is None else _by_tile(zeros.to(torch.uint8)))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """The values that the codes stand for, rounded to ``dtype``."""
        if dtype not in hip.FLOAT_TYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        return hip.int4_dequantize(self.codes, self.scales, self.zeros, *self.shape, self.group, dtype)

    def __repr__(self):
        return f"Int4Tensor(shape={tuple(self.shape)}, group={self.group}, device={self.device})"


def int4_quantize(weight, *, group=32, scale_dtype=None):
    """``weight`` [o, k] (float32, bfloat16 or float16) as an Int4Tensor: scales ``max|w| / 7`` of each
    group, rounded to ``scale_dtype`` (the weight's dtype by default, or float32), and the nearest codes
    about a zero point of 8: -7 .. 7, and -8 .. 7 where a subnormal scale was rounded down.  A group with a NaN
    or an infinity stands for NaN.  No gradient flows through it."""
    _check_floating("weight", weight)
    _check_group(group)
    if weight.ndim != 2:
        raise ValueError("weight must have two dimensions")
    scale_dtype = weight.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in (torch.float32, weight.dtype):
        raise ValueError("scale_dtype must be float32 or the weight's dtype")
    _check_sizes(*weight.shape)
    hip.require_device(weight)
    rows = weight.detach()
    rows = hip.rows_of(rows) if rows.numel() else rows
    codes, scales = hip.int4_quantize(rows, group, scale_dtype)
    return Int4Tensor(codes, scales, weight.shape, group=group)


def int4_linear(x, weight, bias=None):
    """``x W^T + bias`` for ``x`` [..., k] and an Int4Tensor ``weight`` [o, k], in x's dtype, with FP32 sums.

    The weight's scales have x's dtype or float32, and ``bias`` [o] x's dtype.  It is a product for serving:
    an operand that wants a gradient is refused while gradients are recorded, one with a tangent of
    forward mode always.  Rows of x are below 2**27, o below 2**25 and k below 2**24.  A NaN or an infinity in a
    row of x, or sums of a group's 15 |x| beyond FP32, leave that row without finite values.  Codes are summed as
    they are and the zero point's share is taken off, so the sums' roundings are those of ``|x| s (q + z)``."""
    _check_floating("x", x)
    if not isinstance(weight, Int4Tensor):
        raise TypeError("weight must be an Int4Tensor")
    if bias is not None:
        _check_floating("bias", bias)
        if bias.dtype != x.dtype:
            raise ValueError("x and bias must have the same dtype")
        if bias.device != x.device:
            raise ValueError("x and bias must use the same device")
    if weight.scales.dtype not in (torch.float32, x.dtype):
        raise ValueError("the weight's scales must be float32 or of x's dtype")
    if weight.device != x.device:
        raise ValueError("x and weight must use the same device")
    (o, k) = weight.shape
    if x.ndim == 0 or x.shape[-1] != k:
        raise ValueError("x and weight have incompatible reduction dimensions")
    if bias is not None and bias.shape != (o,):
        raise ValueError("bias must have one value per output")
    if torch.is_grad_enabled() and (x.requires_grad or weight.scales.requires_grad or
                                    bias is not None and bias.requires_grad):
        raise NotImplementedError("int4_linear has no gradient; call it under torch.no_grad()")
    _refuse_tangents("int4_linear", x, weight.scales, bias)
    hip.require_device(x)
    shape = x.shape[:-1] + (o,)
    if x.numel() == 0 or o == 0:
        y = torch.zeros(shape, dtype=x.dtype, device=x.device)
        return y if bias is None else y + bias
    if x.numel() // k > MOST_ROWS:
        raise NotImplementedError(f"more than {MOST_ROWS} rows")
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    y = hip.int4_linear(hip.rows_of(x), weight.codes, weight.scales, weight.zeros, o, weight.group, bias)
    return y if y.shape == shape else y.reshape(shape)


__all__ = ["Int4Tensor", "int4_quantize", "int4_linear"]
