"""Dropout whose mask is a function of a seed and an event, made anew where it is needed.

Nothing is stored between forward and backward, and the same seed and event give the same mask on
any layout, in a checkpointed layer's second forward, or after a restart.  The numbers come from
Philox 4x32-10 (Salmon et al. 2011) with the value's place, the event and the seed as its counter and key, 16
bits a value: the probability is taken to the nearest 65536th, and what is kept is divided by the exact
share that is kept.
"""

import torch

from . import hip
from .microscaling import _check_floating, _refuse_tangents

MOST_VALUES = 1 << 40


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, dropped, seed, event):
        if isinstance(event, torch.Tensor):
            ctx.save_for_backward(event)
            ctx.options = dropped, seed, None
        else:
            ctx.options = dropped, seed, event
        return hip.dropout(x, residual, dropped, seed, event)

    @staticmethod
    def backward(ctx, dy):
        dropped, seed, event = ctx.options
        if event is None:
            event, = ctx.saved_tensors
        wants_x, wants_residual = ctx.needs_input_grad[:2]
        dx = None
        if wants_x:     # linear in dy: the mask once more, and differentiable again
            dx = _apply(dy if dy.is_contiguous() else dy.contiguous(), None, dropped, seed, event)
        return dx, dy if wants_residual else None, None, None, None


def _apply(x, residual, dropped, seed, event):
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad):
        return _Dropout.apply(x, residual, dropped, seed, event)
    return hip.dropout(x, residual, dropped, seed, event)


def _number(label, value):
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{label} must be an integer")
    if not 0 <= value < 1 << 64:
        raise ValueError(f"{label} must be between 0 and 2**64 - 1")
    return value


def _check_probability(p):
    if isinstance(p, bool) or not isinstance(p, (int, float)):
        raise TypeError("p must be a number")
    if not 0 <= p <= 1:
        raise ValueError("p must be between 0 and 1")
    return p


def dropout(x, p=0.5, *, seed, event=0, residual=None, training=True):
    """``residual + x m / (1 - p)`` with ``m`` 0 for a share ``p`` of the values and 1 for the others (a
    dropped value is gone whatever it was), in x's dtype (float32, bfloat16 or float16).

    The mask is given by ``seed`` and ``event`` (whole numbers of 64 bits) and the value's place in ``x``
    taken row by row, whatever x's strides.  ``event`` may also be an int64 tensor of one value on
    x's device: a captured graph then makes a new mask wherever the tensor was counted up between
    replays.  ``p`` is taken to the nearest 65536th; with ``training=False`` or nothing to drop it is x
    itself, or ``residual + x``.  ``residual`` has x's shape and dtype.  At most 2**40 values.  An operand
    with a tangent of forward mode is refused."""
    _check_floating("x", x)
    dropped = round(_check_probability(p) * 65536)
    seed = _number("seed", seed)
    if isinstance(event, torch.Tensor):
        if event.dtype != torch.int64 or event.numel() != 1:
            raise TypeError("event must be an integer or an int64 tensor of one value")
        if event.device != x.device:
            raise ValueError("x and event must use the same device")
    else:
        event = _number("event", event)
    if residual is not None:
        _check_floating("residual", residual)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("residual must have the shape and dtype of x")
        if residual.device != x.device:
            raise ValueError("x and residual must use the same device")
    if x.numel() > MOST_VALUES:
        raise NotImplementedError(f"more than {MOST_VALUES} values")
    _refuse_tangents("dropout", x, residual)
    hip.require_device(x)
    if not training or dropped == 0 or x.numel() == 0:
        return x if residual is None else residual + x
    if not x.is_contiguous():
        x = x.contiguous()
    if residual is not None and not residual.is_contiguous():
        residual = residual.contiguous()
    return _apply(x, residual, dropped, seed, event)


__all__ = ["dropout"]
