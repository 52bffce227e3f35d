"""Distillation of a student from a teacher's top logits.

A network converted to analog layers (``convert_model(..., training=True)``) is tuned against
its digital original.  The original's whole output need not be kept: ``top_logits`` gives its k
largest logits per row and the logarithm of the mass of all others, and ``distillation_loss``
the student's loss against them, with its gradient.

Sums over the classes are held in FP32, over the entries and buckets in FP64, and nothing is read
back to the host; a row whose indices are wrong has a NaN loss.  The largest logits take one pass
over a row, or up to ten where it holds a NaN or many candidates (it rises all along, or k is above
about 800); the loss takes one, with its gradient two.  Temperatures are normal numbers of FP32.
"""

import torch
from torch.autograd.function import once_differentiable

from . import hip
from .microscaling import _check_floating, _refuse_tangents

MOST_ENTRIES, MOST_CLASSES = 1024, 1 << 20
# 1 / T is formed in FP32: below its smallest normal number it would be infinite.
LEAST_TEMPERATURE, MOST_TEMPERATURE = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def _check_temperature(temperature):
    if isinstance(temperature, bool) or not isinstance(temperature, (int, float)):
        raise TypeError("temperature must be a number")
    if not LEAST_TEMPERATURE <= temperature <= MOST_TEMPERATURE:
        raise ValueError("temperature must be a positive normal number of float32")
    return float(temperature)


def _check_logits(logits):
    _check_floating("logits", logits)
    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must have at least one class in their last dimension")
    if logits.shape[-1] > MOST_CLASSES:
        raise NotImplementedError(f"more than {MOST_CLASSES} classes")


def top_logits(logits, k, *, temperature=1.0):
    """(values, indices, tail) of ``logits`` [..., V]: the ``k`` largest in descending order
    [..., k], the lowest index first among equal ones (NaN counts as the largest), their indices
    (int64), and ``log(sum(exp(logits / temperature)))`` of the others [...] in FP32 (-inf where
    none is left).  No gradient flows through them."""
    _check_logits(logits)
    temperature = _check_temperature(temperature)
    if isinstance(k, bool) or not isinstance(k, int):
        raise TypeError("k must be an integer")
    if not 1 <= k <= logits.shape[-1]:
        raise ValueError("k must be between 1 and the number of classes")
    if k > MOST_ENTRIES:
        raise NotImplementedError(f"more than {MOST_ENTRIES} entries")
    hip.require_device(logits)
    lead = logits.shape[:-1]
    rows = logits.detach()
    rows = hip.rows_of(rows) if rows.numel() else rows.reshape(0, rows.shape[-1])
    values, indices, tail = hip.top_logits(rows, k, temperature)
    return values.reshape(lead + (k,)), indices.reshape(lead + (k,)), tail.reshape(lead)


class _Distillation(torch.autograd.Function):
    """A sum or mean computes its gradient with the loss, while a row is in the cache: for an
    incoming gradient of 1, as a loss that is differentiated itself gets. The first backward hands
    it out, computed again from the logits where the incoming gradient is another; further ones
    through the same graph compute their own."""

    @staticmethod
    def forward(ctx, logits, values, indices, tail, weight, temperature, reduction):
        loss, stats, grad = hip.distill_loss(
            logits, values, indices, tail, temperature, weight, reduction, reduction != "none")
        ctx.save_for_backward(logits, indices, weight, stats)
        ctx.options, ctx.ready = (temperature, reduction), grad
        return _weighted(loss, weight) if reduction == "none" else loss

    @staticmethod
    def backward(ctx, incoming):
        if torch.is_grad_enabled():     # create_graph: the gradient is not differentiable
            return once_differentiable(_Distillation._grad)(ctx, incoming)
        return _Distillation._grad(ctx, incoming)

    @staticmethod
    def _grad(ctx, incoming):
        logits, indices, weight, stats = ctx.saved_tensors
        temperature, reduction = ctx.options
        ready, ctx.ready = ctx.ready, None
        if incoming.dtype != torch.float32 or not incoming.is_contiguous():
            incoming = incoming.to(torch.float32).contiguous()
        grad = hip.distill_grad(logits, indices, temperature, weight, stats, reduction, incoming,
                                ready)
        return grad, None, None, None, None, None, None


def _weighted(row_loss, weight):
    return row_loss if weight is None else torch.where(weight == 0, 0.0, weight * row_loss)


def distillation_loss(logits, values, indices, tail=None, *, temperature=1.0, weight=None,
                      reduction="mean"):
    """Loss of the student's ``logits`` [..., V] against a teacher's top logits.

    ``values`` and ``indices`` [..., k] are the teacher's logits and their classes, ``tail`` [...]
    the logarithm of its other classes' sum at ``temperature`` (``top_logits`` gives all three).
    An index of -1 marks an entry that is absent.  With ``p = softmax([values / T, tail])`` and ``q``
    the student's ``softmax(logits / T)`` over the same entries and one bucket for all other
    classes, a row's loss is ``T**2 * sum(p * log(p / q))``; without ``tail`` the teacher's bucket is
    empty.  A row without any entry or tail has no loss.  A row with an index outside -1 .. V - 1
    or with a repeated one has a NaN loss.

    ``weight`` [...] weighs the rows (bool or floating; a row of weight 0 is not read).
    ``reduction``: "mean" (over the weights' sum; 0 if that is 0), "sum" or "none".  The loss is FP32;
    gradients reach ``logits`` alone.  A sum or mean writes the gradient with the loss, for a loss that is
    differentiated itself; where it is first scaled or joined by another factor, the backward writes it
    again (``reduction="none"`` writes it in the backward alone).  An operand with a tangent of forward
    mode is refused."""
    _check_logits(logits)
    _check_floating("values", values)
    temperature = _check_temperature(temperature)
    if reduction not in hip.REDUCTIONS:
        raise ValueError("reduction must be mean, sum or none")
    if not isinstance(indices, torch.Tensor) or indices.dtype not in (torch.int64, torch.int32):
        raise TypeError("indices must be an int64 or int32 tensor")
    lead = logits.shape[:-1]
    if values.ndim != logits.ndim or values.shape[:-1] != lead or values.shape[-1] == 0:
        raise ValueError("values must have the rows of logits and at least one entry")
    if indices.shape != values.shape:
        raise ValueError("values and indices must have the same shape")
    k = values.shape[-1]
    if k > logits.shape[-1]:
        raise ValueError("more entries than classes")
    if k > MOST_ENTRIES:
        raise NotImplementedError(f"more than {MOST_ENTRIES} entries")
    for label, value in (("tail", tail), ("weight", weight)):
        if value is None:
            continue
        if not isinstance(value, torch.Tensor) or not (
                value.is_floating_point() or label == "weight" and value.dtype == torch.bool):
            raise TypeError(f"{label} must be a floating tensor")
        if value.shape != lead:
            raise ValueError(f"{label} must have one value per row")
    for label, value in (("values", values), ("indices", indices), ("tail", tail),
                         ("weight", weight)):
        if value is not None and value.device != logits.device:
            raise ValueError(f"logits and {label} must use the same device")
    _refuse_tangents("distillation_loss", logits, values, tail, weight)
    hip.require_device(logits)
    if logits.numel() == 0:
        zero = logits.sum(-1).float()
        return zero if reduction == "none" else zero.sum()

    rows = hip.rows_of(logits)
    entries = _matrix(values, k)
    indices = _matrix(indices if indices.dtype == torch.int64 else indices.to(torch.int64), k)
    tail, weight = _per_row(tail), _per_row(weight)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = _Distillation.apply(rows, entries, indices, tail, weight, temperature, reduction)
    else:
        loss = hip.distill_loss(rows, entries, indices, tail, temperature, weight, reduction, False)[0]
        if reduction == "none":
            loss = _weighted(loss, weight)
    return loss.reshape(lead) if reduction == "none" else loss


def _matrix(value, k):
    return value if value.ndim == 2 and value.is_contiguous() else value.reshape(-1, k).contiguous()


def _per_row(value):
    if value is None or value.dtype == torch.float32 and value.ndim == 1 and value.is_contiguous():
        return value
    return value.detach().to(torch.float32).reshape(-1).contiguous()


__all__ = ["top_logits", "distillation_loss"]
