"""A gated linear recurrence over sequences, with its gradients.

The recurrence of a GRU whose gates depend on the input alone: every projection of a sequence is
then one product (one read of an analog layer, where ``AnalogGRU`` makes one a step), and each channel is
left with ``h_t = u_t h_{t-1} + (1 - u_t) c_t``.  ``nn.GatedRecurrence`` is the layer.

States are held in FP32 from the first step to the last.  The gradients need the input and one state in
128 steps; the states between are made again.
"""

import torch

from . import hip
from .microscaling import _check_floating, _refuse_tangents

ACTIVATIONS = ("tanh", None)
MOST_STEPS, MOST_WIDTH = (1 << 31) - 1, 1 << 24


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, state, lengths, reverse, tanh, batch_first):
        y, last, marks = hip.recurrence(x, state, lengths, reverse, tanh, batch_first, True)
        ctx.save_for_backward(x, lengths, marks)
        ctx.options = reverse, tanh, batch_first
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        x, lengths, marks = ctx.saved_tensors
        args = (x, dy, dlast, lengths, marks, ctx.options, ctx.needs_input_grad[1])
        # create_graph: the gradients depend on x too, which a second backward must not pass over.
        dx, dstate = _Gradients.apply(*args) if torch.is_grad_enabled() else _gradients(*args)
        return dx if ctx.needs_input_grad[0] else None, dstate, None, None, None, None


def _gradients(x, dy, dlast, lengths, marks, options, with_state):
    if dy is not None and dy.stride(2) != 1:
        dy = dy.contiguous()
    if dlast is not None and not dlast.is_contiguous():
        dlast = dlast.contiguous()
    return hip.recurrence_grad(x, lengths, *options, marks, dy, dlast, with_state)


class _Gradients(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        return _gradients(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("gated_recurrence has no second derivative")


def gated_recurrence(projected, state=None, *, activation="tanh", lengths=None, reverse=False,
                     batch_first=False):
    """(states [T, B, H], last state [B, H]) of ``projected`` [T, B, 2H], which holds the update gates
    g and then the candidates v: from ``h_0 = state`` (zeros by default)
    ``h_t = u_t h_{t-1} + (1 - u_t) c_t`` with ``u = sigmoid(g)`` and ``c = tanh(v)``, or v itself with
    ``activation=None``.

    ``batch_first`` takes and gives [B, T, ...]; without a batch dimension ([T, 2H], ``state`` [H]) the
    results have none.  ``lengths`` [B] (whole numbers on the same device, taken within 0 .. T) ends each
    sequence: later steps are neither read nor passed, their states are 0 and their gradients too.
    ``reverse`` runs from the last step of each sequence to the first.  States have the input's dtype
    (float32, bfloat16 or float16); ``state`` has that or float32, and the last state is float32, so
    that a sequence taken in parts is the sequence.  A gate below -104, whose ``u`` is 0 in float32, drops a
    state of any size (an infinite one becomes NaN there, and stays infinite before).  Fewer than 2**31
    steps and sequences, H at most 2**24.  An operand with a tangent of forward mode is refused."""
    _check_floating("projected", projected)
    if activation not in ACTIVATIONS:
        raise ValueError("activation must be 'tanh' or None")
    single = projected.ndim == 2
    if projected.shape[-1] % 2 if single or projected.ndim == 3 else True:
        raise ValueError("projected must be [T, B, 2H], [B, T, 2H] or [T, 2H]")
    x = projected.unsqueeze(1) if single else projected
    batch_first = bool(batch_first) and not single
    steps, batch, width = x.shape
    if batch_first:
        steps, batch = batch, steps
    width //= 2
    if steps > MOST_STEPS or batch > MOST_STEPS or width > MOST_WIDTH:
        raise NotImplementedError(f"more than {MOST_STEPS} steps or sequences or {MOST_WIDTH} channels")
    device, start = projected.device, state
    if state is not None:
        _check_floating("state", state)
        if state.shape != ((width,) if single else (batch, width)):
            raise ValueError("state must have one value per sequence and channel")
        if state.dtype not in (torch.float32, projected.dtype):
            raise ValueError("state must be float32 or of the input's dtype")
        if state.device != device:
            raise ValueError("projected and state must use the same device")
        if single:
            start = start.unsqueeze(0)
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int64, torch.int32):
            raise TypeError("lengths must be an int64 or int32 tensor")
        if lengths.shape != (() if single else (batch,)):
            raise ValueError("lengths must have one value per sequence")
        if lengths.device != device:
            raise ValueError("projected and lengths must use the same device")
        lengths = lengths.reshape(-1).to(torch.int64).contiguous()
    _refuse_tangents("gated_recurrence", projected, state)
    hip.require_device(projected)
    if start is not None and (start.dtype != torch.float32 or not start.is_contiguous()):
        start = start.to(torch.float32).contiguous()
    if steps == 0 or batch == 0 or width == 0:
        # No step to take, or no channel: states without values and the state that came in.
        y = x[..., :width] * 1
        last = start.clone() if start is not None else \
            torch.zeros((batch, width), dtype=torch.float32, device=device)
    else:
        if x.stride(2) != 1:
            x = x.contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or start is not None and start.requires_grad):
            y, last = _Recurrence.apply(x, start, lengths, bool(reverse), activation is not None,
                                        batch_first)
        else:
            y, last, _ = hip.recurrence(x, start, lengths, reverse, activation is not None, batch_first,
                                        False)
    return (y.squeeze(1), last.squeeze(0)) if single else (y, last)


__all__ = ["gated_recurrence"]
