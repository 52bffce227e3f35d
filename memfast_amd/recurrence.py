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
    that a sequence taken in parts is the sequence.  Fewer than 2**31 steps and sequences, H at
    most 2**24.  An operand with a tangent of forward mode is refused."""
    _check_floating("projected", projected)
    if activation not in ACTIVATIONS:
        raise ValueError("activation must be 'tanh' or None")
    if projected.ndim not in (2, 3) or projected.shape[-1] % 2:
        raise ValueError("projected must be [T, B, 2H], [B, T, 2H] or [T, 2H]")
    single = projected.ndim == 2
    x = projected.unsqueeze(1) if single else projected
    batch_first = bool(batch_first) and not single
    t, b = (1, 0) if batch_first else (0, 1)
    steps, batch, width = x.shape[t], x.shape[b], x.shape[2] // 2
    if steps > MOST_STEPS or batch > MOST_STEPS or width > MOST_WIDTH:
        raise NotImplementedError(f"more than {MOST_STEPS} steps or sequences or {MOST_WIDTH} channels")
    if state is not None:
        _check_floating("state", state)
        if state.shape != ((width,) if single else (batch, width)):
            raise ValueError("state must have one value per sequence and channel")
        if state.dtype not in (torch.float32, projected.dtype):
            raise ValueError("state must be float32 or of the input's dtype")
        if state.device != projected.device:
            raise ValueError("projected and state must use the same device")
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int64, torch.int32):
            raise TypeError("lengths must be an int64 or int32 tensor")
        if lengths.shape != (() if single else (batch,)):
            raise ValueError("lengths must have one value per sequence")
        if lengths.device != projected.device:
            raise ValueError("projected and lengths must use the same device")
    _refuse_tangents("gated_recurrence", projected, state)
    hip.require_device(projected)
    start = None if state is None else (state.unsqueeze(0) if single else state).to(torch.float32)
    if x.numel() == 0:
        # No step to take, or no channel: states without values and the state that came in.
        y = x[..., :width] * 1
        last = start.clone() if start is not None else \
            torch.zeros((batch, width), dtype=torch.float32, device=x.device)
    else:
        if x.stride(2) != 1:
            x = x.contiguous()
        if start is not None and not start.is_contiguous():
            start = start.contiguous()
        if lengths is not None:
            lengths = lengths.reshape(-1).to(torch.int64).contiguous()
        reverse, tanh = bool(reverse), activation == "tanh"
        if torch.is_grad_enabled() and (x.requires_grad or start is not None and start.requires_grad):
            y, last = _Recurrence.apply(x, start, lengths, reverse, tanh, batch_first)
        else:
            y, last, _ = hip.recurrence(x, start, lengths, reverse, tanh, batch_first, False)
    return (y.squeeze(1), last.squeeze(0)) if single else (y, last)


__all__ = ["gated_recurrence"]
