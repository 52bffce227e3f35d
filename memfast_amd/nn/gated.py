"""Recurrent layers without hidden projections, and dropout that stores no mask.

A ``GatedRecurrence`` projects a whole sequence at once, so that an analog projection (``convert_model``
replaces its nn.Linear layers) makes one read a layer and direction, where ``AnalogGRU`` makes two a step,
and leaves the gated linear recurrence of memfast_amd/recurrence.py.
"""

import torch
from torch import nn

from .. import hip
from ..recurrence import ACTIVATIONS, gated_recurrence
from ..regularization import _check_probability, dropout


# What captured dropouts count up, by device index: events from 1 on, where eager passes have 0. Graphs hold their
# addresses, so they stay for the process.
_counters = {}


class Dropout(nn.Module):
    """Dropout by ``memfast_amd.dropout``, each forward in training mode with a seed that it draws from torch's
    default CPU generator: ``torch.manual_seed`` makes the masks again, and so does a checkpointed
    layer's second forward, for which torch restores the generator.

    A captured forward keeps the seed of its capture and takes its event from a counter on the device, which the
    graph counts up: every replay has a mask of its own, and a captured backward that of its forward, also where
    checkpointing takes the forward again. The counter is made by the first forward in training mode on a
    device, so one has to run there before a capture."""

    def __init__(self, p=0.5):
        super().__init__()
        self.p = _check_probability(p)
        self._captured = {}     # by seed: the capture and its event, until an eager forward (then None)

    def __getstate__(self):     # copies and pickles have captured nothing
        return {**self.__dict__, "_captured": {}}

    def __setstate__(self, state):
        super().__setstate__({"_captured": {}, **state})

    def _event(self, x, seed):
        if torch._C._current_graph_task_id() != -1:     # within a backward: a checkpointed forward once more
            event = self._captured.get(seed, (0, 0))[1]
            if event is None:
                raise RuntimeError("a captured forward is taken again after an eager one in training mode")
            return event
        capture = hip.capture_id(x.device)
        counter = _counters.get(x.device.index)
        if not capture:
            if counter is None:
                with torch.inference_mode(False):
                    _counters[x.device.index] = torch.ones(1, dtype=torch.int64, device=x.device)
            if self._captured:
                self._captured = {s: (0, None) for s in self._captured if s != seed}
            return 0
        if counter is None:
            raise RuntimeError("a Dropout layer in training mode has to run on the device before one is captured")
        known = self._captured.get(seed)
        if known is None or known[0] != capture:
            # A sum, not a copy: kernels alone in the graph. The counter goes on before the backward reads it.
            self._captured[seed] = capture, counter + 0
            counter.add_(1)
        return self._captured[seed][1]

    def forward(self, x, residual=None):
        if not (self.training and self.p):
            return dropout(x, self.p, seed=0, residual=residual, training=self.training)
        seed = int(torch.randint(1 << 62, (), device="cpu"))
        event = self._event(x, seed) if isinstance(x, torch.Tensor) and x.is_cuda else 0
        return dropout(x, self.p, seed=seed, event=event, residual=residual)

    def extra_repr(self):
        return f"p={self.p}"


class GatedRecurrence(nn.Module):
    """Stacked gated linear recurrences with nn.GRU's arguments: every layer and direction is a projection
    to update gates and candidates and ``gated_recurrence`` of them, with ``Dropout`` between layers.

    ``projections`` holds the nn.Linear layers, one for each layer and direction; any layer with the same
    outputs may take their place (analog layers, ``MXLinear``, ``Int4Linear``)."""

    def __init__(self, input_size, hidden_size, num_layers=1, *, bias=True, batch_first=False,
                 dropout=0.0, bidirectional=False, activation="tanh", device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError("activation must be 'tanh' or None")
        if min(input_size, hidden_size, num_layers) < 1:
            raise ValueError("input_size, hidden_size and num_layers must be positive")
        self.input_size, self.hidden_size, self.num_layers = input_size, hidden_size, num_layers
        self.batch_first, self.bidirectional = bool(batch_first), bool(bidirectional)
        self.activation = activation
        self.directions = 2 if bidirectional else 1
        self.projections = nn.ModuleList(
            nn.Linear(input_size if layer == 0 else self.directions * hidden_size, 2 * hidden_size,
                      bias=bias, device=device, dtype=dtype)
            for layer in range(num_layers) for _ in range(self.directions))
        self.dropouts = nn.ModuleList(Dropout(dropout) for _ in range(num_layers - 1))

    def forward(self, x, hx=None, lengths=None):
        """(states, last states [layers * directions, B, H] in FP32) of ``x`` [T, B, input_size], or
        [B, T, input_size] with ``batch_first``, or [T, input_size]; ``hx`` as the last states, ``lengths``
        as in ``gated_recurrence``."""
        if not torch.is_tensor(x) or x.ndim not in (2, 3) or x.shape[-1] != self.input_size:
            raise ValueError("input must be a sequence with matching input_size")
        steps = x.shape[1] if x.ndim == 3 and self.batch_first else x.shape[0]
        if steps == 0:
            raise ValueError("sequence must contain at least one timestep")
        if hx is not None:
            batch = () if x.ndim == 2 else (x.shape[0] if self.batch_first else x.shape[1],)
            expected = (len(self.projections), *batch, self.hidden_size)
            if not torch.is_tensor(hx) or hx.shape != expected:
                raise ValueError("hidden state must match layers, directions and batch")
        finals = []
        for layer in range(self.num_layers):
            outputs = []
            for direction in range(self.directions):
                index = layer * self.directions + direction
                states, final = gated_recurrence(
                    self.projections[index](x), None if hx is None else hx[index],
                    activation=self.activation, lengths=lengths, reverse=bool(direction),
                    batch_first=self.batch_first)
                outputs.append(states)
                finals.append(final)
            x = outputs[0] if len(outputs) == 1 else torch.cat(outputs, -1)
            if layer + 1 < self.num_layers:
                x = self.dropouts[layer](x)
        return x, torch.stack(finals)

    def extra_repr(self):
        return (f"{self.input_size}, {self.hidden_size}, num_layers={self.num_layers}, "
                f"batch_first={self.batch_first}, bidirectional={self.bidirectional}, "
                f"activation={self.activation!r}")


__all__ = ["Dropout", "GatedRecurrence"]
