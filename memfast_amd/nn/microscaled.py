"""Linear layers in 4-bit microscaled floating point.

The digital counterpart of the analog layers: what a model's layers that stay digital, or the
teacher of a distilled student, run on (memfast_amd/microscaling.py).
"""

import torch
from torch import nn

from ..microscaling import MXTensor, mx_linear, mx_quantize
from .training import _master


class MXLinear(nn.Module):
    """``nn.Linear`` on 4-bit operands.

    By default the weight is quantized once, on its own device, and held in its codes and
    scales (buffers; 17 bits for 4 values); the input still gets gradients. ``trainable=True``
    keeps Parameters of its own, which every forward quantizes and whose gradients pass straight
    through."""

    def __init__(self, source, *, trainable=False):
        super().__init__()
        if not isinstance(source, nn.Linear):
            raise TypeError("source must be torch.nn.Linear")
        self.in_features, self.out_features = source.in_features, source.out_features
        self.trainable = bool(trainable)
        if self.trainable:
            self.weight = _master(source.weight, source.weight.device)
            self.register_parameter("bias", _master(source.bias, source.weight.device))
        else:
            held = mx_quantize(source.weight)
            self.register_buffer("codes", held.codes)
            self.register_buffer("scales", held.scales)
            self.register_buffer("bias", None if source.bias is None
                                 else source.bias.detach().clone())
        self.train(source.training)

    def forward(self, x):
        weight = self.weight if self.trainable else MXTensor(
            self.codes, self.scales, (self.out_features, self.in_features))
        # Operands keep their dtypes under autocast, as the analog layers' do.
        with torch.autocast(device_type=x.device.type, enabled=False):
            return mx_linear(x, weight, self.bias)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, trainable={self.trainable}")


__all__ = ["MXLinear"]
