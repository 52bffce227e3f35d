"""Linear layers whose weight is held in 4-bit whole numbers (memfast_amd/int4.py)."""

from torch import nn

from ..int4 import Int4Tensor, int4_linear, int4_quantize


class Int4Linear(nn.Module):
    """``nn.Linear`` for serving: the weight is quantized once, on its own device, and held in codes and
    scales (buffers; 4.5 bits a value with groups of 32 and 16-bit scales), the input is not quantized.
    ``from_tensor`` takes an Int4Tensor that is held already, imported codes among them.  It has no
    gradient: call it where none are recorded."""

    def __init__(self, source, *, group=32, scale_dtype=None):
        super().__init__()
        if not isinstance(source, nn.Linear):
            raise TypeError("source must be torch.nn.Linear")
        self._hold(int4_quantize(source.weight, group=group, scale_dtype=scale_dtype), source.bias)
        self.train(source.training)

    @classmethod
    def from_tensor(cls, weight, bias=None):
        if not isinstance(weight, Int4Tensor):
            raise TypeError("weight must be an Int4Tensor")
        layer = cls.__new__(cls)
        nn.Module.__init__(layer)
        layer._hold(weight, bias)
        return layer

    def _hold(self, weight, bias):
        self.out_features, self.in_features = weight.shape
        self.group = weight.group
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    def forward(self, x):
        # No operation of it is subject to autocast: operands keep their dtypes, as the analog layers' do.
        return int4_linear(x, Int4Tensor(self.codes, self.scales, (self.out_features, self.in_features),
                                         group=self.group, zeros=self.zeros), self.bias)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, group={self.group}")


__all__ = ["Int4Linear"]
