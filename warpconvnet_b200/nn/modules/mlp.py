"""Linear layers over the features of a geometry, with what follows them, and the feed-forward block that they make with RMS norm and
dropout (see ``nn/functional/linear.py``).  Stands for the reference's MLP layers (warpconvnet/nn/modules/mlp.py)."""
import math
from typing import Optional, Union

import torch
import torch.nn as nn
from torch import Tensor

from ...geometry.base.geometry import Geometry
from ..functional.dropout import check_probability, dropout
from ..functional.group_norm import check_activation
from ..functional.linear import linear, linear_8bit
from ..functional.rms_norm import check_eps, quantize_rows, rms_norm, rms_norm_8bit
from .base_module import BaseSpatialModule

Features = Union[Geometry, Tensor]


def features_of(input: Features) -> Tensor:
    return input.feature_tensor if isinstance(input, Geometry) else input


def with_features(input: Features, features: Tensor) -> Features:
    return input.replace(batched_features=features) if isinstance(input, Geometry) else features


def _parameters(inputs: int, outputs: int, bias: bool):
    """Weight and bias as ``nn.Linear`` begins with them."""
    bound = 1 / math.sqrt(inputs)
    return (nn.Parameter(torch.empty(outputs, inputs).uniform_(-bound, bound)), nn.Parameter(torch.empty(outputs).uniform_(-bound, bound)) if bias else None)


class Linear(BaseSpatialModule):
    """``residual + dropout(act(x W^T + b))`` of a geometry's features, or of ``[N, C]`` features; dropout in training alone."""

    def __init__(self, in_channels: int, out_channels: int, bias: bool = True, activation: Optional[str] = None, dropout: float = 0.0):
        super().__init__()
        check_activation(activation)
        check_probability(dropout)
        self.in_channels, self.out_channels, self.activation, self.dropout = in_channels, out_channels, activation, dropout
        self.weight, self.bias = _parameters(in_channels, out_channels, bias)

    def extra_repr(self):
        return f"{self.in_channels}, {self.out_channels}, bias={self.bias is not None}, activation={self.activation!r}, dropout={self.dropout}"

    def forward(self, input: Features, residual: Optional[Features] = None) -> Features:
        y = linear(features_of(input), self.weight, self.bias, self.activation, None if residual is None else features_of(residual),
                   self.dropout if self.training else 0.0)
        return with_features(input, y)


class Dropout(BaseSpatialModule):
    """Dropout of a geometry's features, or of ``[N, C]`` features, in training alone; no mask is kept."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        check_probability(p)
        self.p = p

    def extra_repr(self):
        return f"p={self.p}"

    def forward(self, input: Features, residual: Optional[Features] = None) -> Features:
        if not self.training and residual is None:
            return input
        y = dropout(features_of(input), self.p if self.training else 0.0, residual=None if residual is None else features_of(residual))
        return with_features(input, y)


class FeedForward(BaseSpatialModule):
    """``x + dropout(W2 dropout(act(W1 rms_norm(x) + b1)) + b2)`` of a geometry's features, or of ``[N, C]`` features: three kernels
    forward.  :meth:`to_8bit` gives the same for inference with 8-bit products."""

    def __init__(self, channels: int, hidden_channels: int, activation: Optional[str] = "gelu", dropout: float = 0.0, eps: float = 1e-6):
        super().__init__()
        check_activation(activation)
        check_probability(dropout)
        check_eps(eps)
        self.channels, self.hidden_channels, self.activation, self.dropout, self.eps = channels, hidden_channels, activation, dropout, eps
        self.norm_weight = nn.Parameter(torch.ones(channels))
        self.weight1, self.bias1 = _parameters(channels, hidden_channels, True)
        self.weight2, self.bias2 = _parameters(hidden_channels, channels, True)

    def extra_repr(self):
        return f"{self.channels}, {self.hidden_channels}, activation={self.activation!r}, dropout={self.dropout}, eps={self.eps}"

    def forward(self, input: Features) -> Features:
        x, p = features_of(input), self.dropout if self.training else 0.0
        hidden = linear(rms_norm(x, self.norm_weight, self.eps), self.weight1, self.bias1, self.activation, dropout_p=p)
        return with_features(input, linear(hidden, self.weight2, self.bias2, residual=x, dropout_p=p))

    def to_8bit(self) -> "FeedForward8Bit":
        return FeedForward8Bit(self)


class FeedForward8Bit(BaseSpatialModule):
    """A :class:`FeedForward` for inference: its weights in e4m3 with a scale for each output, its activations in e4m3 with a scale for
    each row, products in 8 bits.  Features are float16 or bfloat16, as are the results."""

    def __init__(self, block: FeedForward):
        super().__init__()
        self.channels, self.hidden_channels, self.activation, self.eps = block.channels, block.hidden_channels, block.activation, block.eps
        with torch.no_grad():
            for i, weight in ((1, block.weight1), (2, block.weight2)):
                q, scale = quantize_rows(weight)
                self.register_buffer(f"weight{i}", q)
                self.register_buffer(f"scale{i}", scale)
            for name in ("norm_weight", "bias1", "bias2"):
                self.register_buffer(name, getattr(block, name).detach().float().clone())

    def extra_repr(self):
        return f"{self.channels}, {self.hidden_channels}, activation={self.activation!r}, eps={self.eps}"

    @torch.no_grad()
    def forward(self, input: Features) -> Features:
        x = features_of(input)
        hidden = linear_8bit(*rms_norm_8bit(x, self.norm_weight, self.eps), self.weight1, self.scale1, self.bias1, self.activation, out_dtype=x.dtype)
        return with_features(input, linear_8bit(*quantize_rows(hidden), self.weight2, self.scale2, self.bias2, residual=x, out_dtype=x.dtype))

    def _apply(self, fn, recurse: bool = True):
        """Moves to another device; codes and scales keep their types whatever the module is brought to."""
        kept = {name: buffer for name, buffer in self._buffers.items()}
        super()._apply(fn, recurse)
        for name, buffer in kept.items():
            if self._buffers[name].dtype != buffer.dtype:
                self._buffers[name] = buffer.to(self._buffers[name].device)
        return self
