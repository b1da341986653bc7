"""The classes of a network and their loss in one layer (see ``nn/functional/linear_cross_entropy.py``)."""
import math
from typing import Union

import torch
import torch.nn as nn
from torch import Tensor

from ...geometry.base.geometry import Geometry
from ..functional.linear_cross_entropy import check_reduction, linear_cross_entropy
from .base_module import BaseSpatialModule


class LinearCrossEntropy(BaseSpatialModule):
    """A linear layer to ``num_classes`` and the cross entropy of what it gives, without the logits in memory.  Takes a geometry
    or ``[N, C]`` features and a label for each row; :meth:`logits` gives the logits themselves."""

    def __init__(self, in_channels: int, num_classes: int, bias: bool = True, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        check_reduction(reduction)
        self.in_channels, self.num_classes, self.ignore_index, self.reduction = in_channels, num_classes, ignore_index, reduction
        bound = 1 / math.sqrt(in_channels)
        self.weight = nn.Parameter(torch.empty(num_classes, in_channels).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(num_classes).uniform_(-bound, bound)) if bias else None

    def extra_repr(self):
        return f"{self.in_channels}, {self.num_classes}, bias={self.bias is not None}, ignore_index={self.ignore_index}, reduction={self.reduction!r}"

    def forward(self, input: Union[Geometry, Tensor], labels: Tensor) -> Tensor:
        x = input.feature_tensor if isinstance(input, Geometry) else input
        return linear_cross_entropy(x, self.weight, labels, self.bias, self.ignore_index, self.reduction)

    def logits(self, input: Union[Geometry, Tensor]) -> Tensor:
        x = input.feature_tensor if isinstance(input, Geometry) else input
        return nn.functional.linear(x, self.weight, self.bias)
