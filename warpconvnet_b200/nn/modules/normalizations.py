"""Normalisations over geometry features: BatchNorm (warpconvnet/nn/modules/normalizations.py:49-63), group norm per scene and RMS norm."""
from typing import Optional

import torch
import torch.nn as nn

from ...geometry.base.geometry import Geometry
from ..functional.group_norm import check_activation, segmented_group_norm
from ..functional.rms_norm import check_eps, rms_norm
from ..functional.transforms import apply_feature_transform
from .base_module import BaseSpatialModule


class BatchNorm(BaseSpatialModule):
    def __init__(self, num_features: int, eps: float = 1e-5, momentum: float = 0.1):
        super().__init__()
        self.norm = nn.BatchNorm1d(num_features, eps=eps, momentum=momentum)

    def __repr__(self):
        return f"{self.__class__.__name__}({self.norm})"

    def forward(self, input: Geometry):
        return apply_feature_transform(input, self.norm)


class SegmentedGroupNorm(BaseSpatialModule):
    """Group norm with statistics per scene: over all rows of a scene and the channels of a group, then the activation
    (None, ``"relu"``, ``"silu"`` or ``"gelu"``).  What a scene becomes does not depend on the others of its batch, in training
    and evaluation alike, but for the last bits: its sums are divided by the size of the whole batch.  (The reference's ``GroupNorm`` is ``nn.GroupNorm`` of ``[N, C]`` rows: statistics per row.)"""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True, activation: Optional[str] = None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"num_channels ({num_channels}) must be divisible by num_groups ({num_groups})")
        check_activation(activation)
        self.num_groups, self.num_channels, self.eps, self.activation = num_groups, num_channels, eps, activation
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def extra_repr(self):
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, activation={self.activation!r}"

    def forward(self, input: Geometry):
        return apply_feature_transform(input, lambda x: segmented_group_norm(x, input.offsets, self.num_groups, self.weight, self.bias,
                                                                              self.eps, self.activation))


class RMSNorm(BaseSpatialModule):
    """Root-mean-square norm of each row of a geometry's features.  With a second geometry of the same coordinates, the residual, it
    gives ``(norm, sum)``: the norm of the sum, and the sum."""

    def __init__(self, num_channels: int, eps: float = 1e-6, affine: bool = True):
        super().__init__()
        check_eps(eps)
        self.num_channels, self.eps = num_channels, eps
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None

    def extra_repr(self):
        return f"{self.num_channels}, eps={self.eps}, affine={self.weight is not None}"

    def forward(self, input: Geometry, residual: Optional[Geometry] = None):
        if residual is None:
            return apply_feature_transform(input, lambda x: rms_norm(x, self.weight, self.eps))
        y, h = rms_norm(input.feature_tensor, self.weight, self.eps, residual.feature_tensor)
        return input.replace(batched_features=y), input.replace(batched_features=h)
