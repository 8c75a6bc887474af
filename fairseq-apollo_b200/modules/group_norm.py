"""Group norm with an activation, channels last: the norm in front of a layer that reads (B, L, D) memory.

SequenceNorm (fairseq/modules/norm_layer/sequence_norm.py:55-72) with groups takes the same statistics; here the activation is
part of the operator in both directions and the positions may have any number of axes.  weight and bias (D) are offsets as
there (effective scale weight + 1).
"""
from typing import Optional

import torch
import torch.nn as nn
from torch.nn.parameter import Parameter

from .. import ops
from ..functions import group_norm


class GroupNorm(nn.Module):
    def __init__(self, num_features: int, num_groups: int, eps: float = 1e-5, activation: Optional[str] = None) -> None:
        super().__init__()
        assert num_groups >= 1 and num_features % num_groups == 0
        ops._silu(activation)
        self.num_features = num_features
        self.num_groups = num_groups
        self.eps = eps
        self.activation = activation
        self.weight = Parameter(torch.zeros(num_features))
        self.bias = Parameter(torch.zeros(num_features))

    def forward(self, x: torch.Tensor, padding_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x (B, ..., D); padding_mask of x's shape without the channels, non-zero = padded (0 in the result)."""
        if x.size(-1) != self.num_features:
            raise ValueError("x has %d channels, not %d" % (x.size(-1), self.num_features))
        return group_norm(x, self.weight, self.bias, self.num_groups, padding_mask, self.eps, self.activation)

    def extra_repr(self) -> str:
        return 'num_features={num_features}, num_groups={num_groups}, eps={eps}, activation={activation}'.format(**self.__dict__)
