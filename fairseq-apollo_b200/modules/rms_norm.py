"""Root-mean-square norm, channels last, with the residual's addition: the norm in front of a layer on a residual stream, or, in
groups, of each head's output.

TimestepNorm and SequenceNorm (fairseq/modules/norm_layer) take statistics over time; this one is of a position alone.  weight (D) is an
offset as there (effective scale weight + 1).
"""
from typing import Optional

import torch
import torch.nn as nn
from torch.nn.parameter import Parameter

from .. import functions, ops
from ..functions import needs_grad


def rms_norm(x, weight, residual=None, num_groups=1, eps=1e-5):
    """The operator by itself: see ops.rms_norm_fwd; differentiable in x, the residual and weight."""
    fn = functions.rms_norm if needs_grad(x, weight, residual) else ops.rms_norm_fwd
    return fn(x, weight, residual, num_groups, eps)


class RMSNorm(nn.Module):
    def __init__(self, num_features: int, num_groups: int = 1, eps: float = 1e-5) -> None:
        super().__init__()
        assert num_groups >= 1 and num_features % num_groups == 0
        self.num_features = num_features
        self.num_groups = num_groups
        self.eps = eps
        self.weight = Parameter(torch.zeros(num_features))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """x (B, ..., D) -> y; with a residual of its shape (y, x + residual)."""
        if x.size(-1) != self.num_features:
            raise ValueError("x has %d channels, not %d" % (x.size(-1), self.num_features))
        return rms_norm(x, self.weight, residual, self.num_groups, self.eps)

    def extra_repr(self) -> str:
        return 'num_features={num_features}, num_groups={num_groups}, eps={eps}'.format(**self.__dict__)
