"""``nn.Module`` wrapper of the root-mean-square norm."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch import Tensor

from .kernel import rms_norm


class RMSNorm(nn.Module):
    """Norm over the last dimension of width ``d_model``; ``forward(x, residual)`` returns ``(y, x + residual)``."""

    def __init__(self, d_model: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d_model))
        self.eps = eps

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
        return rms_norm(x, self.weight, self.eps, residual)
