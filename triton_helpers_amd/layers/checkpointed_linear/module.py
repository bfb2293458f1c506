"""``nn.Module`` wrapper of the linear layer with 8-bit checkpoints."""
from __future__ import annotations

import torch.nn as nn
from torch import Tensor

from .kernel import checkpointed_linear


class CheckpointedLinear(nn.Linear):
    """``nn.Linear`` (its parameters and initialisation) behind ``activation``, with its input kept in 8 bits."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device, dtype)
        self.activation = activation

    def forward(self, x: Tensor) -> Tensor:
        return checkpointed_linear(x, self.weight, self.bias, self.activation)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
