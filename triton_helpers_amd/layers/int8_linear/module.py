"""``nn.Module`` wrapper of the 8-bit linear layer."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from .kernel import int8_linear, quantize_rows


class Int8Linear(nn.Module):
    """A trained linear layer in 8 bits, for inference: ``from_linear(linear)`` quantizes its weight once (on its GPU).

    ``forward(x)`` quantizes the rows of ``x``; ``forward(q, scale)`` takes rows that are 8-bit already.  Buffers: ``weight`` int8
    ``(N, K)``, ``weight_scale`` float32 ``(N,)``, ``bias`` ``(N,)`` or ``None``.
    """

    def __init__(self, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor] = None, activation: str = "none", dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)
        self.activation = activation
        self.dtype = dtype

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Module, activation: str = "none", dtype: torch.dtype = torch.bfloat16) -> "Int8Linear":
        """``linear``: any module with ``weight`` ``(N, K)`` and ``bias``."""
        q, scale = quantize_rows(linear.weight.detach())
        return cls(q, scale, None if linear.bias is None else linear.bias.detach().clone(), activation, dtype)

    def _apply(self, fn, recurse=True):
        # a change of the module's floating type leaves the scales in float32
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != scale.dtype:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    @torch.no_grad()
    def forward(self, x: Tensor, scale: Optional[Tensor] = None) -> Tensor:
        q, s = quantize_rows(x) if scale is None else (x, scale)
        return int8_linear(q, s, self.weight, self.weight_scale, self.bias, self.activation, self.dtype)
