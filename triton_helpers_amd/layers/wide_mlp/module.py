"""A residual MLP of any width: what the fused MLP (up to 64 wide) and the reversible MLP (up to 128) leave open.

    stream = residual + x;   out = W2 act(W1 norm(stream) + b1) + b2

Both modules return ``(out, stream)``: the next block adds the two in its norm, and the last one's caller adds them.  ``WideMLP`` trains, with
the inputs of both linear layers kept in 8 bits; ``Int8WideMLP`` is the trained block with weights and rows in 8 bits, for inference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from ..checkpointed_linear import CheckpointedLinear
from ..int8_linear import Int8Linear
from ..rms_norm import RMSNorm, rms_norm_int8


class WideMLP(nn.Module):
    """``forward(x, residual=None)``: ``(out, stream)``.  float16 or bfloat16 parameters and rows, or float32 parameters under autocast; the
    residual is of the rows' type or float32."""

    def __init__(self, d_model: int, d_hidden: int, activation: str = "gelu", bias: bool = True, eps: float = 1e-6):
        super().__init__()
        self.norm = RMSNorm(d_model, eps)
        self.up = CheckpointedLinear(d_model, d_hidden, bias)
        self.down = CheckpointedLinear(d_hidden, d_model, bias, activation)

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        y, stream = (self.norm(x), x) if residual is None else self.norm(x, residual)
        return self.down(self.up(y)), stream

    def to_int8(self, dtype: Optional[torch.dtype] = None) -> "Int8WideMLP":
        """This block for inference, its weights rounded to 8 bits (on their GPU); results in ``dtype``, by default in the block's own type (in
        bfloat16 where its parameters are float32), so that the next block takes them beside a residual of that type."""
        if dtype is None:
            dtype = torch.bfloat16 if self.up.weight.dtype == torch.float32 else self.up.weight.dtype
        return Int8WideMLP(self.norm.weight.detach().clone(), Int8Linear.from_linear(self.up, self.down.activation, dtype),
                           Int8Linear.from_linear(self.down, "none", dtype), self.norm.eps)


class Int8WideMLP(nn.Module):
    """``forward(x, residual=None)``: ``(out, stream)`` of a :class:`WideMLP` in 8 bits."""

    def __init__(self, norm_weight: Tensor, up: Int8Linear, down: Int8Linear, eps: float = 1e-6):
        super().__init__()
        self.register_buffer("norm_weight", norm_weight)
        self.up, self.down, self.eps = up, down, eps

    @torch.no_grad()
    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        q, scale, *stream = rms_norm_int8(x, self.norm_weight, self.eps, residual)
        return self.down(self.up(q, scale)), stream[0] if stream else x
