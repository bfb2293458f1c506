"""A linear layer behind an activation that keeps its input in 8 bits for the backward, on MI355X.

The reference has no such layer; the surface follows its siblings' style.

    y = act(x) W^T + b

What autograd keeps of the input is its 8-bit rows (``q = rint(x * (127 / a))`` and one float32 scale ``a / 127`` a row, ``a`` the largest
magnitude of the row): half of a 16-bit tensor, and the activation's output, which a linear layer would keep for its weight's gradient, is
not kept at all.  The forward is computed from ``x`` as it is.  The backward works on ``x^ = scale * q``:

    dx = (dy W) * act'(x^);   dW = dy^T act(x^);   db = sum over rows of dy

so ``dx`` is exact without an activation, and the others carry the rounding to 8 bits: half a step, ``a / 254``, for each value of a row, independent of
the value.  Gates that open at zero (``"relu"``, ``"relu2"``) see a value below half a step as zero, that is closed.  A row that holds
an infinity or a NaN is NaN in ``x^``.

``act(x)`` and ``act(x^)`` enter the products rounded to the tensors' 16-bit type, whose range they have to keep: ``"relu2"`` leaves that of float16
from ``x = 256`` on, and the infinity goes on into the row's ``y``, into ``dW``'s column and, times a zero of ``dy``, into it as NaN.  bfloat16 has
float32's range.

float16 and bfloat16; under autocast float32 tensors are cast to its type, and the weight's gradient comes back as float32.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib

_ACTIVATIONS = ("gelu", "relu", "relu2", "silu", "none")
_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_CODE = {torch.float32: _lib.NF_F32, torch.float16: _lib.NF_F16, torch.bfloat16: _lib.NF_BF16}


def _validate(x: Tensor, w: Tensor, b: Optional[Tensor], activation: str) -> None:
    assert x.ndim >= 1 and x.shape[-1] >= 1, "x must have a last dimension of at least one value"
    assert w.ndim == 2 and w.shape[0] >= 1 and w.shape[1] == x.shape[-1], f"w must be (N, {x.shape[-1]})"
    assert b is None or b.shape == w.shape[:1], f"b must be ({w.shape[0]},)"
    assert activation in _ACTIVATIONS, f"Invalid activation function: {activation}"
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        if any(t.dtype not in _TYPES for t in (x, w)) or dtype not in _TYPES[:2]:
            raise NotImplementedError(f"checkpointed_linear runs under autocast to float16 / bfloat16, got {x.dtype}, {w.dtype} and {dtype}")
    elif x.dtype not in _TYPES[:2] or w.dtype != x.dtype:
        raise NotImplementedError(
            f"checkpointed_linear runs on float16 / bfloat16 storage of one type, got {x.dtype} and {w.dtype}; cast the tensors or use autocast")
    if b is not None and b.dtype not in _TYPES:
        raise NotImplementedError(f"the bias is float16 / bfloat16 / float32, got {b.dtype}")
    for t in (w, b):
        assert t is None or t.device == x.device, "All tensors must be on the same device"
    assert x.device.type == "cuda", "All tensors must be on a GPU device"


class _checkpointed_linear(Function):
    @staticmethod
    def forward(ctx, x: Tensor, w: Tensor, b: Optional[Tensor] = None, activation: str = "none") -> Tensor:
        _validate(x, w, b, activation)
        ctx.float_dw = w.dtype == torch.float32
        ctx.x_dtype = x.dtype
        ctx.b_code = _CODE[torch.float32 if b is None else b.dtype]
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            x, w = x.to(dtype), w.to(dtype)
        y, q, scale = _lib.native().checkpointed_linear_launch_forward(x, w, b, _lib.NF_ACT[activation])
        ctx.save_for_backward(q, scale, w)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, dy: Tensor):
        need_dx, need_dw, need_db = (*ctx.needs_input_grad, False)[:3]  # (the bias may have been left out)
        dx, dw, db = _lib.native().checkpointed_linear_launch_backward(
            *ctx.saved_tensors, _lib.NF_ACT[ctx.activation], dy, need_dx, need_dw, need_db, ctx.float_dw, ctx.b_code)
        return None if dx is None else dx.to(ctx.x_dtype), dw, db, None


def checkpointed_linear(x: Tensor, w: Tensor, b: Optional[Tensor] = None, activation: str = "none") -> Tensor:
    r"""``act(x) @ w.T + b`` with the input kept in 8 bits for the backward; differentiable once in all tensors.

    Shapes:
        - x: :math:`(..., K)`, any row strides; w: :math:`(N, K)`; b: :math:`(N,)` or ``None``
        - Output: :math:`(..., N)` of the type of ``x`` (of autocast's type under autocast)

    ``activation`` is one of ``"none"``, ``"relu"``, ``"relu2"``, ``"silu"``, ``"gelu"`` and is applied to the INPUT.
    """
    y = _lib.native().checkpointed_linear(x, w, b, activation)
    if y is not None:
        return y
    # a mode, a subclass, or arguments to be refused
    _lib.native().refuse_eager_graphs(x, w, b)
    return _checkpointed_linear.apply(x, w, b, activation)
