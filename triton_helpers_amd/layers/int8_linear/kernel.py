"""Linear layers in 8-bit integers on MI355X, for inference: a scale for every row of the input and for every output channel.

The reference has no such layer; the surface follows its siblings' style.

An 8-bit row of ``v`` is ``q = rint(v * (127 / a))`` with the scale ``s = a / 127``, ``a`` the largest magnitude of the row: it stands for
``s * q``.  A row that holds an infinity or a NaN gets the scale NaN (and zeros), so that what is made of it is NaN, too; a row of zeros, or
of magnitudes below 2^-120, the scale zero.

    y = act(scale[m] * w_scale[n] * sum_k q[m, k] * w[n, k] + bias[n])

The sums are exact (32-bit integers, at most 131071 products); scales, bias and activation are applied in float32, and the result is rounded once.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib

# A sum of more products of 8-bit values (at most 2^14 each) could leave 32 bits.
INT8_MAX_CHANNELS = 131071

_ACTIVATIONS = ("gelu", "relu", "relu2", "silu", "none")
_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_CODE = {torch.float32: _lib.NF_F32, torch.float16: _lib.NF_F16, torch.bfloat16: _lib.NF_BF16}


def _no_grad(name: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


def _validate_rows(x: Tensor) -> None:
    assert x.ndim >= 1 and x.shape[-1] >= 1, "x must have a last dimension of at least one value"
    if x.dtype not in _TYPES:
        raise NotImplementedError(f"quantize_rows takes float16 / bfloat16 / float32 rows, got {x.dtype}")
    assert x.device.type == "cuda", "All tensors must be on a GPU device"


def _validate(q: Tensor, scale: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor], activation: str, dtype: torch.dtype) -> None:
    for t, name in ((q, "q"), (w, "w")):
        assert t.dtype == torch.int8, f"{name} must be int8, got {t.dtype}"
    for t, name in ((scale, "scale"), (w_scale, "w_scale")):
        assert t.dtype == torch.float32, f"{name} must be float32, got {t.dtype}"
    assert q.ndim >= 1 and q.shape[-1] >= 1, "q must have a last dimension of at least one value"
    assert w.ndim == 2 and w.shape[0] >= 1 and w.shape[1] == q.shape[-1], f"w must be (N, {q.shape[-1]})"
    assert q.shape[-1] <= INT8_MAX_CHANNELS, f"{q.shape[-1]} input channels: at most {INT8_MAX_CHANNELS} products fit a 32-bit sum"
    assert scale.shape == q.shape[:-1], "scale must have the shape of q without its last dimension"
    assert w_scale.shape == w.shape[:1], f"w_scale must be ({w.shape[0]},)"
    assert bias is None or bias.shape == w.shape[:1], f"bias must be ({w.shape[0]},)"
    assert activation in _ACTIVATIONS, f"Invalid activation function: {activation}"
    if dtype not in _TYPES or (bias is not None and bias.dtype not in _TYPES):
        raise NotImplementedError("int8_linear gives, and takes biases in, float16 / bfloat16 / float32")
    for t in (scale, w, w_scale, bias):
        assert t is None or t.device == q.device, "All tensors must be on the same device"
    assert q.device.type == "cuda", "All tensors must be on a GPU device"


# The launches as autograd Functions, though they have no gradient: a traced function then holds the operator (the tracer would record the
# allocation of the results and nothing of the launch), and tangents and transforms are refused.
# A call of the traced function comes to ``forward`` alone, with whatever tensors it is given.
class _quantize_rows(Function):
    @staticmethod
    def forward(ctx, x: Tensor) -> Tuple[Tensor, Tensor]:
        _validate_rows(x)
        return _lib.native().quantize_rows_launch(x)


class _int8_linear(Function):
    @staticmethod
    def forward(ctx, q: Tensor, scale: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor], activation: str, dtype: torch.dtype) -> Tensor:
        _validate(q, scale, w, w_scale, bias, activation, dtype)
        return _lib.native().int8_linear_launch(q, scale, w, w_scale, bias, _lib.NF_ACT[activation], _CODE[dtype])


def quantize_rows(x: Tensor) -> Tuple[Tensor, Tensor]:
    r"""The 8-bit form of the rows of ``x``, also that of a weight :math:`(N, K)`; for inference.

    Shapes:
        - x: :math:`(..., K)`, float32 / float16 / bfloat16, any row strides
        - Output: ``(q, scale)``, int8 :math:`(..., K)` and float32 :math:`(...)`
    """
    out = _lib.native().quantize_rows(x)
    if out is not None:
        return out
    _validate_rows(x)
    _no_grad("quantize_rows", x)
    return _quantize_rows.apply(x)


def int8_linear(q: Tensor, scale: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, activation: str = "none",
                dtype: torch.dtype = torch.bfloat16) -> Tensor:
    r"""Product of 8-bit rows with 8-bit weight rows; for inference.

    Shapes:
        - q: int8 :math:`(..., K)`, scale: float32 :math:`(...)` (what :func:`quantize_rows` and ``rms_norm_int8`` return)
        - w: int8 :math:`(N, K)`, w_scale: float32 :math:`(N,)`; bias: :math:`(N,)` or ``None``
        - Output: :math:`(..., N)` of type ``dtype``

    ``activation`` is one of ``"none"``, ``"relu"``, ``"relu2"``, ``"silu"``, ``"gelu"``.  Rows on 16-byte boundaries whose length is a multiple of 16
    are the fast case beyond 64 rows; others are copied to such boundaries first.
    """
    code = _CODE.get(dtype, -1)
    y = _lib.native().int8_linear(q, scale, w, w_scale, bias, activation, code)
    if y is not None:
        return y
    _validate(q, scale, w, w_scale, bias, activation, dtype)
    _no_grad("int8_linear", scale, w_scale, bias)
    return _int8_linear.apply(q, scale, w, w_scale, bias, activation, dtype)
