"""Root-mean-square norm of rows on MI355X, with a residual's addition in front and an 8-bit form behind.

The reference has no such layer; the surface follows its siblings' style.

    h = x + residual;   y = h * (mean(h^2) + eps)^-1/2 * weight;   new residual = h

Sums and the statistics are float32 whatever the types.  ``x`` is float32, float16 or bfloat16; ``residual`` is of the same type or
float32 (a residual stream kept wider than the layers), ``weight`` of any of the three (autocast leaves all of them as they are).  The norm is
taken of the unrounded ``h``; the backward works on the new residual as it was rounded and kept.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib

_TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _validate(x: Tensor, weight: Optional[Tensor], eps: float, residual: Optional[Tensor]) -> None:
    assert x.ndim >= 1 and x.shape[-1] >= 1, "x must have a last dimension of at least one value"
    for t, name in ((x, "x"), (weight, "weight"), (residual, "residual")):
        if t is not None and t.dtype not in _TYPES:
            raise NotImplementedError(f"rms_norm runs on float16 / bfloat16 / float32 storage, got {name} of {t.dtype}")
    assert weight is None or weight.shape == x.shape[-1:], f"weight must be ({x.shape[-1]},)"
    if residual is not None:
        assert residual.shape == x.shape, "residual must have the shape of x"
        assert residual.dtype in (x.dtype, torch.float32), f"residual must be {x.dtype} or float32, got {residual.dtype}"
    assert eps >= 0, "eps must be >= 0"
    for t in (weight, residual):
        assert t is None or t.device == x.device, "All tensors must be on the same device"
    assert x.device.type == "cuda", "All tensors must be on a GPU device"


class _rms_norm(Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], eps: float = 1e-6, residual: Optional[Tensor] = None):
        _validate(x, weight, eps, residual)
        y, _, stream, rstd = _lib.native().rms_norm_launch_forward(x, weight, float(eps), residual, False)
        ctx.save_for_backward(x if residual is None else stream, rstd, weight)
        ctx.like = x.new_empty(0)  # its type
        ctx.residual = residual is not None
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, stream)

    @staticmethod
    def backward(ctx, dy: Optional[Tensor], d_residual: Optional[Tensor] = None):
        h, rstd, weight = ctx.saved_tensors
        need_x, need_w, _, need_r = (*ctx.needs_input_grad, False, False)[:4]  # (eps and the residual may have been left out)
        dx, dw, dr = _lib.native().rms_norm_launch_backward(h, rstd, weight, ctx.like, dy, d_residual, ctx.residual, need_x or need_r, need_w)
        return dx, dw, None, dr


class _rms_norm_int8(Function):
    """The launch as a Function, though it has no gradient: a traced function then holds the operator (the tracer would record the allocation of the
    results and nothing of the launch), and tangents and transforms are refused.  A call of the traced function comes to ``forward`` alone, with
    whatever tensors it is given."""

    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], eps: float, residual: Optional[Tensor]) -> Tuple[Tensor, ...]:
        _validate(x, weight, eps, residual)
        q, scale, stream, _ = _lib.native().rms_norm_launch_forward(x, weight, float(eps), residual, True)
        return (q, scale) if residual is None else (q, scale, stream)


def rms_norm(x: Tensor, weight: Optional[Tensor], eps: float = 1e-6, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    r"""Norm of the rows of ``x`` (of ``x + residual``); differentiable once in all tensors.

    Shapes:
        - x, residual: :math:`(..., K)`, any row strides; weight: :math:`(K,)` or ``None`` (ones)
        - Output: ``y`` of the shape and type of ``x``; with a residual ``(y, new residual)``, the latter of the residual's type
    """
    y = _lib.native().rms_norm(x, weight, eps, residual)
    if y is not None:
        return y
    # a mode, a subclass, or arguments to be refused
    _lib.native().refuse_eager_graphs(x, weight, residual)
    return _rms_norm.apply(x, weight, eps, residual)


def rms_norm_int8(x: Tensor, weight: Optional[Tensor], eps: float = 1e-6, residual: Optional[Tensor] = None) -> Tuple[Tensor, ...]:
    r"""The norm as 8-bit rows, what :func:`~triton_helpers_amd.layers.int8_linear.int8_linear` takes; for inference.

    ``q = rint(v * (127 / a))`` and ``scale = a / 127`` with ``a`` the largest magnitude of the normed row ``v``: the norm is rounded once, to
    8 bits.  A row that holds an infinity or a NaN gets the scale NaN and zeros.

    Shapes:
        - x, residual: :math:`(..., K)`; weight: :math:`(K,)` or ``None``
        - Output: ``(q, scale)``, int8 :math:`(..., K)` and float32 :math:`(...)`; with a residual ``(q, scale, new residual)``
    """
    out = _lib.native().rms_norm_int8(x, weight, eps, residual)
    if out is not None:
        return out
    _validate(x, weight, eps, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_int8 has no gradient: call it under torch.no_grad(), or rms_norm where one is needed")
    return _rms_norm_int8.apply(x, weight, eps, residual)
