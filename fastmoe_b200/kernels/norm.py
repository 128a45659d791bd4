"""Root-mean-square norm of the residual stream, with its gradient and with an 8-bit output.

  rms_norm(x, w)               y = x / sqrt(mean(x^2) + eps) * w
  add_rms_norm(x, residual, w) s = x + residual (rounded to the rows' type: what the stream holds),
                               (rms_norm(s, w), s), one pass over the rows
  rms_norm_int8(x, w, ...)     the normed rows in 8 bits with a scale per row, for the products of
                               `kernels/int8.py`; for inference

The norm of a pre-norm block (`models/tiny_model.py`, `norm="rms"`); the reference's blocks
normalise with LayerNorm (src/fastmoe/models/tiny_model.py:424-463). Rows are the last dimension,
in float32, bfloat16 or float16; the weight is float32 or of the rows' type. Statistics, products
and gradients are computed in 32 bits or more and rounded once. There is a gradient, no second derivative
and no forward mode: both are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from . import ops
from .int8 import Int8Rows, _rows, empty_rows
from .ops import _DTYPES, _require_cuda

__all__ = ["rms_norm", "add_rms_norm", "rms_norm_int8", "NormInt8"]


class NormInt8(NamedTuple):
    rows: Int8Rows  # the normed rows in 8 bits
    stream: torch.Tensor | None  # x + residual, None without a residual
    y: torch.Tensor | None  # the normed rows in x's type, when asked for


def _check(x, weight, residual, eps):
    _require_cuda(x, "x")
    _require_cuda(weight, "weight")
    dtype, shape = x.dtype, x.shape
    if len(shape) < 1 or dtype not in _DTYPES:
        raise ValueError(f"x must be float32/bfloat16/float16 rows, got {tuple(shape)} {dtype}")
    D = shape[-1]
    if D == 0:
        raise ValueError("rows of width 0 have no norm")
    dev = x.get_device()
    if weight.shape != (D,) or weight.dtype not in (dtype, torch.float32) or weight.get_device() != dev:
        raise ValueError(
            f"weight must be a [{D}] vector of {dtype} or float32 on {x.device}, got {tuple(weight.shape)} "
            f"{weight.dtype} on {weight.device}"
        )
    if residual is not None and (
        residual.shape != shape or residual.dtype != dtype or residual.get_device() != dev
    ):
        raise ValueError(
            f"residual must match x ({tuple(shape)}, {dtype}, {x.device}), got {tuple(residual.shape)}, "
            f"{residual.dtype}, {residual.device}"
        )
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    ops._refuse_tangents("the RMS norm", x, weight, residual)


def _empty(x):
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)  # the first is the faster call


def _forward(x, residual, weight, eps, want_y, want_rstd, want_q):
    """One launch over the rows of x; returns (y, stream, rstd, Int8Rows), y and stream in x's shape."""
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    T, D = x2.shape
    y = _empty(x) if want_y else None
    stream = _empty(x) if r2 is not None else None
    rstd = x2.new_empty((T,), dtype=torch.float32) if want_rstd else None
    rows = empty_rows(x2, T, D) if want_q else None
    ops._launch(
        x2.get_device(), "fmoe_rms_norm", 1, x2.data_ptr(), x2.stride(0), None if r2 is None else r2.data_ptr(),
        0 if r2 is None else r2.stride(0), weight.data_ptr(), _DTYPES[weight.dtype],
        None if y is None else y.data_ptr(), None if stream is None else stream.data_ptr(),
        None if rstd is None else rstd.data_ptr(), None if rows is None else rows.q.data_ptr(),
        0 if rows is None else rows.q.stride(0), None if rows is None else rows.scale.data_ptr(), T, D, eps,
        _DTYPES[x2.dtype],
    )  # fmt: skip
    return y, stream, rstd, rows


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        weight = weight.contiguous()
        y, stream, rstd, _ = _forward(x, residual, weight, eps, True, True, False)
        ctx.save_for_backward(x if stream is None else stream, rstd, weight)
        return y if stream is None else (y, stream)

    @staticmethod
    def backward(ctx, dy, dstream=None):
        if dy is None:  # the normed rows were not used: the stream's gradient passes through
            return dstream, dstream if ctx.needs_input_grad[1] else None, None, None
        stream, rstd, weight = ctx.saved_tensors
        s = _rows(stream)
        T, D = s.shape
        dtype = s.dtype
        dy2 = _rows(dy if dy.dtype == dtype else dy.to(dtype))
        ds2 = None
        if dstream is not None:
            ds2 = _rows(dstream if dstream.dtype == dtype else dstream.to(dtype))
        dx = _empty(stream)
        dw = scratch = None
        nbytes = 0
        if ctx.needs_input_grad[2]:
            dw = torch.empty_like(weight)
            nbytes = _lib.lib().fmoe_rms_norm_bwd_bytes(T, D)
            scratch = s.new_empty((nbytes,), dtype=torch.uint8)
        ops._launch(
            s.get_device(), "fmoe_rms_norm_bwd", 1 if dw is None else 2, dy2.data_ptr(), dy2.stride(0),
            None if ds2 is None else ds2.data_ptr(), 0 if ds2 is None else ds2.stride(0), s.data_ptr(), s.stride(0),
            rstd.data_ptr(), weight.data_ptr(), _DTYPES[weight.dtype], dx.data_ptr(),
            None if dw is None else dw.data_ptr(), None if scratch is None else scratch.data_ptr(), nbytes, T, D,
            _DTYPES[dtype],
        )  # fmt: skip
        if torch.is_grad_enabled():  # create_graph
            dx = ops._NoSecondDerivative.apply(dx, "the RMS norm", stream, weight, dy)
            if dw is not None:
                dw = ops._NoSecondDerivative.apply(dw, "the RMS norm", stream, weight, dy)
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """x / sqrt(mean(x^2 over the last dimension) + eps) * weight, in x's type. Differentiable in x
    and weight."""
    _check(x, weight, None, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _RmsNorm.apply(x, None, weight, eps)
    return _forward(x, None, weight.contiguous(), eps, True, False, False)[0]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6):
    """(rms_norm(stream, weight), stream) with stream = x + residual, rounded to x's type before the
    norm is taken: the norm is that of the stream which the next block reads. Differentiable in x,
    residual and weight."""
    if residual is None:
        raise ValueError("add_rms_norm needs a residual (rms_norm goes without)")
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad):
        return _RmsNorm.apply(x, residual, weight, eps)
    return _forward(x, residual, weight.contiguous(), eps, True, False, False)[:2]


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                  with_y: bool = False) -> NormInt8:  # fmt: skip
    """The normed rows in 8 bits: `rows` ([T, D] int8 and a float32 scale per row, T = all leading
    dimensions), quantised from the fp32 values; `stream` = x + residual when a residual is given; `y`,
    the normed rows in x's type, with `with_y` (a router reads them beside the 8-bit experts). The
    8-bit rows carry no gradient: calling this where one would be needed raises."""
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and (
        x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)
    ):
        raise ValueError("rms_norm_int8 has no gradient: call it under torch.no_grad(), or use rms_norm / add_rms_norm")
    y, stream, _, rows = _forward(x, residual, weight.contiguous(), eps, with_y, False, True)
    return NormInt8(rows, stream, y)
