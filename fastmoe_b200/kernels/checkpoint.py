"""Activations kept in 8 bits between the forward and the backward pass.

  pack_activation(x)      int8 values and one float32 scale per group of 128 columns of a row
  unpack_activation(p)    back to the rows' type
  packed_swiglu_backward  the SwiGLU derivative straight from packed gate/up pre-activations, with
  packed_gelu_backward    the hidden rows recomputed on the way (the GELU form likewise)

What a training forward of the expert FFN keeps (`experts.grouped_swiglu_ffn(..., packed=True)`):
1.03 bytes per value of the rows and the pre-activations, nothing for the hidden rows. The forward
result is the unpacked one's; the gradients are taken at the values that the 8 bits stand for. A
value is off by at most its group's largest magnitude / 254. A group that holds NaN or infinity
unpacks as NaN.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _lib
from . import ops
from .int8 import _padded, _rows
from .ops import _DTYPES, _require_cuda

__all__ = ["PackedActivation", "pack_activation", "unpack_activation", "packed_swiglu_backward", "packed_gelu_backward"]

GROUP = 128


class PackedActivation(NamedTuple):
    q: torch.Tensor  # int8 [T, D], rows at 16-byte steps
    scale: torch.Tensor  # float32 [T, ceil(D / 128)]
    shape: torch.Size  # of the packed tensor
    dtype: torch.dtype


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """x (float32, bfloat16 or float16, any leading dimensions) in 8 bits. No gradient flows through the packed
    values: a leaf is read as it is, a tensor out of a graph is refused (pack `x.detach()`)."""
    _require_cuda(x, "x")
    if x.dim() < 1 or x.dtype not in _DTYPES or x.shape[-1] == 0:
        raise ValueError(f"x must be float32/bfloat16/float16 rows, got {tuple(x.shape)} {x.dtype}")
    if x.requires_grad and not x.is_leaf and torch.is_grad_enabled():
        raise ValueError("pack_activation has no gradient: call it under torch.no_grad() or on detached tensors")
    ops._refuse_tangents("pack_activation", x)
    x2 = _rows(x.detach())
    T, D = x2.shape
    Dp = _padded(D)
    q = x2.new_empty((T, Dp), dtype=torch.int8)
    scale = x2.new_empty((T, (D + GROUP - 1) // GROUP), dtype=torch.float32)
    ops._launch(x.get_device(), "fmoe_pack_activation", 1, x2.data_ptr(), x2.stride(0), q.data_ptr(), Dp,
                scale.data_ptr(), T, D, _DTYPES[x.dtype])  # fmt: skip
    return PackedActivation(q if Dp == D else q[:, :D], scale, x.shape, x.dtype)


def _check_packed(p: PackedActivation):
    T, D = p.q.shape
    _require_cuda(p.q, "packed activation")
    if p.q.dtype != torch.int8 or p.q.stride() != (_padded(D), 1) or p.q.data_ptr() % 16:
        raise ValueError("a packed activation's values must be laid out as pack_activation returns them")
    if p.scale.dtype != torch.float32 or p.scale.shape != (T, (D + GROUP - 1) // GROUP) or not p.scale.is_contiguous():
        raise ValueError("a packed activation's scales must be laid out as pack_activation returns them")
    if p.scale.device != p.q.device or p.dtype not in _DTYPES:
        raise ValueError("a packed activation's parts must live on one device and stand for a supported type")
    if len(p.shape) < 1 or p.shape[-1] != D or math.prod(p.shape[:-1]) != T:
        raise ValueError(f"a packed activation of shape {tuple(p.shape)} does not have [{T}, {D}] values")
    return T, D


def unpack_activation(p: PackedActivation) -> torch.Tensor:
    """The values that `p` stands for, in the packed tensor's shape and type."""
    T, D = _check_packed(p)
    if p.scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("unpack_activation has no gradient: call it under torch.no_grad() or on detached scales")
    ops._refuse_tangents("unpack_activation", p.scale)
    out = p.q.new_empty((T, D), dtype=p.dtype)
    ops._launch(p.q.get_device(), "fmoe_unpack_activation", 1, p.q.data_ptr(), p.q.stride(0), p.scale.data_ptr(),
                out.data_ptr(), T, D, _DTYPES[p.dtype])  # fmt: skip
    return out if len(p.shape) == 2 else out.view(p.shape)


def _backward(p, grad, act):
    T, D = _check_packed(p)
    if act == _lib.ACT_SWIGLU and D % 2:
        raise ValueError(f"SwiGLU pre-activations are [gate | up]: an even width is needed, got {D}")
    cols = D // 2 if act == _lib.ACT_SWIGLU else D
    want = (*p.shape[:-1], cols)
    if grad.shape != want or grad.dtype != p.dtype or grad.device != p.q.device:
        raise ValueError(f"grad must be {want} {p.dtype} on {p.q.device}, got {tuple(grad.shape)} {grad.dtype} "
                         f"on {grad.device}")  # fmt: skip
    if (grad.requires_grad or p.scale.requires_grad) and torch.is_grad_enabled():
        raise ValueError("a derivative from packed activations has no gradient itself: call it under torch.no_grad() "
                         "or on detached tensors")  # fmt: skip
    ops._refuse_tangents("a derivative from packed activations", p.scale, grad)
    g2 = _rows(grad.detach())
    grad_h = g2.new_empty((T, D))
    hidden = g2.new_empty((T, cols))
    ops._launch(p.q.get_device(), "fmoe_packed_act_bwd", 1, p.q.data_ptr(), p.q.stride(0), p.scale.data_ptr(), g2.data_ptr(),
                g2.stride(0), grad_h.data_ptr(), hidden.data_ptr(), T, D, act, _DTYPES[p.dtype])  # fmt: skip
    if len(want) == 2:
        return grad_h, hidden
    return grad_h.view(p.shape), hidden.view(want)


def packed_swiglu_backward(p: PackedActivation, grad: torch.Tensor):
    """(gradient of the pre-activations, hidden rows) of hidden = silu(gate) * up at the packed
    pre-activations [gate | up], for the gradient `grad` of hidden."""
    return _backward(p, grad, _lib.ACT_SWIGLU)


def packed_gelu_backward(p: PackedActivation, grad: torch.Tensor):
    """(gradient of the pre-activations, hidden rows) of hidden = gelu(h) (the erf form) at the packed
    pre-activations, for the gradient `grad` of hidden."""
    return _backward(p, grad, _lib.ACT_GELU)
