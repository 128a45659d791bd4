"""Matrix products in 8-bit integers with a scale per token and per output channel, for inference.

  quantize_rows(x)       rows of activations in 8 bits, a scale per row
  quantize_weight(w)     [N, K] or [E, N, K] weights in 8 bits, a scale per output channel
  int8_linear(a, w)      (sum_k a[r, k] w[n, k]) * a_scale[r] * w_scale[n]: nn.Linear without bias
  grouped_int8_gemm(...) the same per expert over ragged row ranges, with the activations that
                         `experts.grouped_gemm` fuses
  grouped_swiglu_ffn_int8 / grouped_gelu_ffn_int8
                         an expert's two products with the requantisation in between

They stand beside the bf16 grouped GEMM of `kernels/experts.py` (the expert loop of
src/fastmoe/models/tiny_model.py:282-294) with half the weight bytes and the integer tensor-core
rate. The sum over k is exact in 32-bit integers. A run of values is held as
q = round(v * 127 / a), scale = a / 127 with a its largest magnitude (at least 2^-100), rounding
ties to even; a row that holds NaN or infinity has scale NaN.

Rows of q lie at 16-byte steps: `Int8Rows.q` and `Int8Weight.q` are views of padded storage
where K is not a multiple of 16. Nothing here has a gradient: a call whose inputs ask for one is refused
(`quantize_weight` reads a parameter as it is).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from . import ops
from .ops import _DTYPES, _require_cuda, _status_word

__all__ = [
    "Int8Rows",
    "Int8Weight",
    "quantize_rows",
    "dequantize_rows",
    "quantize_weight",
    "int8_linear",
    "grouped_int8_gemm",
    "grouped_swiglu_ffn_int8",
    "grouped_gelu_ffn_int8",
]

MAX_K = 131071  # 128 * 128 * K stays inside a signed 32-bit sum
MAX_EXPERTS = 1024


class Int8Rows(NamedTuple):
    q: torch.Tensor  # int8 [T, K]
    scale: torch.Tensor  # float32 [T]


class Int8Weight(NamedTuple):
    q: torch.Tensor  # int8 [N, K] or [E, N, K]
    scale: torch.Tensor  # float32 [N] or [E, N]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as [T, D] rows with unit column stride, without a copy where its strides allow."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _padded(K: int) -> int:
    return (K + 15) // 16 * 16


def empty_rows(like: torch.Tensor, T: int, K: int) -> Int8Rows:
    """Uninitialised 8-bit rows [T, K] and their scales, on the device of `like`."""
    Kp = _padded(K)
    q = like.new_empty((T, Kp), dtype=torch.int8)
    return Int8Rows(q if Kp == K else q[:, :K], like.new_empty((T,), dtype=torch.float32))


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """The rows (last dimension) of x in 8 bits: `q` [T, K] with T = all leading dimensions, `scale`
    float32 [T]."""
    _require_cuda(x, "x")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be float32/bfloat16/float16 rows, got {tuple(x.shape)} {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("quantize_rows has no gradient: call it under torch.no_grad() or on detached tensors")
    ops._refuse_tangents("quantize_rows", x)
    x2 = _rows(x)
    T, K = x2.shape
    out = empty_rows(x2, T, K)
    q, scale = out
    ops._launch(x.get_device(), "fmoe_quantize_rows", 1, x2.data_ptr(), x2.stride(0), q.data_ptr(), q.stride(0),
                scale.data_ptr(), T, K, dtype)  # fmt: skip
    return out


def dequantize_rows(rows: Int8Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """q * scale as a [T, K] matrix of `dtype`."""
    q, scale = rows
    _check_rows(q, scale)
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype}; use float32, bfloat16 or float16")
    if scale.requires_grad and torch.is_grad_enabled():
        raise ValueError("dequantize_rows has no gradient: call it under torch.no_grad() or on detached scales")
    ops._refuse_tangents("dequantize_rows", scale)
    q, scale = _rows(q), scale.contiguous()
    T, K = q.shape
    out = q.new_empty((T, K), dtype=dtype)
    ops._launch(q.get_device(), "fmoe_dequantize_rows", 1, q.data_ptr(), q.stride(0), scale.data_ptr(), out.data_ptr(), T, K,
                _DTYPES[dtype])  # fmt: skip
    return out


def quantize_weight(w: torch.Tensor) -> Int8Weight:
    """A weight [N, K] (nn.Linear layout) or [E, N, K] in 8 bits with a scale per output channel. Done
    once per weight, not per call; a trained parameter is read through `w.detach()`."""
    if w.dim() not in (2, 3):
        raise ValueError(f"w must be [N, K] or [E, N, K], got {tuple(w.shape)}")
    ops._refuse_tangents("quantize_weight", w)
    r = quantize_rows(w.detach())
    lead = w.shape[:-1]
    return Int8Weight(r.q.unflatten(0, lead) if w.dim() == 3 else r.q, r.scale.view(lead))


def _check_rows(q, scale):
    _require_cuda(q, "q")
    if q.dtype != torch.int8 or q.dim() != 2 or q.shape[1] == 0:
        raise ValueError(f"q must be int8 [T, K], got {tuple(q.shape)} {q.dtype}")
    if scale.dtype != torch.float32 or scale.shape != q.shape[:1] or scale.get_device() != q.get_device():
        raise ValueError(f"scale must be float32 {tuple(q.shape[:1])} on {q.device}, got {tuple(scale.shape)} "
                         f"{scale.dtype} on {scale.device}")  # fmt: skip


def _operand(q: torch.Tensor) -> torch.Tensor:
    """q with rows at 16-byte steps and readable up to the last step: q itself where its strides and
    storage say so (what the functions above return), else a padded copy."""
    shape = q.shape
    K = shape[-1]
    if K % 16 == 0 and q.is_contiguous() and q.data_ptr() % 16 == 0:
        return q
    lead, strides = shape[:-1], q.stride()
    ok = (K == 1 or strides[-1] == 1) and q.data_ptr() % 16 == 0 and strides[-2] % 16 == 0 and strides[-2] >= K
    if len(shape) == 3:
        ok = ok and strides[0] % 16 == 0 and strides[0] >= shape[-2] * strides[-2]
    if ok and K % 16:
        last = q.storage_offset() + sum((n - 1) * s for n, s in zip(lead, strides[:-1])) + _padded(K)
        ok = last <= q.untyped_storage().nbytes()
    if ok or q.numel() == 0:
        return q
    out = torch.zeros(*lead, _padded(K), dtype=torch.int8, device=q.device)
    out[..., :K] = q
    return out[..., :K]


def _product(a, w, offsets, counts, act, out, E):
    # held in names until the launch: a copy made only for its address would be freed before it
    aq, wq, sa, sw = _operand(a.q), _operand(w.q), a.scale.contiguous(), w.scale.contiguous()
    wshape, wstride = wq.shape, wq.stride()
    N, K = wshape[-2:]
    R = aq.shape[0]
    dev = aq.get_device()
    # a single row (or expert) may have any stride
    w_row = wstride[-2] if N > 1 else _padded(K)
    ops._launch(
        dev, "fmoe_int8_gemm", 1, aq.data_ptr(), aq.stride(0) if R > 1 else _padded(K), sa.data_ptr(), wq.data_ptr(),
        w_row, wstride[0] if E > 1 else N * w_row, sw.data_ptr(), out.data_ptr(),
        None if offsets is None else offsets.data_ptr(), None if counts is None else counts.data_ptr(), E, R, N, K, act,
        _DTYPES[out.dtype], _status_word(aq.device).data_ptr(),
    )  # fmt: skip
    ops._maybe_check(aq.device, "fmoe_int8_gemm")
    return out


def _check_operands(a, w, dims, out_dtype):
    q, wq, ws = a.q, w.q, w.scale
    _check_rows(q, a.scale)
    _require_cuda(wq, "w")
    wshape, K = wq.shape, q.shape[1]
    if wq.dtype != torch.int8 or len(wshape) != dims or wshape[-1] != K:
        raise ValueError(f"a must be int8 [R, K] and w int8 {'[E, N, K]' if dims == 3 else '[N, K]'}; got "
                         f"{tuple(q.shape)} and {tuple(wshape)} {wq.dtype}")  # fmt: skip
    if ws.dtype != torch.float32 or ws.shape != wshape[:-1]:
        raise ValueError(f"w's scale must be float32 {tuple(wshape[:-1])}, got {tuple(ws.shape)} {ws.dtype}")
    dev = q.get_device()
    if wq.get_device() != dev or ws.get_device() != dev:
        raise ValueError(f"a lives on {q.device}, w on {wq.device} and {ws.device}")
    if wshape[-2] == 0:
        raise ValueError("w has no output channels")
    if K > MAX_K:
        raise ValueError(f"K={K} could overflow the 32-bit sums (K <= {MAX_K})")
    if out_dtype not in _DTYPES:
        raise ValueError(f"unsupported out_dtype {out_dtype}; use float32, bfloat16 or float16")
    if (a.scale.requires_grad or ws.requires_grad) and torch.is_grad_enabled():
        raise ValueError("a product in 8 bits has no gradient: call it under torch.no_grad() or on detached scales")
    ops._refuse_tangents("a product in 8 bits", a.scale, ws)


def int8_linear(a: Int8Rows, w: Int8Weight, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [T, K] times w [N, K] transposed, both in 8 bits: [T, N] in `out_dtype`, rounded once."""
    _check_operands(a, w, 2, out_dtype)
    out = a.q.new_empty((a.q.shape[0], w.q.shape[0]), dtype=out_dtype)
    return _product(a, w, None, None, _lib.ACT_NONE, out, 1)


def grouped_int8_gemm(a: Int8Rows, w: Int8Weight, offsets, counts, activation: int = _lib.ACT_NONE,
                      covers_all_rows: bool = False, out_dtype: torch.dtype = torch.bfloat16):  # fmt: skip
    """Per expert e, over its rows [offsets[e], offsets[e] + counts[e]) (int64 [E] on the device): rows of
    a [R, K] times w[e] [N, K] transposed, both in 8 bits, then the activation (`experts.ACT_NONE`,
    `ACT_SWIGLU`: the first N/2 channels are the gate, or `ACT_GELU`), rounded once to `out_dtype`: [R, N], or
    [R, N/2] for SwiGLU. No two experts may have a row in common. Rows that belong to no expert read zero; `covers_all_rows=True` promises that
    there are none, which saves the zero-fill."""
    _check_operands(a, w, 3, out_dtype)
    E, N = w.q.shape[:2]
    act = int(activation)
    if act not in (_lib.ACT_NONE, _lib.ACT_SWIGLU, _lib.ACT_GELU):
        raise ValueError(f"activation must be ACT_NONE, ACT_SWIGLU or ACT_GELU, got {activation!r}")
    if act == _lib.ACT_SWIGLU and N % 2:
        raise ValueError(f"SwiGLU needs N = 2*ff, got N={N}")
    if E > MAX_EXPERTS:
        raise ValueError(f"grouped_int8_gemm supports up to {MAX_EXPERTS} experts, got {E}")
    for name, t in (("offsets", offsets), ("counts", counts)):
        if t.dtype != torch.int64 or t.shape != (E,) or t.device != a.q.device:
            raise ValueError(f"{name} must be int64 [{E}] on {a.q.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    cols = N // 2 if act == _lib.ACT_SWIGLU else N
    alloc = a.q.new_empty if covers_all_rows else a.q.new_zeros
    out = alloc((a.q.shape[0], cols), dtype=out_dtype)
    if E == 0:
        return out
    return _product(a, w, offsets.contiguous(), counts.contiguous(), act, out, E)


def grouped_swiglu_ffn_int8(a: Int8Rows, w_gate_up: Int8Weight, w_down: Int8Weight, offsets, counts,
                            covers_all_rows: bool = False, out_dtype: torch.dtype = torch.bfloat16):  # fmt: skip
    """down(silu(gate(a)) * up(a)) per expert, both products in 8 bits. The hidden rows are rounded to
    `out_dtype` and quantised row by row between the two. w_gate_up [E, 2*ff, D], w_down [E, D, ff]."""
    hidden = grouped_int8_gemm(a, w_gate_up, offsets, counts, _lib.ACT_SWIGLU, covers_all_rows, out_dtype)
    return grouped_int8_gemm(quantize_rows(hidden), w_down, offsets, counts, _lib.ACT_NONE, covers_all_rows, out_dtype)


def grouped_gelu_ffn_int8(a: Int8Rows, w1: Int8Weight, w2: Int8Weight, offsets, counts,
                          covers_all_rows: bool = False, out_dtype: torch.dtype = torch.bfloat16):  # fmt: skip
    """fc2(gelu(fc1(a))) per expert, both products in 8 bits, as grouped_swiglu_ffn_int8."""
    hidden = grouped_int8_gemm(a, w1, offsets, counts, _lib.ACT_GELU, covers_all_rows, out_dtype)
    return grouped_int8_gemm(quantize_rows(hidden), w2, offsets, counts, _lib.ACT_NONE, covers_all_rows, out_dtype)
