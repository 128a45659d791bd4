"""Activations kept in 8 bits: the packed values against the definition, the activation derivatives
against the formulas in 64 bits at the values that the 8 bits stand for."""

import pytest
import torch

from eight_bit import GROUP, U, assert_quantised, assert_within, gelu_backward, half, smallest, swiglu_backward
from fastmoe_b200.kernels import checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (1, 128), (2, 2), (3, 30), (5, 127), (4, 129), (7, 256), (33, 1000), (200, 514), (3, 4096), (100, 2056),
          (5, 16), (3, 144), (7, 2000), (6, 528)]  # fmt: skip


def _x(T, D, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + T * 7 + D)
    return (2 * torch.randn(T, D, generator=g, device=DEV)).to(dtype)


def _values(p):
    """What the packed values stand for, in 64 bits from the fp32 scale."""
    scale = p.scale.double().repeat_interleave(GROUP, 1)[:, : p.q.shape[1]]
    return p.q.double() * scale


def _check_packed(p, x):
    D = x.shape[1]
    for k in range(0, D, GROUP):
        assert_quantised(p.q[:, k : k + GROUP], p.scale[:, k // GROUP], x[:, k : k + GROUP])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_pack_and_unpack(T, D, dtype):
    x = _x(T, D, dtype)
    p = checkpoint.pack_activation(x)
    _check_packed(p, x)
    back = checkpoint.unpack_activation(p)
    ref = _values(p)
    assert back.shape == x.shape
    assert_within(back, ref, (half(dtype) + 2 * U) * ref.abs() + smallest(dtype), "unpacked")
    # and next to x: half a step of the group, and the roundings of the value read back
    step = p.scale.double().repeat_interleave(GROUP, 1)[:, :D]
    assert_within(back, x, step * (0.5 + 127 * (half(dtype) + 4 * U)) + smallest(dtype), "against x")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("act", ["swiglu", "gelu"])
def test_backward_from_packed(T, D, dtype, act):
    if act == "swiglu" and D % 2:
        D += 1
    x = _x(T, D, dtype)
    cols = D // 2 if act == "swiglu" else D
    grad = _x(T, cols, dtype, seed=1)
    p = checkpoint.pack_activation(x)
    run = checkpoint.packed_swiglu_backward if act == "swiglu" else checkpoint.packed_gelu_backward
    grad_h, hidden = run(p, grad)
    d, h, bound_d, bound_h = (swiglu_backward if act == "swiglu" else gelu_backward)(_values(p), grad.double())
    # the dequantised value itself is rounded to fp32 once: slopes of the results in it, per relative U,
    # are below (2 + |x|) times the terms that the bounds already count in multiples of eight
    assert_within(grad_h, d, 2 * bound_d + half(dtype) * d.abs() + smallest(dtype), "grad")
    assert_within(hidden, h, 2 * bound_h + half(dtype) * h.abs() + smallest(dtype), "hidden")


def test_strides_leading_dimensions_and_autograd_leaves():
    x = _x(24, 300, torch.bfloat16)
    p = checkpoint.pack_activation(x[:, 5:261].requires_grad_(True))
    _check_packed(p, x[:, 5:261])
    x3 = x[:, :256].reshape(2, 12, 256)
    p3 = checkpoint.pack_activation(x3)
    assert checkpoint.unpack_activation(p3).shape == (2, 12, 256)
    grad = _x(24, 260, torch.bfloat16, seed=2)[:, 2:130]
    a = checkpoint.packed_swiglu_backward(p3, grad.reshape(2, 12, 128))
    b = checkpoint.packed_swiglu_backward(checkpoint.pack_activation(x3.reshape(24, 256)), grad)
    assert a[0].shape == (2, 12, 256) and a[1].shape == (2, 12, 128)
    assert torch.equal(a[0].view(24, 256), b[0]) and torch.equal(a[1].view(24, 128), b[1])
    # columns that are not contiguous, an expanded gradient
    pt = checkpoint.pack_activation(x.t().contiguous().t())
    assert torch.equal(pt.q, checkpoint.pack_activation(x).q)
    one = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(24, 300)
    _, h = checkpoint.packed_gelu_backward(pt, one)
    assert torch.equal(h, checkpoint.packed_gelu_backward(pt, one.contiguous())[1])


@pytest.mark.parametrize("D", [512, 300])
def test_on_a_side_stream_and_in_a_graph(D):
    """Captured once, replayed on new values, beside eager calls on another stream."""
    x, grad, side = _x(70, D, torch.bfloat16), _x(70, D // 2, torch.bfloat16, seed=3), torch.cuda.Stream()

    def run():
        p = checkpoint.pack_activation(x)
        return (p.q, p.scale, checkpoint.unpack_activation(p), *checkpoint.packed_swiglu_backward(p, grad))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = run()
    x.copy_(_x(70, D, torch.bfloat16, seed=9))
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(side):
            graph.replay()
        eager = run()
    torch.cuda.synchronize()
    for a, b in zip(captured, eager):
        assert torch.equal(a, b)


def test_groups_of_zeros_and_of_infinities():
    x = _x(4, 384, torch.float32)
    x[0, :128] = 0
    x[1, 130] = float("inf")
    x[2, 300] = float("nan")
    x[3, 128:256] = 1e-38
    p = checkpoint.pack_activation(x)
    _check_packed(p, x)
    back = checkpoint.unpack_activation(p)
    assert not back[0, :128].any() and torch.isnan(back[1, 128:256]).all() and torch.isnan(back[2, 256:]).all()
    assert torch.isfinite(back[1, :128]).all() and torch.isfinite(back[3]).all()


def test_values_past_32_bits():
    """More than 2^31 values: the last rows come out as they do alone."""
    D, tail = 8200, 5
    T = (1 << 31) // D + 300
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = _x(tail, D, torch.bfloat16)
    p, few = checkpoint.pack_activation(x), checkpoint.pack_activation(x[-tail:])
    assert torch.equal(p.q[-tail:], few.q) and torch.equal(p.scale[-tail:], few.scale)
    assert torch.equal(checkpoint.unpack_activation(p)[-tail:], checkpoint.unpack_activation(few))
    for derivative, cols in ((checkpoint.packed_swiglu_backward, D // 2), (checkpoint.packed_gelu_backward, D)):
        for got, want in zip(derivative(p, x[:, :cols]), derivative(few, x[-tail:, :cols])):
            assert bool(want.any()) and torch.equal(got[-tail:], want)


def test_no_rows_and_refusals():
    p = checkpoint.pack_activation(torch.empty(0, 64, device=DEV))
    assert checkpoint.unpack_activation(p).shape == (0, 64)
    assert checkpoint.packed_gelu_backward(p, torch.empty(0, 64, device=DEV))[0].shape == (0, 64)
    x = _x(4, 65, torch.float32)
    p = checkpoint.pack_activation(x)
    with pytest.raises(ValueError, match="even width"):
        checkpoint.packed_swiglu_backward(p, x)
    with pytest.raises(ValueError, match="grad must be"):
        checkpoint.packed_gelu_backward(p, x.bfloat16())
    with pytest.raises(ValueError, match="grad must be"):
        checkpoint.packed_gelu_backward(p, x[:, :64])
    with pytest.raises(ValueError, match="laid out"):
        checkpoint.unpack_activation(p._replace(q=p.q.contiguous()))
    with pytest.raises(ValueError, match="laid out"):
        checkpoint.unpack_activation(p._replace(scale=p.scale[:2]))
    for shape in ((2, 65), (4, 64), (2, 2, 66), ()):
        with pytest.raises(ValueError, match="does not have"):
            checkpoint.unpack_activation(p._replace(shape=torch.Size(shape)))
        with pytest.raises(ValueError, match="does not have"):
            checkpoint.packed_gelu_backward(p._replace(shape=torch.Size(shape)), x[: shape[0] if shape else 4])
    with pytest.raises(ValueError, match="float32/bfloat16/float16"):
        checkpoint.pack_activation(x.double())
    with pytest.raises(RuntimeError, match="no CPU path"):
        checkpoint.pack_activation(x.cpu())
