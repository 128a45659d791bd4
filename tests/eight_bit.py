"""The 8-bit operators in 64 bits, and how far a kernel may be from them.

U = 2^-24 is half a step of fp32 relative to the value, `half(dtype)` half a step of a stored type.
A kernel that rounds k intermediate fp32 results and stores once is off by at most
(k * U + half(dtype)) * |value| where no terms cancel; sums of n fp32 terms by at most n * U times the
sum of the terms' magnitudes.
"""

import math

import torch

U = 2.0**-24
TINY = 2.0**-100
GROUP = 128


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Values below the smallest normal number are rounded to this step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def quantise(v):
    """(quotients v * 127 / a before rounding, a) of rows of float64 values, NaN where a row is not finite."""
    top = v.abs().amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top.clamp_min(TINY), torch.full_like(top, math.nan))
    return v * 127.0 / top, top


def scale_of(top):
    """a / 127 in fp32, as a correctly rounded quotient (a is an fp32 value)."""
    return (top.double() / 127.0).float().squeeze(-1)


def assert_quantised(q, scale, values):
    """q and scale are exactly what the definition gives for rows whose values are known exactly."""
    quot, top = quantise(values.double())
    fine = ~torch.isnan(top)
    want = torch.where(fine, torch.round(quot), torch.zeros_like(quot))
    assert torch.equal(q.double(), want.double())
    want_scale = scale_of(top)
    assert torch.equal(torch.isnan(scale), torch.isnan(want_scale))
    assert torch.equal(scale.nan_to_num(), want_scale.nan_to_num())


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound, element by element; NaN exactly where `want` has NaN."""
    got, want = got.double(), want.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    off = torch.where(nan, torch.zeros_like(want), (got - want).abs() - bound)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0.0, f"{what}: over the bound by {worst:.3e}"


def act_bound(h, act):
    """(activation of the float64 pre-activations h, bound of its fp32 evaluation where h is given with
    relative error e: derivative of the activation is at most 1.13, times what SwiGLU multiplies by)."""
    if act == "swiglu":
        gate, up = h.chunk(2, -1)
        s = torch.sigmoid(gate)
        out = gate * s * up
        # the fast exponential is off by (2 + |x|) steps of 2^-23 or less, the rest by four roundings
        c = (4 + 2 * gate.abs()) * 2 * U + 6 * U
        return out, c * out.abs() + 1.13 * 4 * U * (gate.abs() + TINY) * up.abs() + 4 * U * out.abs()
    if act == "gelu":
        out = 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
        # erf near -1 cancels against 1: its rounding counts against |h|, not against the result
        return out, 8 * U * h.abs() + 1.13 * 4 * U * h.abs()
    return h, 4 * U * h.abs()


def swiglu_backward(h, grad):
    gate, up = h.chunk(2, -1)
    s = torch.sigmoid(gate)
    inner = 1 + gate * (1 - s)
    c = (4 + 2 * gate.abs()) * 2 * U + 8 * U
    d_gate, d_up, hidden = grad * up * s * inner, grad * gate * s, gate * s * up
    b_gate = (grad * up * s).abs() * (1 + gate.abs()) * 2 * c
    return torch.cat([d_gate, d_up], -1), hidden, torch.cat([b_gate, c * d_up.abs()], -1), c * hidden.abs()


def gelu_backward(h, grad):
    cdf = 0.5 * (1 + torch.erf(h * math.sqrt(0.5)))
    pdf = torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    c = (4 + h * h) * 2 * U + 8 * U
    return grad * (cdf + h * pdf), h * cdf, grad.abs() * (8 * U + c * (h * pdf).abs()), 8 * U * h.abs()
