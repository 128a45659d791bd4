"""What the norm, the 8-bit products and the packed activations refuse, without a GPU: the C entry
points answer before any launch, the Python layer has no CPU path."""

import pytest
import torch

from fastmoe_b200 import _lib
from fastmoe_b200.kernels import checkpoint, int8, norm

F32, BF16 = _lib.FMOE_F32, _lib.FMOE_BF16
P = 4096  # an address that is aligned and never read: every call below is refused


def _norm(x=P, xs=64, r=None, rs=0, w=P, wd=F32, y=P, s=None, q=None, qs=0, sc=None, T=2, D=64, eps=1e-6, dt=F32):
    return _lib.call("fmoe_rms_norm", x, xs, r, rs, w, wd, y, s, None, q, qs, sc, T, D, eps, dt, None)


@pytest.mark.parametrize("kw,match", [
    (dict(dt=7), "bad dtype"), (dict(wd=BF16), "bad dtype"), (dict(D=0), "bad sizes"), (dict(T=-1), "bad sizes"),
    (dict(T=1 << 31), "bad sizes"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=None), "null"),
    (dict(y=None), "null"), (dict(r=P, rs=64), "come together"), (dict(s=P), "come together"), (dict(xs=63), "row strides"),
    (dict(q=P), "come together"), (dict(q=P, sc=P, qs=63), "16-byte"), (dict(q=P + 8, sc=P, qs=64), "16-byte"),
    (dict(q=P, sc=P, qs=48), "16-byte"),
])  # fmt: skip
def test_norm_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _norm(**kw)


def test_norm_backward_refusals():
    def call(dw=P, scratch=P, nbytes=1 << 20, T=2, D=64, dy=P, dys=64, dt=F32):
        return _lib.call("fmoe_rms_norm_bwd", dy, dys, None, 0, P, 64, P, P, F32, P, dw, scratch, nbytes, T, D, dt, None)

    need = _lib.lib().fmoe_rms_norm_bwd_bytes(2, 64)
    assert need >= 64 * 4 and _lib.lib().fmoe_rms_norm_bwd_bytes(0, 64) == 0
    for kw, match in [(dict(nbytes=need - 1), "scratch"), (dict(scratch=None), "scratch"), (dict(dy=None), "null"),
                      (dict(dys=10), "row strides"), (dict(dt=9), "bad dtype"), (dict(D=-4), "bad sizes")]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            call(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(act=5), "activation"), (dict(out=3), "dtype"), (dict(N=0), "bad sizes"), (dict(act=1, N=33), "2\\*ff"),
    (dict(E=1025, off=P, cnt=P), "E <="), (dict(K=131072), "overflow"), (dict(off=P), "come together"),
    (dict(E=2), "several experts"), (dict(a=None), "null"), (dict(c=None), "null"), (dict(a=P + 1), "16-byte"),
    (dict(w=P + 4), "16-byte"), (dict(as_=40), "16-byte"), (dict(ws=24), "16-byte"), (dict(ws=16), "16-byte"),
    (dict(E=2, off=P, cnt=P, es=24), "16-byte"), (dict(E=2, off=P, cnt=P, es=16), "16-byte"), (dict(R=1 << 31), "int32"),
])  # fmt: skip
def test_product_refusals(kw, match):
    d = dict(a=P, as_=32, w=P, ws=32, es=32 * 32, c=P, off=None, cnt=None, E=1, R=4, N=32, K=32, act=0, out=BF16) | kw
    with pytest.raises(ValueError, match=match):
        _lib.call("fmoe_int8_gemm", d["a"], d["as_"], P, d["w"], d["ws"], d["es"], P, d["c"], d["off"], d["cnt"], d["E"],
                  d["R"], d["N"], d["K"], d["act"], d["out"], None, None)  # fmt: skip


def test_rows_and_packed_refusals():
    def rows(**kw):
        d = dict(x=P, xs=40, q=P, qs=48, T=3, D=40, dt=BF16) | kw
        return _lib.call("fmoe_quantize_rows", d["x"], d["xs"], d["q"], d["qs"], P, d["T"], d["D"], d["dt"], None)

    for kw, match in [(dict(dt=4), "dtype"), (dict(x=None), "null"), (dict(qs=40), "16-byte"), (dict(q=P + 2), "16-byte"),
                      (dict(xs=39), "row stride"), (dict(D=0), "sizes")]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            rows(**kw)
    with pytest.raises(ValueError, match="row stride"):
        _lib.call("fmoe_dequantize_rows", P, 39, P, P, 3, 40, BF16, None)

    def pack(**kw):
        d = dict(x=P, xs=40, q=P, qs=48, T=3, D=40, dt=BF16) | kw
        return _lib.call("fmoe_pack_activation", d["x"], d["xs"], d["q"], d["qs"], P, d["T"], d["D"], d["dt"], None)

    for kw, match in [(dict(dt=4), "dtype"), (dict(x=None), "null"), (dict(qs=40), "16-byte"), (dict(qs=64), "16-byte"),
                      (dict(q=None), "null"), (dict(xs=39), "row stride")]:  # fmt: skip
        with pytest.raises(ValueError, match=match):
            pack(**kw)
    for act, D, match in [(0, 40, "activation"), (1, 41, "2\\*ff"), (2, 40, "null")]:
        with pytest.raises(ValueError, match=match):
            _lib.call("fmoe_packed_act_bwd", P, 48, P, None if act == 2 else P, 40, P, P, 3, D, act, BF16, None)


def test_empty_calls_succeed_without_a_device():
    assert _norm(x=None, w=None, y=None, T=0) == 0
    assert _lib.call("fmoe_quantize_rows", None, 0, None, 0, None, 0, 8, BF16, None) == 0
    assert _lib.call("fmoe_dequantize_rows", None, 0, None, None, 0, 8, BF16, None) == 0
    assert _lib.call("fmoe_int8_gemm", None, 0, None, None, 0, 0, None, None, None, None, 1, 0, 8, 8, 0, BF16, None, None) == 0
    assert _lib.call("fmoe_pack_activation", None, 0, None, 0, None, 0, 8, BF16, None) == 0
    assert _lib.call("fmoe_packed_act_bwd", None, 0, None, None, 0, None, None, 0, 8, 1, BF16, None) == 0


def test_there_is_no_cpu_path():
    x, w = torch.randn(2, 16), torch.ones(16)
    q, scale = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    calls = [
        lambda: norm.rms_norm(x, w),
        lambda: norm.add_rms_norm(x, x, w),
        lambda: norm.rms_norm_int8(x, w),
        lambda: int8.quantize_rows(x),
        lambda: int8.dequantize_rows(int8.Int8Rows(q, scale)),
        lambda: int8.quantize_weight(x),
        lambda: int8.int8_linear(int8.Int8Rows(q, scale), int8.Int8Weight(q, scale)),
        lambda: checkpoint.pack_activation(x),
        lambda: checkpoint.unpack_activation(checkpoint.PackedActivation(q, torch.ones(2, 1), x.shape, x.dtype)),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def _entry_points(x, w, q, scale):
    """Every call of the three modules that takes floating-point tensors: the one that it is about, the call, and
    whether it follows gradients ("yes"), refuses them ("no") or reads a value on purpose ("reads")."""
    rows, weight = int8.Int8Rows(q, scale), int8.Int8Weight(q, torch.ones(2))
    packed = checkpoint.PackedActivation(q, torch.ones(2, 1), x.shape, x.dtype)
    zero, one = torch.zeros(2, 16), torch.zeros(1, dtype=torch.int64)
    unit = int8.Int8Rows(q, torch.ones(2))
    return [
        ("x", lambda: norm.rms_norm(x, w), "yes"),
        ("x", lambda: norm.add_rms_norm(x, zero, w), "yes"),
        ("x", lambda: norm.add_rms_norm(zero, x, w), "yes"),
        ("w", lambda: norm.rms_norm(zero, w), "yes"),
        ("x", lambda: norm.rms_norm_int8(x, w), "no"),
        ("x", lambda: norm.rms_norm_int8(zero, w, residual=x), "no"),
        ("w", lambda: norm.rms_norm_int8(zero, w), "no"),
        ("x", lambda: int8.quantize_rows(x), "no"),
        ("x", lambda: int8.quantize_weight(x), "reads"),
        ("scale", lambda: int8.dequantize_rows(rows), "no"),
        ("scale", lambda: int8.int8_linear(rows, weight), "no"),
        ("scale", lambda: int8.int8_linear(unit, int8.Int8Weight(q, scale)), "no"),
        ("scale", lambda: int8.grouped_int8_gemm(rows, int8.Int8Weight(q[None], torch.ones(1, 2)), one, one), "no"),
        ("scale", lambda: int8.grouped_int8_gemm(unit, int8.Int8Weight(q[None], scale[None]), one, one), "no"),
        ("x", lambda: checkpoint.pack_activation(x), "no"),
        ("scale", lambda: checkpoint.unpack_activation(packed._replace(scale=scale[:, None])), "no"),
        ("x", lambda: checkpoint.packed_gelu_backward(packed, x), "no"),
        ("x", lambda: checkpoint.packed_swiglu_backward(packed, x[:, :8]), "no"),
        ("scale", lambda: checkpoint.packed_gelu_backward(packed._replace(scale=scale[:, None]), x), "no"),
    ]


@pytest.fixture
def launches(monkeypatch):
    """The host's part of the calls without a device: CPU tensors pass, launches are counted and do nothing."""
    from fastmoe_b200.kernels import ops

    seen = []
    for module in (norm, int8, checkpoint):
        monkeypatch.setattr(module, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(int8, "_status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(ops, "_launch", lambda *args: seen.append(args[1]))
    monkeypatch.setattr(ops, "_maybe_check", lambda *args: None)
    return seen


def _given():
    return dict(x=torch.randn(2, 16), w=torch.ones(16), q=torch.zeros(2, 16, dtype=torch.int8), scale=torch.ones(2))


def test_forward_mode_is_refused_not_dropped(launches):
    """A result without a tangent would count as one that does not depend on the input."""
    from torch.autograd import forward_ad

    given = _given()
    n = len(_entry_points(**given))
    for _, call, _ in _entry_points(**given):
        call()
    assert len(launches) == n
    with forward_ad.dual_level():
        for _, call, _ in _entry_points(**given):  # nothing dual: they run
            call()
        assert len(launches) == 2 * n
        for i in range(n):
            name = _entry_points(**given)[i][0]
            dual = given | {name: forward_ad.make_dual(given[name], torch.ones_like(given[name]))}
            with pytest.raises(NotImplementedError, match="forward-mode"):
                _entry_points(**dual)[i][1]()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                _entry_points(**dual)[i][1]()
        assert len(launches) == 2 * n


def test_a_gradient_is_refused_not_dropped(launches):
    """What runs beside autograd and is given something out of a graph says so; under no_grad it runs."""
    given = _given()
    for i in range(len(_entry_points(**given))):
        name = _entry_points(**given)[i][0]
        out_of_a_graph = given | {name: given[name].clone().requires_grad_(True) * 1}
        _, call, follows = _entry_points(**out_of_a_graph)[i]
        with torch.no_grad():
            call()
        launches.clear()
        if follows == "no":
            with pytest.raises(ValueError, match="no gradient"):
                call()
            assert not launches
        else:
            result = call()
            result = result[0] if isinstance(result, tuple) else result
            assert len(launches) == 1 and result.requires_grad == (follows == "yes")
    checkpoint.pack_activation(torch.randn(2, 16).requires_grad_(True))  # a leaf is read as it is


@pytest.mark.parametrize("expert_type", ["gelu", "swiglu"])
def test_packing_that_is_not_served_is_refused(expert_type):
    """Where the experts would train with their activations unpacked all the same; without gradients nothing is
    kept, and they run."""
    from fastmoe_b200.consts import MoEImplementation
    from fastmoe_b200.models.tiny_model import MoEFeedForward

    moe = MoEFeedForward(64, 32, 2, 1, MoEImplementation.FAST, expert_type=expert_type, pack_activations=True)
    x = torch.randn(6, 64)
    with pytest.raises(ValueError, match="pack_activations"):
        moe.compute_experts(x, [2, 4])
    with torch.no_grad():
        assert moe.compute_experts(x, [2, 4]).shape == (6, 64)
    moe.requires_grad_(False)
    assert moe.compute_experts(x, [2, 4]).shape == (6, 64)
    with pytest.raises(ValueError, match="pack_activations"):
        moe.compute_experts(x.requires_grad_(True), [2, 4])
