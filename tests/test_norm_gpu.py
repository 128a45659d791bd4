"""The RMS norm, its gradient and its 8-bit output against the formulas in 64 bits. The bounds count
roundings (see eight_bit.py); they are not fitted to what the kernels return."""

import pytest
import torch

from eight_bit import U, assert_quantised, assert_within, half, quantise, smallest
from fastmoe_b200.kernels import int8, norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# one token and many; a warp's row and a block's; 16-byte vectors and single elements; widths around the
# block shapes' borders, and rows too wide for registers
SHAPES = [(1, 1), (1, 7168), (3, 64), (5, 63), (300, 257), (9, 1024), (2, 1032), (700, 2056), (7, 4099), (310, 4104),
          (3, 8193), (2, 16384), (299, 16384), (2, 20001), (3, 33000),
          (400, 3001), (400, 814), (400, 600), (1300, 1000), (1300, 300)]  # fmt: skip


def _inputs(T, D, dtype, wdtype=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, r, dy, ds = (rnd(T, D).to(dtype) for _ in range(4))
    return x, r, dy, ds, (1 + 0.3 * rnd(D)).to(wdtype or dtype)


def _norm64(s, w):
    s = s.double()
    rstd = 1 / (s.square().mean(-1, keepdim=True) + EPS).sqrt()
    return s * rstd * w.double(), rstd


def _check_forward(y, s, w):
    ref, _ = _norm64(s, w)
    # rstd, two products and the store
    assert_within(y, ref, (half(y.dtype) + 4 * U) * ref.abs() + smallest(y.dtype), "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_forward_and_backward(T, D, dtype):
    x, r, dy, ds, w = _inputs(T, D, dtype)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = norm.add_rms_norm(x, r, w, EPS)
    assert torch.equal(s, (x.detach().float() + r.detach().float()).to(dtype))
    _check_forward(y.detach(), s.detach(), w.detach())
    gx, gr, gw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    assert torch.equal(gx, gr)
    _check_backward(gx, gw, s.detach(), w.detach(), dy, ds)
    # the same without a residual
    y1 = norm.rms_norm(x, w, EPS)
    _check_forward(y1.detach(), x.detach(), w.detach())
    gx, gw = torch.autograd.grad(y1, (x, w), dy)
    _check_backward(gx, gw, x.detach(), w.detach(), dy, None)


def _check_backward(gx, gw, s, w, dy, ds):
    T, D = s.shape
    _, rstd = _norm64(s, w)
    xh, g = s.double() * rstd, dy.double() * w.double()
    mean = (g * xh).mean(-1, keepdim=True)
    add = torch.zeros_like(g) if ds is None else ds.double()
    ref = rstd * (g - xh * mean) + add
    # every term rounded a few times; the mean: D terms, added by at least 32 threads and then in a tree
    mean_off = (D / 32 + 32) * U * (g * xh).abs().mean(-1, keepdim=True)
    bound = 8 * U * (rstd * (g.abs() + (xh * mean).abs()) + add.abs()) + rstd * xh.abs() * mean_off
    assert_within(gx, ref, bound + half(gx.dtype) * ref.abs() + smallest(gx.dtype), "dx")
    term = dy.double() * xh
    ref = term.sum(0)
    assert_within(gw, ref, (T + 8) * U * term.abs().sum(0) + half(gw.dtype) * ref.abs() + smallest(gw.dtype), "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_width_has_a_shape_that_launches(dtype):
    """Block shapes and shared memory go by the width: a step of 61 columns passes through all of them."""
    for T in (2, 300):
        for D in range(61, 9000, 61):
            x, r, dy, ds, w = _inputs(T, D, dtype)
            x.requires_grad_(True)
            w.requires_grad_(True)
            y, s = norm.add_rms_norm(x, r, w, EPS)
            gx, gw = torch.autograd.grad((y, s), (x, w), (dy, ds))
    _check_backward(gx, gw, s.detach(), w.detach(), dy, ds)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [512, 515])
def test_fp32_weight_beside_16_bit_rows(dtype, D):
    x, r, dy, ds, w = _inputs(40, D, dtype, torch.float32)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = norm.add_rms_norm(x, r, w, EPS)
    assert y.dtype == s.dtype == dtype
    _check_forward(y.detach(), s.detach(), w.detach())
    gx, gw = torch.autograd.grad((y, s), (x, w), (dy, ds))
    assert gw.dtype == torch.float32
    _check_backward(gx, gw, s.detach(), w.detach(), dy, ds)


def _assert_norm_quantised(rows, s, w):
    """q next to the quotient of the 64-bit norm: half a step, and what three roundings of y and of the
    largest |y| can shift a quotient of up to 127."""
    ref, _ = _norm64(s, w)
    quot, top = quantise(ref)
    assert_within(rows.q, quot, 0.5 + 127 * 8 * U, "q")
    assert_within(rows.scale, top.squeeze(-1) / 127, 6 * U * top.squeeze(-1) / 127, "scale")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_eight_bit_output(T, D, dtype):
    x, r, _, _, w = _inputs(T, D, dtype, seed=3)
    out = norm.rms_norm_int8(x, w, EPS, residual=r, with_y=True)
    s = (x.float() + r.float()).to(dtype)
    assert torch.equal(out.stream, s) and out.rows.q.shape == (T, D)
    _check_forward(out.y, s, w)
    _assert_norm_quantised(out.rows, s, w)
    plain = norm.rms_norm_int8(x, w, EPS)
    assert plain.stream is None and plain.y is None
    _assert_norm_quantised(plain.rows, x, w)
    # the bytes between D and the next multiple of 16 are zeros
    padded = out.rows.q.as_strided((T, (D + 15) // 16 * 16), out.rows.q.stride())
    assert not padded[:, D:].any()


@pytest.mark.parametrize("T", [1, 2, 400, 1500])
def test_a_row_does_not_depend_on_its_batch(T):
    """The sums run in 64 bits: a row has the same bits alone and in a batch, whatever shape runs."""
    for D in (1016, 7168, 5001):
        x, r, _, _, w = _inputs(T, D, torch.bfloat16, seed=4)
        out = norm.rms_norm_int8(x, w, EPS, residual=r, with_y=True)
        one = norm.rms_norm_int8(x[-1:], w, EPS, residual=r[-1:], with_y=True)
        assert torch.equal(out.rows.q[-1:], one.rows.q) and torch.equal(out.rows.scale[-1:], one.rows.scale)
        assert torch.equal(out.y[-1:], one.y)


@pytest.mark.parametrize("D", [8200, 8203, 200])
def test_values_past_32_bits(D):
    """More than 2^31 values, in each form of the kernels: the last rows come out as they do alone."""
    T, tail = (1 << 31) // D + 300, 5
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=DEV)
    x[-tail:], r, dy, ds, w = _inputs(tail, D, torch.bfloat16)
    grads = torch.zeros_like(x)
    grads[-tail:] = dy
    few = x[-tail:].clone()
    xg, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    gx, gw = torch.autograd.grad(norm.rms_norm(xg, wg, EPS), (xg, wg), grads)
    _check_backward(gx[-tail:], gw, few, w, dy, None)  # rows of zeros add nothing to dw
    assert not gx[:-tail].any()
    del gx, grads, xg
    rows, alone = int8.quantize_rows(x), int8.quantize_rows(few)
    assert torch.equal(rows.q[-tail:], alone.q) and torch.equal(rows.scale[-tail:], alone.scale)
    assert torch.equal(int8.dequantize_rows(rows)[-tail:], int8.dequantize_rows(alone))
    out, alone = norm.rms_norm_int8(x, w, EPS, with_y=True), norm.rms_norm_int8(few, w, EPS, with_y=True)
    assert torch.equal(out.rows.q[-tail:], alone.rows.q) and torch.equal(out.y[-tail:], alone.y)


@pytest.mark.parametrize("D", [200, 204, 2051])
def test_rows_with_strides(D):
    x, r, dy, ds, w = _inputs(30, 2 * D + 3, torch.bfloat16)
    w = w[:D].clone().requires_grad_(True)
    x, r, dy = x[:, 3 : D + 3], r[::2, :D].repeat(2, 1), dy[:, :D]  # views that start off the 16-byte grid
    xs, rs = x.detach().requires_grad_(True), r.detach().requires_grad_(True)
    y, s = norm.add_rms_norm(xs, rs, w, EPS)
    _check_forward(y.detach(), s.detach(), w.detach())
    gx, gw = torch.autograd.grad((y, s), (xs, w), (dy, ds[:, D : 2 * D]))
    _check_backward(gx, gw, s.detach(), w.detach(), dy, ds[:, D : 2 * D])
    # columns that are not contiguous, and rows of a 3-D tensor
    xt = x.t().contiguous().t()
    assert torch.equal(norm.rms_norm(xt, w, EPS), norm.rms_norm(x.contiguous(), w, EPS))
    x3 = x.reshape(5, 6, D)
    out = norm.rms_norm_int8(x3, w.detach(), EPS, residual=x3, with_y=True)
    assert out.stream.shape == out.y.shape == x3.shape and out.rows.q.shape == (30, D)


@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_a_weight_off_the_16_byte_grid(wdtype):
    x, r, dy, ds, w = _inputs(20, 513, torch.bfloat16, wdtype)
    x, r, dy, ds, w = x[:, 1:].contiguous(), r[:, :512], dy[:, :512], ds[:, :512], w[1:]
    xs, ws = x.clone().requires_grad_(True), w.detach().requires_grad_(True)
    y, s = norm.add_rms_norm(xs, r, ws, EPS)
    _check_forward(y.detach(), s.detach(), w)
    gx, gw = torch.autograd.grad((y, s), (xs, ws), (dy, ds))
    _check_backward(gx, gw, s.detach(), w, dy, ds)


def test_no_second_derivative():
    x, r, dy, ds, w = _inputs(3, 64, torch.float32)
    x.requires_grad_(True)
    y, _ = norm.add_rms_norm(x, r, w, EPS)
    (gx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    (plain,) = torch.autograd.grad(norm.add_rms_norm(x, r, w, EPS)[0], x, dy)
    assert torch.equal(gx, plain)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(gx.sum() + x.sum(), x)


def test_a_stream_changed_in_place_is_noticed():
    x, r, dy, ds, w = _inputs(3, 64, torch.float32)
    x.requires_grad_(True)
    for shape in ((3, 64), (1, 3, 64)):
        y, s = norm.add_rms_norm(x.view(shape), r.view(shape), w, EPS)
        s.add_(1)
        with pytest.raises(RuntimeError, match="inplace operation"):
            torch.autograd.grad(y, x, dy.view(shape))


def test_one_tensor_as_both_inputs_and_leaves_that_accumulate():
    x, _, dy, ds, w = _inputs(5, 96, torch.float32)
    x.requires_grad_(True)
    y, s = norm.add_rms_norm(x, x, w, EPS)
    torch.autograd.backward((y, s), (dy, ds))
    r = x.detach().clone().requires_grad_(True)
    x2 = x.detach().clone().requires_grad_(True)
    y, s = norm.add_rms_norm(x2, r, w, EPS)
    torch.autograd.backward((y, s), (dy, ds))
    assert torch.equal(x.grad, 2 * x2.grad) and torch.equal(x2.grad, r.grad)
    r.grad.add_(1)  # each leaf has a gradient of its own
    assert not torch.equal(x2.grad, r.grad)


def test_rows_of_zeros_and_of_infinities():
    x = torch.randn(6, 300, device=DEV)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 299] = float("nan")
    x[4] = 1e-30
    w = torch.ones(300, device=DEV)
    out = norm.rms_norm_int8(x, w, EPS, with_y=True)
    assert float(out.y[1].abs().max()) == 0 and float(out.rows.scale[1]) > 0 and not out.rows.q[1].any()
    assert torch.isnan(out.rows.scale).tolist() == [False, False, True, True, False, False]
    assert not out.rows.q[2:4].any()
    _check_forward(out.y[[0, 1, 4, 5]], x[[0, 1, 4, 5]], w)
    # eps = 0 and a row of zeros: 0 * inf
    assert torch.isnan(norm.rms_norm(x[1:2], w, 0.0)).all()


def test_only_one_of_the_outputs_has_a_gradient():
    x, r, dy, ds, w = _inputs(12, 136, torch.float32)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = norm.add_rms_norm(x, r, w, EPS)
    gx, gr, gw = torch.autograd.grad(s, (x, r, w), ds, allow_unused=True, retain_graph=True)
    assert torch.equal(gx, ds) and torch.equal(gr, ds) and gw is None
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    _check_backward(gx, gw, s.detach(), w.detach(), dy, None)
    # a frozen residual and weight, then a frozen input
    y, s = norm.add_rms_norm(x, r.detach(), w.detach(), EPS)
    (gx2,) = torch.autograd.grad((y, s), x, (dy, ds))
    _check_backward(gx2, gw, s.detach(), w.detach(), dy, ds)
    y2 = norm.rms_norm(x.detach(), w, EPS)
    (gw2,) = torch.autograd.grad(y2, w, dy)
    _check_backward(torch.autograd.grad(norm.rms_norm(x, w, EPS), x, dy)[0], gw2, x.detach(), w.detach(), dy, None)
    # the gradient of a broadcast (expanded) upstream
    y3 = norm.rms_norm(x, w, EPS)
    gx3, gw3 = torch.autograd.grad(y3.sum(), (x, w))
    _check_backward(gx3, gw3, x.detach(), w.detach(), torch.ones_like(x), None)


def test_gradient_against_differences():
    """Central differences of the fp32 kernel along a random direction. Rounding: each y carries 4 U,
    so L(x) = <dy, y> carries 4 U sum|dy y|, twice, over 2h; truncation: the difference between the
    quotients at h and 2h, which is three times the error of the one at h."""
    x, r, dy, ds, w = _inputs(3, 264, torch.float32, seed=9)
    d, dr, dw = torch.randn_like(x), torch.randn_like(r), torch.randn_like(w)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, s = norm.add_rms_norm(x, r, w, EPS)
    gx, gr, gw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    slope = float((gx.double() * d).sum() + (gr.double() * dr).sum() + (gw.double() * dw).sum())

    def loss(h):
        with torch.no_grad():
            yh, sh = norm.add_rms_norm(x + h * d, r + h * dr, w + h * dw, EPS)
            return float((yh.double() * dy).sum() + (sh.double() * ds).sum())

    h = 2.0**-6
    one, two = (loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)
    size = float((y.detach().double() * dy).abs().sum() + (s.detach().double() * ds).abs().sum())
    # the inputs x + h d are rounded too: another 2 U of the sum, through a slope of rstd or 1
    rounding = 2 * 8 * U * size / (2 * h)
    assert abs(slope - one) <= rounding + abs(one - two)


def test_dw_has_the_same_bits_from_run_to_run():
    x, r, dy, ds, w = _inputs(2000, 1024, torch.bfloat16)
    for t in (x, w):
        t.requires_grad_(True)
    first = [torch.autograd.grad(norm.rms_norm(x, w, EPS), (x, w), dy) for _ in range(3)]
    assert all(torch.equal(a, b) for other in first[1:] for a, b in zip(first[0], other))


def test_no_rows_and_refusals():
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    y, s = norm.add_rms_norm(x, x.detach(), w, EPS)
    gx, gw = torch.autograd.grad((y, s), (x, w), (y.detach(), s.detach()))
    assert y.shape == gx.shape == (0, 64) and not gw.any()
    assert norm.rms_norm_int8(x.detach(), w.detach()).rows.q.shape == (0, 64)
    x = torch.randn(4, 64, device=DEV)
    with pytest.raises(ValueError, match="no gradient"):
        norm.rms_norm_int8(x, w)
    w = w.detach()
    with pytest.raises(ValueError, match="weight must be"):
        norm.rms_norm(x, w[:63])
    with pytest.raises(ValueError, match="weight must be"):
        norm.rms_norm(x, w.bfloat16())
    with pytest.raises(ValueError, match="residual must match"):
        norm.add_rms_norm(x, x[:3], w)
    with pytest.raises(ValueError, match="residual must match"):
        norm.add_rms_norm(x, x.half(), w)
    with pytest.raises(ValueError, match="residual"):
        norm.add_rms_norm(x, None, w)
    with pytest.raises(ValueError, match="eps"):
        norm.rms_norm(x, w, -1.0)
    with pytest.raises(ValueError, match="float32/bfloat16/float16"):
        norm.rms_norm(x.double(), w.double())
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm.rms_norm(x, w.cpu())


def test_on_a_side_stream_and_in_a_graph():
    x, r, dy, ds, w = _inputs(64, 1000, torch.bfloat16)
    for t in (x, r, w):
        t.requires_grad_(True)

    def step():  # returns no graph: torch cannot capture a backward while an eager graph of its leaves lives
        y, s = norm.add_rms_norm(x, r, w, EPS)
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), (x, r, w), (dy, ds)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    for _ in range(2):
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), captured))


def test_quantised_rows_are_exact():
    from fastmoe_b200.kernels import int8

    for dtype in DTYPES:
        for T, D in SHAPES:
            x = _inputs(T, D, dtype, seed=T + D)[0]
            rows = int8.quantize_rows(x)
            assert_quantised(rows.q, rows.scale, x)
            back = int8.dequantize_rows(rows, dtype)
            assert torch.equal(back, (rows.q.float() * rows.scale[:, None]).to(dtype))


def test_backward_of_two_widths_from_two_threads():
    """One instantiation serves rows of many widths with different amounts of shared memory; a call lets go of
    the interpreter's lock, so two threads' calls interleave on the host."""
    import threading

    from fastmoe_b200 import _lib

    T, calls, errors, outs = 300, 4000, [], {}
    nbytes = {D: _lib.lib().fmoe_rms_norm_bwd_bytes(T, D) for D in (4104, 16384)}
    data = {D: _inputs(T, D, torch.bfloat16) for D in nbytes}
    torch.cuda.synchronize()

    def work(D):
        x, _, dy, _, w = data[D]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            rstd = (1 / (x.double().square().mean(-1) + EPS).sqrt()).float()
            dx, dw, scratch = torch.empty_like(x), torch.empty_like(w), torch.empty(nbytes[D], dtype=torch.uint8, device=DEV)
        args = (dy.data_ptr(), D, None, 0, x.data_ptr(), D, rstd.data_ptr(), w.data_ptr(), _lib.FMOE_BF16, dx.data_ptr(),
                dw.data_ptr(), scratch.data_ptr(), nbytes[D], T, D, _lib.FMOE_BF16, stream.cuda_stream)  # fmt: skip
        try:
            for _ in range(calls):
                _lib.call("fmoe_rms_norm_bwd", *args)
        except Exception as e:  # noqa: BLE001
            errors.append((D, e))
        stream.synchronize()
        outs[D] = (dx, dw)

    threads = [threading.Thread(target=work, args=(D,)) for D in nbytes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for D, (dx, dw) in outs.items():
        x, _, dy, _, w = data[D]
        _check_backward(dx, dw, x, w, dy, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [11, 13, 15, 333, 1003, 7001, 8965])
def test_nothing_behind_the_weight_counts(dtype, D):
    """Every shift of rows of odd width, with NaN where the weight ends (what may be read is checked where the
    kernels are compiled)."""
    for T in (9, 400):
        x, r, dy, ds, w = _inputs(T, D, dtype, seed=D)
        behind = torch.full((D + 40,), float("nan"), dtype=dtype, device=DEV)
        behind[:D] = w
        xs, ws = x.clone().requires_grad_(True), behind[:D].requires_grad_(True)
        y, s = norm.add_rms_norm(xs, r, ws, EPS)
        _check_forward(y.detach(), s.detach(), w)
        gx, gw = torch.autograd.grad((y, s), (xs, ws), (dy, ds))
        _check_backward(gx, gw, s.detach(), w, dy, ds)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2, 300])
def test_every_width_is_right(T, dtype):
    """Block shapes and shared memory go by the width: a step of 61 columns passes through all of them, and
    the widths around their borders follow. Each output of each of them is looked at."""
    borders = [k * v + d for v in (4, 8) for k in (32, 64, 128, 256, 512, 1024, 2048) for d in (-1, 0, 1, v - 1)]
    for D in sorted({*range(61, 9000, 61), *borders}):
        x, r, dy, ds, w = _inputs(T, D, dtype, seed=D)
        x.requires_grad_(True)
        w.requires_grad_(True)
        y, s = norm.add_rms_norm(x, r, w, EPS)
        gx, gw = torch.autograd.grad((y, s), (x, w), (dy, ds))
        s, w = s.detach(), w.detach()
        _check_forward(y.detach(), s, w)
        _check_backward(gx, gw, s, w, dy, ds)
        out = norm.rms_norm_int8(x.detach(), w, EPS, residual=r, with_y=True)
        assert torch.equal(out.stream, s) and torch.equal(out.y, y)
        _assert_norm_quantised(out.rows, s, w)
        rows = int8.quantize_rows(s)
        assert_quantised(rows.q, rows.scale, s)
