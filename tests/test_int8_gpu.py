"""8-bit rows, weights and products against the definition in 64 bits. The sum over k is exact, so a
product may differ from 64 bits by the roundings of its conversion, its two scales and its store."""

import pytest
import torch

from eight_bit import TINY, U, act_bound, assert_quantised, assert_within, half, smallest
from fastmoe_b200 import _lib
from fastmoe_b200.kernels import experts, int8, norm, ops
from fastmoe_b200.kernels.int8 import Int8Rows, Int8Weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
KERNELS = {"by the sizes": -1, "tiles": 0, "few rows": 1, "split K": 2, "pairs": 3}


@pytest.fixture(params=sorted(KERNELS), autouse=True)
def kernel(request):
    """Every test of this file runs with the kernel that the library picks and with each of the four behind
    fmoe_int8_gemm."""
    _lib.tune("int8_kernel", KERNELS[request.param])
    yield request.param
    _lib.tune("int8_kernel", -1)


ACTS = {"none": _lib.ACT_NONE, "swiglu": _lib.ACT_SWIGLU, "gelu": _lib.ACT_GELU}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _operand(g, *shape, scale):
    K = shape[-1]
    q = torch.full((*shape[:-1], (K + 15) // 16 * 16), 77, dtype=torch.int8, device=DEV)  # what lies past K does not count
    q[..., :K] = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
    return q[..., :K], (0.5 + torch.rand(*shape[:-1], generator=g, device=DEV)) * scale


def _case(R, K, *wshape, seed=0):
    g = _gen(seed)
    a = Int8Rows(*_operand(g, R, K, scale=1 / 40))
    return a, Int8Weight(*_operand(g, *wshape, K, scale=1 / (73 * K**0.5)))


def _product64(a, wq, ws):
    return (a.q.double() @ wq.double().t()) * a.scale.double()[:, None] * ws.double()


def _check(out, h, act, dtype):
    ref, bound = act_bound(h, act)
    assert out.dtype == dtype and out.shape == ref.shape
    assert_within(out, ref, bound * (1 + half(dtype)) + half(dtype) * ref.abs() + smallest(dtype) + TINY, act)


LINEAR = [(1, 1, 1), (1, 16, 8), (1, 7168, 515), (2, 15, 33), (3, 17, 64), (7, 127, 100), (8, 128, 256), (9, 129, 257),
          (16, 1000, 255), (17, 640, 130), (32, 96, 31), (33, 2048, 1024), (48, 7168, 300), (64, 512, 4100), (65, 200, 96),
          (100, 1001, 513), (128, 128, 256), (129, 144, 20), (200, 4096, 7), (300, 320, 1999), (1000, 1024, 768),
          # K in 2, 4 and 8 parts with 128, 32 and 16 tokens to a tile, and in 4 with ragged ones
          (256, 5200, 7168), (20, 4104, 7100), (16, 4111, 600), (130, 2304, 515)]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K,N", LINEAR)
def test_linear(R, K, N, dtype):
    a, w = _case(R, K, N, seed=R + K + N)
    out = int8.int8_linear(a, w, out_dtype=dtype)
    torch.cuda.synchronize()
    assert ops.read_status() == 0
    _check(out, _product64(a, w.q, w.scale), "none", dtype)


def test_the_sum_is_exact_at_its_largest():
    """All products +-127^2 over the widest K whose sums stay inside 32 bits: nothing saturates or wraps."""
    K = 131071
    q = torch.full((2, 131072), 127, dtype=torch.int8, device=DEV)
    q[1] = -128
    ones = torch.ones(2, device=DEV)
    a, w = Int8Rows(q[:, :K], ones), Int8Weight(q[:, :K], ones)
    out = int8.int8_linear(a, w, out_dtype=torch.float32)
    want = torch.tensor([[127 * 127, -127 * 128], [-127 * 128, 128 * 128]], dtype=torch.float64, device=DEV) * K
    assert_within(out, want, U * want.abs(), "sum")
    with pytest.raises(ValueError, match="32-bit sums"):
        int8.int8_linear(Int8Rows(q, ones), Int8Weight(q, ones))


GROUPED = [
    ([1], 64, 32),
    ([0, 0, 3, 0], 100, 65),
    ([1] * 40, 128, 256),
    ([2, 0, 1, 3, 0, 0, 1, 1], 520, 330),
    ([8, 9, 16, 17, 0, 31], 208, 514),
    ([33, 1, 64, 65], 256, 128),
    ([200, 0, 5, 300], 512, 512),
    ([128, 256, 127, 129], 130, 258),
    ([700, 33], 1000, 250),
    ([2100, 1, 2050], 192, 600),  # more row blocks than share their column blocks' weights
    ([40], 4104, 7168), ([9, 0, 7], 2048, 384), ([31, 20, 0, 3], 3333, 259), ([100, 28], 2000, 512),  # a long K in parts
]


def _spread(counts, gap=0):
    cnt = torch.tensor(counts, dtype=torch.int64, device=DEV)
    return torch.cumsum(cnt + gap, 0) - cnt - gap, cnt


@pytest.mark.parametrize("act", ["none", "swiglu", "gelu"])
@pytest.mark.parametrize("counts,K,N", GROUPED)
def test_grouped(counts, K, N, act):
    a, w = _case(sum(counts), K, len(counts), N, seed=K + N)
    if act == "swiglu" and N % 2:
        w = Int8Weight(w.q[:, : N - 1], w.scale[:, : N - 1])
    off, cnt = _spread(counts)
    for dtype in (torch.bfloat16, torch.float32):
        out = int8.grouped_int8_gemm(a, w, off, cnt, ACTS[act], out_dtype=dtype)
        torch.cuda.synchronize()
        assert ops.read_status() == 0
        h = torch.cat([_product64(Int8Rows(a.q[o : o + n], a.scale[o : o + n]), w.q[e], w.scale[e])
                       for e, (o, n) in enumerate(zip(off.tolist(), counts))])  # fmt: skip
        _check(out, h, act, dtype)


@pytest.mark.parametrize("counts", [[3, 0, 2], [300, 40, 129]])
def test_rows_of_no_expert(counts):
    gap = 5
    R = sum(counts) + gap * len(counts) + 4
    a, w = _case(R, 96, 3, 70, seed=1)
    off, cnt = _spread(counts, gap)
    mine = torch.zeros(R, dtype=torch.bool, device=DEV)
    for o, n in zip(off.tolist(), counts):
        mine[o : o + n] = True
    out = int8.grouped_int8_gemm(a, w, off, cnt)
    assert not out[~mine].any() and out[mine].any()
    # the kernel itself leaves them alone: a buffer that held something keeps it
    kept = torch.full_like(out, 3.0)
    int8._product(a, w, off, cnt, _lib.ACT_NONE, kept, 3)
    assert torch.equal(kept[mine], out[mine]) and bool((kept[~mine] == 3.0).all())


@pytest.mark.parametrize("R", [10, 400])
def test_a_range_past_the_rows_is_cut_off(R):
    a, w = _case(R, 64, 3, 64, seed=2)
    off = torch.tensor([0, R - 3, R + 7], dtype=torch.int64, device=DEV)
    cnt = torch.tensor([R - 3, 900, 2], dtype=torch.int64, device=DEV)
    ops.read_status()
    out = int8.grouped_int8_gemm(a, w, off, cnt, out_dtype=torch.float32)
    assert ops.read_status() & _lib.STATUS_BAD_EXPERT
    h = torch.cat([_product64(Int8Rows(a.q[:-3], a.scale[:-3]), w.q[0], w.scale[0]),
                   _product64(Int8Rows(a.q[-3:], a.scale[-3:]), w.q[1], w.scale[1])])  # fmt: skip
    _check(out, h, "none", torch.float32)


def test_values_past_32_bits():
    """More than 2^31 values in the rows, in the result and in the experts' weights."""
    tail = 5
    for R, K, N in (((1 << 31) // 8208 + 300, 8208, 8), ((1 << 31) // 8208 + 300, 16, 8208)):
        a, w = _case(tail, K, N)
        q = torch.zeros(R, K, dtype=torch.int8, device=DEV)
        scale = torch.ones(R, device=DEV)
        q[-tail:], scale[-tail:] = a.q, a.scale
        out = int8.int8_linear(Int8Rows(q, scale), w)
        assert not out[:-tail].any()
        _check(out[-tail:], _product64(a, w.q, w.scale), "none", torch.bfloat16)
    del q, out
    E, K, N = 70, 8192, 4096
    a, w = _case(tail, K, 1, N)
    wq = torch.zeros(E, N, K, dtype=torch.int8, device=DEV)
    ws = torch.ones(E, N, device=DEV)
    wq[-1], ws[-1] = w.q[0], w.scale[0]
    cnt = torch.zeros(E, dtype=torch.int64, device=DEV)
    cnt[-1] = tail
    out = int8.grouped_int8_gemm(a, Int8Weight(wq, ws), torch.zeros_like(cnt), cnt)
    _check(out, _product64(a, w.q[0], w.scale[0]), "none", torch.bfloat16)


@pytest.mark.parametrize("K", [512, 2048])
def test_experts_that_claim_the_same_rows(kernel, K):
    """Where this leaves rows without their product (the clusters that the split-K kernel cuts a long K over are
    counted by the rows) the status word says so; nothing outside is touched."""
    a, w = _case(32, K, 4, 96)
    off, cnt = torch.zeros(4, dtype=torch.int64, device=DEV), torch.full((4,), 32, dtype=torch.int64, device=DEV)
    ops.read_status()
    int8.grouped_int8_gemm(a, w, off, cnt)
    torch.cuda.synchronize()
    assert ops.read_status() == (_lib.STATUS_BAD_EXPERT if kernel == "split K" and K == 2048 else 0)


def test_operands_off_the_16_byte_grid_and_with_strides():
    g = _gen(3)
    base = torch.randint(-127, 128, (3, 41, 150), generator=g, device=DEV, dtype=torch.int8)
    q = torch.randint(-127, 128, (20, 301), generator=g, device=DEV, dtype=torch.int8)
    a = Int8Rows(q[::2, 3:104], torch.rand(20, generator=g, device=DEV)[::2])
    w = Int8Weight(base[:, 1:, 7:108], torch.rand(3, 80, generator=g, device=DEV)[:, ::2])
    out = int8.int8_linear(a, Int8Weight(w.q[1], w.scale[1]), torch.float32)
    _check(out, _product64(a, w.q[1], w.scale[1]), "none", torch.float32)
    off, cnt = _spread([4, 0, 6])
    out = int8.grouped_int8_gemm(a, w, off, cnt, out_dtype=torch.float32)
    h = torch.cat([_product64(Int8Rows(a.q[:4], a.scale[:4]), w.q[0], w.scale[0]),
                   _product64(Int8Rows(a.q[4:], a.scale[4:]), w.q[2], w.scale[2])])  # fmt: skip
    _check(out, h, "none", torch.float32)
    # columns of w that are not contiguous
    wt = Int8Weight(base[0, :40, :101].t().contiguous().t(), w.scale[0])
    _check(int8.int8_linear(a, wt, torch.float32), _product64(a, wt.q, wt.scale), "none", torch.float32)


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 11)])
def test_every_quotient_of_16_bit_values(kernel, dtype, bits):
    """A row for each significand of the largest magnitude, with all significands of the values in the nine
    binades below it: among them every exact tie."""
    if kernel != "by the sizes":
        return  # there is no product in it
    one = 2 ** (bits - 1)
    sig = torch.arange(one, 2 * one, device=DEV, dtype=torch.float32) / one
    values = torch.cat([sig * 2.0**-e for e in range(9)])
    x = torch.where(values[None] <= sig[:, None], values[None], -sig[:, None] / 2).to(dtype)
    x[:, 1::2] *= -1
    x = torch.cat([sig[:, None].to(dtype), x], 1)
    assert torch.equal(x.abs().amax(1).float(), sig)
    for scale in (1.0, 2.0**-5):
        rows = int8.quantize_rows(x * scale)
        assert_quantised(rows.q, rows.scale, x * scale)
    # the same values in groups of 128 columns, each with its row's largest value in front
    from fastmoe_b200.kernels import checkpoint

    n = (x.shape[1] - 1) // 127 * 127
    groups = torch.cat([x[:, :1, None].expand(-1, n // 127, 1), x[:, 1 : n + 1].view(one, -1, 127)], 2)
    p = checkpoint.pack_activation(groups.reshape(one, -1))
    for k in range(n // 127):
        assert_quantised(p.q[:, 128 * k : 128 * k + 128], p.scale[:, k], groups[:, k])


@pytest.mark.parametrize("K", [1, 33, 640, 7168])
def test_quantised_operands_end_to_end(K):
    g = _gen(K)
    x = torch.randn(30, K, generator=g, device=DEV)
    x[3] = 0
    x[4] *= 1e-25
    x[5] *= 1e25
    w = torch.nn.Parameter(torch.randn(50, K, generator=g, device=DEV) / K**0.5)
    wq = int8.quantize_weight(w)
    assert_quantised(wq.q, wq.scale, w.detach())
    a = int8.quantize_rows(x)
    assert_quantised(a.q, a.scale, x)
    out = int8.int8_linear(a, wq, torch.float32)
    _check(out, _product64(a, wq.q, wq.scale), "none", torch.float32)
    # the quantised product next to the plain one: each value is off by half a step at most
    ref = x.double() @ w.detach().double().t()
    step_a, step_w = a.scale.double()[:, None], wq.scale.double()
    off = 0.5 * (step_a * w.detach().double().abs().sum(1) + step_w * x.double().abs().sum(1, keepdim=True)) + 0.25 * K * step_a * step_w
    assert_within(out, ref, off * (1 + 1e-5), "against the unquantised product")


@pytest.mark.parametrize("R", [3, 200])
def test_rows_with_nan_and_infinity_stay_visible(R):
    x = torch.randn(R, 64, device=DEV)
    x[1, 5] = float("nan")
    x[2, 63] = float("-inf")
    a, w = int8.quantize_rows(x), int8.quantize_weight(torch.randn(40, 64, device=DEV))
    out = int8.int8_linear(a, w)
    bad = torch.isnan(out)
    assert bad[1:3].all() and not bad[0].any() and not bad[3:].any()
    assert torch.isnan(int8.dequantize_rows(a)[1:3]).all()


def test_no_rows_and_no_experts():
    a, w = _case(0, 64, 32)
    assert int8.int8_linear(a, w).shape == (0, 32)
    a, w = _case(6, 64, 2, 32)
    off, cnt = _spread([0, 0])
    assert not int8.grouped_int8_gemm(a, w, off, cnt).any()
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert not int8.grouped_int8_gemm(a, Int8Weight(w.q[:0], w.scale[:0]), none, none).any()
    assert int8.quantize_rows(torch.empty(0, 5, device=DEV)).q.shape == (0, 5)
    assert int8.dequantize_rows(int8.quantize_rows(torch.empty(0, 5, device=DEV))).shape == (0, 5)


def test_refusals():
    a, w = _case(4, 64, 32)
    off, cnt = _spread([4])
    with pytest.raises(ValueError, match="int8"):
        int8.int8_linear(Int8Rows(a.q.float(), a.scale), w)
    with pytest.raises(ValueError, match="scale must be"):
        int8.int8_linear(Int8Rows(a.q, a.scale[:3]), w)
    with pytest.raises(ValueError, match="scale must be"):
        int8.int8_linear(a, Int8Weight(w.q, w.scale[:3]))
    with pytest.raises(ValueError, match="must be int8"):
        int8.int8_linear(a, Int8Weight(w.q[:, :32], w.scale))
    with pytest.raises(ValueError, match="E, N, K"):
        int8.grouped_int8_gemm(a, w, off, cnt)
    with pytest.raises(ValueError, match="out_dtype"):
        int8.int8_linear(a, w, torch.float64)
    w3 = Int8Weight(w.q[None], w.scale[None])
    with pytest.raises(ValueError, match="counts"):
        int8.grouped_int8_gemm(a, w3, off, cnt.int())
    with pytest.raises(ValueError, match="offsets"):
        int8.grouped_int8_gemm(a, w3, off.cpu(), cnt)
    with pytest.raises(ValueError, match="activation"):
        int8.grouped_int8_gemm(a, w3, off, cnt, activation=9)
    with pytest.raises(ValueError, match="2\\*ff"):
        int8.grouped_int8_gemm(a, Int8Weight(w3.q[:, :31], w3.scale[:, :31]), off, cnt, _lib.ACT_SWIGLU)
    with pytest.raises(ValueError, match="no gradient"):
        int8.quantize_rows(torch.randn(2, 8, device=DEV, requires_grad=True))
    with pytest.raises(RuntimeError, match="no CPU path"):
        int8.quantize_rows(torch.randn(2, 8))
    with pytest.raises(ValueError, match="w must be"):
        int8.quantize_weight(torch.randn(8, device=DEV))


def _ffn64(a, w1, w2, counts, act, dtype):
    """The FFN on the hidden rows that the kernels really have (each stage is held to its own bound above)."""
    off, cnt = _spread(counts)
    hidden = int8.grouped_int8_gemm(a, w1, off, cnt, ACTS[act], out_dtype=dtype)
    rows = int8.quantize_rows(hidden)
    o = 0
    parts = []
    for e, n in enumerate(counts):
        parts.append(_product64(Int8Rows(rows.q[o : o + n], rows.scale[o : o + n]), w2.q[e], w2.scale[e]))
        o += n
    return torch.cat(parts)


@pytest.mark.parametrize("act,ffn", [("swiglu", int8.grouped_swiglu_ffn_int8), ("gelu", int8.grouped_gelu_ffn_int8)])
def test_norm_to_experts_together(act, ffn):
    """The serving chain: residual sum, norm and 8-bit rows in one pass, the experts on them."""
    counts, D, ff = [40, 0, 7, 33], 200, 96
    g = _gen(8)
    x, r = (torch.randn(sum(counts), D, generator=g, device=DEV).bfloat16() for _ in range(2))
    w1 = int8.quantize_weight(torch.randn(4, ff * (2 if act == "swiglu" else 1), D, generator=g, device=DEV) / D**0.5)
    w2 = int8.quantize_weight(torch.randn(4, D, ff, generator=g, device=DEV) / ff**0.5)
    a = norm.rms_norm_int8(x, torch.ones(D, device=DEV), residual=r)
    off, cnt = _spread(counts)
    out = ffn(a.rows, w1, w2, off, cnt, covers_all_rows=True)
    _check(out, _ffn64(a.rows, w1, w2, counts, act, torch.bfloat16), "none", torch.bfloat16)


def test_on_a_side_stream_and_in_graphs():
    """Two captured graphs of the same call, replayed on two streams at once, and an eager call between
    them: no memory is shared between calls."""
    cases = [_case(5, 512, 300, seed=4), _case(300, 512, 300, seed=5), _case(2100, 256, 300, seed=6),
             _case(48, 7168, 300, seed=7), _case(130, 4096, 1000, seed=8)]  # fmt: skip
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    for (a, w), s in zip(cases, streams):
        int8.int8_linear(a, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(int8.int8_linear(a, w))
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = [int8.int8_linear(a, w) for a, w in cases]
    torch.cuda.synchronize()
    for out, e, (a, w) in zip(outs, eager, cases):
        assert torch.equal(out, e)
        _check(out, _product64(a, w.q, w.scale), "none", torch.bfloat16)


def test_waits_that_run_out_are_reported(kernel):
    """With its producer issuing nothing, the product's bounded waits give up: status bit, no hang."""
    if kernel == "few rows":
        return  # it waits for nothing
    a, w = _case(600, 256, 512)
    _lib.tune("gemm_skip_loads", 1)
    _lib.tune("gemm_spin_limit", 2000)
    try:
        int8.int8_linear(a, w)
        torch.cuda.synchronize()
        assert ops.read_status() & _lib.STATUS_WAIT_TIMEOUT
    finally:
        _lib.tune("gemm_skip_loads", 0)
        _lib.tune("gemm_spin_limit", 1 << 24)
    _check(int8.int8_linear(a, w), _product64(a, w.q, w.scale), "none", torch.bfloat16)
    assert ops.read_status() == 0 and experts.ACT_NONE == 0


def test_a_single_row_has_any_stride():
    """One output channel, one expert or one token, cut out of something wider: its stride says nothing."""
    K = 64
    a, w = _case(5, K, 3, 4, seed=1)  # three experts of four channels
    wide = torch.full((4, K + 9), 5, dtype=torch.int8, device=DEV)
    wide[0, :K] = w.q[0, 0]
    one = wide[:1, :K]
    assert one.is_contiguous() and one.stride(0) == K + 9
    narrow = torch.empty(K, 1, dtype=torch.int8, device=DEV)
    narrow[:, 0] = w.q[0, 0]
    off, cnt = _spread([5])
    for q in (one, narrow.t()):
        out = int8.int8_linear(a, Int8Weight(q, w.scale[0, :1]), out_dtype=torch.float32)
        _check(out, _product64(a, q, w.scale[0, :1]), "none", torch.float32)
        out = int8.grouped_int8_gemm(a, Int8Weight(q[None], w.scale[:1, :1]), off, cnt, out_dtype=torch.float32)
        _check(out, _product64(a, q, w.scale[0, :1]), "none", torch.float32)
    expert = torch.empty(4 * K + 7, dtype=torch.int8, device=DEV).as_strided((1, 4, K), (4 * K + 7, K, 1))
    expert.copy_(w.q[:1])
    out = int8.grouped_int8_gemm(a, Int8Weight(expert, w.scale[:1]), off, cnt, out_dtype=torch.float32)
    _check(out, _product64(a, w.q[0], w.scale[0]), "none", torch.float32)
    # one token
    token = Int8Rows(one, a.scale[:1])
    out = int8.int8_linear(token, Int8Weight(w.q[1], w.scale[1]), out_dtype=torch.float32)
    _check(out, _product64(token, w.q[1], w.scale[1]), "none", torch.float32)
    from fastmoe_b200.kernels import routing

    ix = routing.build_index(torch.tensor([[1, 0]], device=DEV), torch.ones(1, 2, device=DEV), 3)
    for q, size in ((one, K), (narrow.t(), K), (wide[:1, : K - 3], K - 3)):
        rows = routing.permute_int8_rows(Int8Rows(q, a.scale[:1]), ix, 2)
        assert torch.equal(rows.q, q.expand(2, size)) and torch.equal(rows.scale, a.scale[:1].expand(2))
    assert torch.equal(int8.dequantize_rows(token, torch.float32), one.float() * a.scale[0])
    torch.cuda.synchronize()
    assert ops.read_status() == 0
