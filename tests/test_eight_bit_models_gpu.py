"""The RMS norm, the int8 products and the packed activations where the models use them."""

import pytest
import torch
import torch.nn.functional as F

from eight_bit import GROUP, U, assert_within, half, swiglu_backward
from fastmoe_b200.consts import MoEImplementation
from fastmoe_b200.kernels import checkpoint, experts, int8, norm, ops, routing
from fastmoe_b200.models.tiny_model import Block, Int8Linear, MoEBlock, MoEFeedForward, PipelinedMoEBlock, RMSNorm, TinyModel

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def _randn(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _values(x):
    """What x's packed form stands for, in 64 bits."""
    p = checkpoint.pack_activation(x)
    return p.q.double() * p.scale.double().repeat_interleave(GROUP, 1)[:, : x.shape[1]]


@pytest.mark.parametrize("with_map", [False, True])
@pytest.mark.parametrize("act", ["swiglu", "gelu"])
def test_packed_ffn(act, with_map):
    """Result as without packing; gradients against the formulas at the packed values. Each bf16
    rounding on the way (hidden rows, their gradient, the pre-activations' gradient, the unpacked
    rows) counts half a step, each fp32 sum of n terms n U of its terms' magnitudes."""
    counts, D, ff = [70, 0, 33, 129], 256, 256
    R, E = sum(counts), len(counts)
    g = torch.Generator(device=DEV).manual_seed(1)
    w1 = _randn(g, E, 2 * ff if act == "swiglu" else ff, D, scale=D**-0.5).requires_grad_(True)
    w2 = _randn(g, E, D, ff, scale=ff**-0.5).requires_grad_(True)
    x, gout = _randn(g, R, D).requires_grad_(True), _randn(g, R, D)
    cnt = torch.tensor(counts, device=DEV)
    off = torch.cumsum(cnt, 0) - cnt
    row_map = torch.randperm(R, generator=g, device=DEV) if with_map else None
    ffn = experts.grouped_swiglu_ffn if act == "swiglu" else experts.grouped_gelu_ffn
    plain = ffn(x, w1, w2, off, cnt, row_map, covers_all_rows=True)
    out = ffn(x, w1, w2, off, cnt, row_map, covers_all_rows=True, packed=True)
    assert torch.equal(plain, out)
    gx, g1, g2 = torch.autograd.grad(out, (x, w1, w2), gout)
    gg = gout if row_map is None else gout[row_map]
    # the pre-activations that the forward packs
    pre = experts.grouped_gemm(x.detach(), w1.detach(), off, cnt, covers_all_rows=True)
    kept, xk = _values(pre), _values(x.detach())
    h = half(BF16)
    o = 0
    for e, n in enumerate(counts):
        r = slice(o, o + n)
        o += n
        a1, a2, go = w1.detach()[e].double(), w2.detach()[e].double(), gg[r].double()
        gh = go @ a2
        e_gh = h * gh.abs() + (D + 2) * U * (go.abs() @ a2.abs())
        k = kept[r]
        if act == "swiglu":
            gp, hid, b, _ = swiglu_backward(k, gh)
            slope = swiglu_backward(k, torch.ones_like(gh))[0].abs()
            e_gp = slope * torch.cat([e_gh, e_gh], -1) * (1 + h) + 4 * b + h * gp.abs()
        else:
            cdf, pdf = 0.5 * (1 + torch.erf(k * 0.5**0.5)), torch.exp(-0.5 * k * k) / (2 * torch.pi) ** 0.5
            gp, hid = gh * (cdf + k * pdf), k * cdf
            e_gp = (cdf + k * pdf).abs() * e_gh * (1 + h) + h * gp.abs() + 64 * U * gh.abs() * (1 + k.abs())
        e_hid = h * hid.abs() + 32 * U * (kept.abs().amax() + 1) ** 2
        ref = go.t() @ hid
        assert_within(g2[e], ref, go.abs().t() @ (e_hid + (n + 2) * U * hid.abs()) + h * ref.abs() + 1e-12, "dw2")
        xv = xk[r]
        ref = gp.t() @ xv
        bound = e_gp.t() @ xv.abs() * (1 + h) + gp.abs().t() @ xv.abs() * (h + (n + 4) * U)
        assert_within(g1[e], ref, bound + h * ref.abs() + 1e-12, "dw1")
        ref = gp @ a1
        bound = e_gp @ a1.abs() + (a1.shape[0] + 2) * U * (gp.abs() @ a1.abs())
        assert_within(gx[r], ref, bound + h * ref.abs() + 1e-12, "dx")
    # only some of the gradients
    (only,) = torch.autograd.grad(ffn(x, w1.detach(), w2.detach(), off, cnt, row_map, covers_all_rows=True, packed=True), x, gout)
    assert torch.equal(only, gx)
    (only,) = torch.autograd.grad(ffn(x.detach(), w1, w2.detach(), off, cnt, row_map, covers_all_rows=True, packed=True), w1, gout)
    assert torch.equal(only, g1)
    with torch.no_grad():
        assert torch.equal(ffn(x, w1, w2, off, cnt, row_map, covers_all_rows=True, packed=True), plain)


def test_packed_ffn_has_no_second_derivative():
    g = torch.Generator(device=DEV).manual_seed(2)
    w1, w2 = _randn(g, 1, 512, 256, scale=1 / 16).requires_grad_(True), _randn(g, 1, 256, 256, scale=1 / 16)
    x = _randn(g, 9, 256).requires_grad_(True)
    cnt = torch.tensor([9], device=DEV)
    out = experts.grouped_swiglu_ffn(x, w1, w2, cnt - cnt, cnt, covers_all_rows=True, packed=True)
    plain = torch.autograd.grad(out.sum(), (x, w1), retain_graph=True)
    again = torch.autograd.grad(out.sum(), (x, w1), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(again[0].float().sum() + w1.float().sum(), w1)


def test_packed_ffn_refusals():
    w1 = torch.zeros(2, 512, 256, dtype=BF16, device=DEV, requires_grad=True)
    x = torch.zeros(4, 256, dtype=BF16, device=DEV)
    cnt = torch.tensor([2, 2], device=DEV)
    off = cnt.cumsum(0) - cnt
    with pytest.raises(ValueError, match="second weight"):
        experts.grouped_swiglu_ffn(x, w1, w1[:, :256, :128].contiguous(), off, cnt, packed=True)
    with pytest.raises(ValueError, match="multiple"):
        experts.grouped_swiglu_ffn(x[:, :64].contiguous(), w1[:, :, :64].contiguous(),
                                   torch.zeros(2, 64, 256, dtype=BF16, device=DEV), off, cnt, packed=True)  # fmt: skip


@pytest.mark.parametrize("expert_type", ["swiglu", "gelu"])
def test_layer_with_packed_activations(expert_type):
    """The same result and router gradient path, less memory held for the backward pass, gradients next
    to the unpacked ones: the kept values are off by a group's largest magnitude / 254, about 4 / 254 of
    the spread of normally distributed values, so 5% of the gradients' norm is well outside of it."""
    torch.manual_seed(0)
    moe = MoEFeedForward(256, 256, 8, 2, MoEImplementation.FAST, expert_type=expert_type).to(DEV).to(BF16)
    moe.grouped_gelu_min_experts = 1
    packed = MoEFeedForward(256, 256, 8, 2, MoEImplementation.FAST, expert_type=expert_type, pack_activations=True)
    packed = packed.to(DEV).to(BF16)
    packed.load_state_dict(moe.state_dict())
    x = torch.randn(2, 2048, 256, device=DEV).to(BF16)
    gout = torch.randn_like(x)
    held, grads, outs = [], [], []
    for layer in (moe, packed):
        xi = x.clone().requires_grad_(True)
        layer(xi)  # once before, so that caches are filled
        before = torch.cuda.memory_allocated()
        out = layer(xi)
        held.append(torch.cuda.memory_allocated() - before)
        grads.append(torch.autograd.grad(out, [xi, *layer.parameters()], gout))
        outs.append(out.detach())
    assert torch.equal(outs[0], outs[1])
    assert held[1] < held[0]
    for a, b in zip(*grads):
        assert float((a.float() - b.float()).norm()) <= 0.05 * float(a.float().norm())
    assert ops.read_status() == 0


def _plain_rms(x, w, eps=1e-6):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w


def _plain_block(block, x):
    """The block in plain float64 torch."""
    a = block.attn
    B, T, D = x.shape
    w = {k: p.detach().double() for k, p in block.named_parameters()}
    h = _plain_rms(x, w["norm1.weight"])
    q, k, v = (h @ w["attn.qkv.weight"].t()).view(B, T, 3, a.n_heads, a.hd).permute(2, 0, 3, 1, 4)
    y = torch.softmax(q @ k.transpose(-1, -2) / a.hd**0.5, -1) @ v
    x = x + y.transpose(1, 2).reshape(B, T, D) @ w["attn.proj.weight"].t()
    h = _plain_rms(x, w["norm2.weight"])
    return x + F.gelu(h @ w["ff.fc1.weight"].t()) @ w["ff.fc2.weight"].t()


def test_block_with_rms_norm_fp32():
    torch.manual_seed(1)
    block = Block(96, 4, 160, norm="rms").to(DEV)
    with torch.no_grad():
        block.norm1.weight.mul_(1 + 0.2 * torch.randn(96, device=DEV))
        block.norm2.weight.mul_(1 + 0.2 * torch.randn(96, device=DEV))
    x = torch.randn(2, 17, 96, device=DEV, requires_grad=True)
    out = block(x)
    ref = _plain_block(block, x.detach().double())
    # fp32 library products of at most 160 terms in four stages: 4 * 160 U of the largest magnitude
    assert float((out.detach().double() - ref).abs().max()) <= 4 * 160 * 2 * U * float(ref.abs().max())
    out.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in [x, *block.parameters()])
    # the gradient along a direction, against differences of the float64 block
    d = torch.randn_like(x)
    e = 1e-4
    slope = (_plain_block(block, x.detach().double() + e * d) - _plain_block(block, x.detach().double() - e * d)).sum() / (2 * e)
    size = float((x.grad.double() * d).abs().sum())
    assert abs(float((x.grad.double() * d).sum() - slope)) <= 8 * 160 * 2 * U * size + 1e-6 * abs(float(slope))


@pytest.mark.parametrize("impl", [MoEImplementation.FAST, MoEImplementation.STANDARD])
def test_models_train_with_rms_norm(impl):
    torch.manual_seed(2)
    kw = dict(pack_activations=True) if impl == MoEImplementation.FAST else {}
    model = TinyModel(128, 256, 4, 256, 2, num_experts=8, top_k=2, implementation=impl, use_moe=True, norm="rms",
                      expert_type="swiglu" if kw else "gelu", **kw).to(DEV).to(BF16)  # fmt: skip
    x = torch.randn(2, 64, 128, device=DEV, dtype=BF16)
    model(x).float().square().mean().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    # under autocast: fp32 modules, the attention's branch in bf16 beside an fp32 stream
    block = Block(64, 4, 128, norm="rms").to(DEV)
    with torch.autocast("cuda", BF16):
        out = block(torch.randn(1, 8, 64, device=DEV))
    assert out.dtype == torch.float32 and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("expert_type", ["swiglu", "gelu"])
def test_layer_in_int8(expert_type, dtype):
    torch.manual_seed(3)
    moe = MoEFeedForward(200, 96, 8, 2, MoEImplementation.FAST, expert_type=expert_type).to(DEV).to(dtype)
    x = torch.randn(3, 5, 200, device=DEV, dtype=dtype)
    moe.quantize_int8()
    assert moe.is_int8 and "w1_q" not in moe.state_dict()
    with torch.no_grad():
        out = moe(x)
        rows = int8.quantize_rows(x)
        assert torch.equal(out, moe(x, rows))
        # the layer by hand, expert by expert
        flat = x.view(-1, 200)
        w, idx = routing.route_topk(moe.router(flat), 2, w_dtype=dtype)
        ffn = int8.grouped_swiglu_ffn_int8 if expert_type == "swiglu" else int8.grouped_gelu_ffn_int8
        want = torch.zeros(15, 200, dtype=torch.float64, device=DEV)
        size = torch.zeros_like(want)
        one, zero = torch.ones(1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
        for t in range(15):
            for k in range(2):
                e = int(idx[t, k])
                a = int8.Int8Rows(rows.q[t : t + 1], rows.scale[t : t + 1])
                y = ffn(a, int8.Int8Weight(moe.w1_q[e : e + 1], moe.w1_scale[e : e + 1]),
                        int8.Int8Weight(moe.w2_q[e : e + 1], moe.w2_scale[e : e + 1]), zero, one, out_dtype=dtype)  # fmt: skip
                want[t] += w[t, k].double() * y[0].double()
                size[t] += (w[t, k].double() * y[0].double()).abs()
        assert_within(out.view(15, 200), want, half(dtype) * want.abs() + 4 * U * size, "layer")
    with pytest.raises(ValueError, match="no gradient"):
        moe(x)
    moe.dequantize()
    assert not moe.is_int8
    with pytest.raises(ValueError, match="8-bit rows"):
        moe(x, rows)
    if dtype == torch.float32 or expert_type == "gelu":  # 200 x 96 is no size of the bf16 grouped product
        assert torch.isfinite(moe(x)).all()


def test_block_in_int8_is_its_stages():
    torch.manual_seed(4)
    for block in (MoEBlock(256, 4, 128, 4, 2, MoEImplementation.FAST, "swiglu", norm="rms"),
                  PipelinedMoEBlock(256, 4, 128, 4, 2, None, None, num_micro_batches=2, expert_type="swiglu", norm="rms"),
                  Block(256, 4, 64, norm="rms")):  # fmt: skip
        block = block.to(DEV).to(BF16)
        x = torch.randn(2, 9, 256, device=DEV, dtype=BF16)
        with torch.no_grad():
            before = block(x)
            block.quantize_int8()
            assert isinstance(block.attn.qkv, Int8Linear) and block.attn.is_int8
            out = block(x)
            ff = block.moe if isinstance(block, PipelinedMoEBlock) else block.ff
            n1 = norm.rms_norm_int8(x, block.norm1.weight)
            a = block.attn(x, n1.rows)
            n2 = norm.rms_norm_int8(a, block.norm2.weight, residual=x, with_y=True)
            assert torch.equal(out, n2.stream + ff(n2.y, n2.rows))
            # three products in 8 bits, each value off by a 254th of its row's largest magnitude or less:
            # about 1% of a product's size; a tenth of the block's output is well outside of it, unless the
            # router changed its mind about a token
            off = (out.float() - before.float()).norm(dim=-1) / before.float().norm(dim=-1)
            assert float(off.median()) <= 0.1
    # a layer-norm block quantises its rows by itself
    block = Block(256, 4, 64).to(DEV).to(BF16)
    with torch.no_grad():
        before = block(x)
        assert float((block.quantize_int8()(x).float() - before.float()).norm()) <= 0.1 * float(before.float().norm())


def test_model_in_int8_serves_one_token_and_a_batch():
    torch.manual_seed(5)
    model = TinyModel(64, 256, 4, 128, 2, num_experts=4, top_k=2, implementation=MoEImplementation.FAST, use_moe=True,
                      expert_type="swiglu", norm="rms").to(DEV).to(BF16)  # fmt: skip
    x = torch.randn(3, 1, 64, device=DEV, dtype=BF16)
    with torch.no_grad():
        ref = model(x)
        out = model.quantize_int8()(x)
        assert out.shape == ref.shape and torch.isfinite(out).all()
        # sequences of one token do not see each other: alone and in a batch they are the same up to the
        # projections outside the blocks, which a library computes
        one = model(x[1:2])
    assert float((one.float() - out[1:2].float()).norm()) <= 4 * half(BF16) * float(out[1:2].float().norm()) + 1e-3
    assert ops.read_status() == 0


def test_refusals():
    moe = MoEFeedForward(64, 64, 4, 2, MoEImplementation.FAST).to(DEV)
    moe.world_size = 2
    with pytest.raises(ValueError, match="single rank"):
        moe.quantize_int8()
    moe.world_size = 1
    moe.quantize_int8()
    with pytest.raises(ValueError, match="int8"):
        moe.enable_fused_exchange(16)
    packed = MoEFeedForward(64, 64, 4, 2, MoEImplementation.FAST, pack_activations=True)
    with pytest.raises(ValueError, match="pack_activations"):
        packed.enable_fused_exchange(16)
    with pytest.raises(ValueError, match="FAST"):
        MoEFeedForward(64, 64, 4, 2, MoEImplementation.STANDARD, pack_activations=True)
    with pytest.raises(ValueError, match="use_moe"):
        TinyModel(64, 64, 4, 64, 1, use_moe=False, pack_activations=True)
    with pytest.raises(ValueError, match="norm must be"):
        Block(64, 4, 64, norm="batch")
    with pytest.raises(ValueError, match="without bias"):
        Int8Linear(torch.nn.Linear(8, 8).to(DEV))
    lin = Int8Linear(torch.nn.Linear(16, 8, bias=False).to(DEV)).to(BF16)
    with pytest.raises(ValueError, match="scale must be float32"):
        lin(torch.randn(2, 16, device=DEV, dtype=BF16))
    ix = routing.build_index(torch.zeros(4, 1, dtype=torch.int64, device=DEV), torch.ones(4, 1, device=DEV), 2)
    rows = int8.quantize_rows(torch.randn(4, 32, device=DEV))
    with pytest.raises(ValueError, match="q must be int8"):
        routing.permute_int8_rows(rows._replace(q=rows.q.float()), ix, 1)
    with pytest.raises(ValueError, match="scale must be float32"):
        routing.permute_int8_rows(rows._replace(scale=rows.scale[:3]), ix, 1)
    assert RMSNorm(8).weight.shape == (8,)


@pytest.mark.parametrize("expert_type", ["swiglu", "gelu"])
def test_a_layer_in_int8_follows_its_weights(expert_type):
    """Weights that are loaded, written in place or replaced after quantize_int8() are the ones that run."""
    import copy

    torch.manual_seed(6)
    kw = dict(expert_type=expert_type)
    moe, other = (MoEFeedForward(64, 96, 4, 2, MoEImplementation.FAST, **kw).to(DEV) for _ in range(2))
    x = torch.randn(2, 7, 64, device=DEV)
    with torch.no_grad():
        want = other.quantize_int8()(x)
        moe.quantize_int8()
        before = moe(x)
        buffers = [moe.w1_q, moe.w1_scale, moe.w2_q, moe.w2_scale]
        addresses = [t.data_ptr() for t in buffers]
        moe.load_state_dict(other.state_dict())
        assert torch.equal(moe(x), want) and not torch.equal(before, want)
        # in place: what a captured graph reads stays where it is
        assert [t.data_ptr() for t in (moe.w1_q, moe.w1_scale, moe.w2_q, moe.w2_scale)] == addresses
        assert torch.equal(copy.deepcopy(moe)(x), want)
        fresh = MoEFeedForward(64, 96, 4, 2, MoEImplementation.FAST, **kw).to(DEV)
        fresh.router.weight.copy_(other.router.weight)
        moe.load_state_dict({k: v.clone() for k, v in fresh.state_dict().items()}, assign=True)  # other Parameter objects
        assert torch.equal(moe(x), fresh.quantize_int8()(x))
        last = list(moe.experts.parameters())[-1]
        last.mul_(2)  # the last (or the only) second weight
        got = moe(x)
        assert torch.equal(got, moe.quantize_int8()(x)) and not torch.equal(got, fresh(x))
        # unseen by torch: the documented way is to quantise again, and a graph reads the refreshed copies
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            captured = moe(x)
        last.data.mul_(2)
        want = moe.quantize_int8()(x)
        graph.replay()
        assert torch.equal(captured, want)
        last.mul_(2)
        with pytest.raises(RuntimeError, match="weights changed"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                moe(x)
    torch.cuda.synchronize()
    assert torch.isfinite(moe.dequantize()(x)).all()


@pytest.mark.parametrize("act", ["swiglu", "gelu"])
@pytest.mark.parametrize("free", ["x", "w1", "w2", "w1 w2", "x w1 w2"])
def test_a_packed_ffn_with_frozen_parts_has_no_second_derivative(free, act):
    """A penalty on a gradient is refused whatever requires one, not counted as a constant."""
    g = torch.Generator(device=DEV).manual_seed(3)
    t = dict(x=_randn(g, 9, 256), w1=_randn(g, 1, 512 if act == "swiglu" else 256, 256, scale=1 / 16),
             w2=_randn(g, 1, 256, 256, scale=1 / 16))  # fmt: skip
    leaves = [t[name].requires_grad_(True) for name in free.split()]
    cnt = torch.tensor([9], device=DEV)
    ffn = experts.grouped_swiglu_ffn if act == "swiglu" else experts.grouped_gelu_ffn
    out = ffn(t["x"], t["w1"], t["w2"], cnt - cnt, cnt, covers_all_rows=True, packed=True)
    plain = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    grads = torch.autograd.grad(out.sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    for gradient in grads:
        with pytest.raises(RuntimeError, match="no second derivative"):
            # beside another loss, as a penalty is used
            torch.autograd.grad(gradient.float().square().sum() + sum(p.float().sum() for p in leaves), leaves,
                                retain_graph=True)  # fmt: skip
    # accumulating them without a further derivative works
    for p in leaves:
        p.grad = None
    out = ffn(t["x"], t["w1"], t["w2"], cnt - cnt, cnt, covers_all_rows=True, packed=True)
    out.sum().backward(create_graph=True)
    assert all(torch.equal(p.grad, a) for p, a in zip(leaves, plain))
    for p in leaves:
        p.grad = None


def test_packing_is_refused_where_it_has_no_effect():
    x = torch.randn(2, 9, 256, device=DEV)
    kw = dict(pack_activations=True)
    for moe, rows in ((MoEFeedForward(256, 256, 4, 2, MoEImplementation.FAST, expert_type="swiglu", **kw).to(DEV), x),
                      (MoEFeedForward(256, 256, 4, 2, MoEImplementation.FAST, **kw).to(DEV), x),
                      # 200 columns are no size of the grouped product
                      (MoEFeedForward(200, 256, 4, 2, MoEImplementation.FAST, **kw).to(DEV).to(BF16), x[..., :200].to(BF16))):
        with pytest.raises(ValueError, match="pack_activations"):
            moe(rows)
        with torch.no_grad():
            assert torch.isfinite(moe(rows)).all()
    # fp32 GELU modules under autocast are served
    moe = MoEFeedForward(256, 256, 4, 2, MoEImplementation.FAST, **kw).to(DEV)
    with torch.autocast("cuda", BF16):
        out = moe(x)
    out.float().square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in moe.experts.parameters())


@pytest.mark.parametrize("expert_type", ["swiglu", "gelu"])
def test_a_layer_in_int8_without_its_floating_point_weights(expert_type, tmp_path):
    """It runs on its 8-bit copies: the weights may be moved off the device or dropped, which frees them, and the
    layer may be copied and saved."""
    import copy

    torch.manual_seed(7)
    moe = MoEFeedForward(512, 1024, 8, 2, MoEImplementation.FAST, expert_type=expert_type).to(DEV)
    x = torch.randn(2, 7, 512, device=DEV)
    with torch.no_grad():
        want = moe.quantize_int8()(x)
        torch.save(moe, tmp_path / "moe.pt")
        loaded = torch.load(tmp_path / "moe.pt", weights_only=False)
        assert torch.equal(loaded(x), want) and torch.equal(copy.deepcopy(moe)(x), want)
        size = sum(p.numel() * p.element_size() for p in moe.experts.parameters())
        del loaded
        before = torch.cuda.memory_allocated()
        moe.experts.to("cpu")
        assert torch.equal(moe(x), want)
        assert torch.cuda.memory_allocated() <= before - size
        assert torch.equal(copy.deepcopy(moe)(x), want)
        for p in moe.experts.parameters():
            p.mul_(2)
        assert torch.equal(moe(x), want)  # not there to be read
        moe.experts.to(DEV)
        got = moe(x)
        assert torch.equal(got, moe.quantize_int8()(x)) and not torch.equal(got, want)
        moe.experts = None
        assert torch.equal(moe(x), got) and torch.equal(copy.deepcopy(moe)(x), got)
