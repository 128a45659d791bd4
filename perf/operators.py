"""Cases of the 8-bit operators and the RMS norm: what they compute, in plain torch, and the calls
that a program makes of this package for the same result.

A case is one call (or the few calls that belong together) out of a transformer block with experts:
the norm of the residual stream with its gradient, the norm with an 8-bit output and the product
that reads it, the experts' product in 8 bits, and the pre-activations kept in 8 bits for the
backward pass.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
TINY = 2.0**-100  # rows and groups whose largest magnitude is below this are scaled as if it were this
GROUP = 128  # columns that share a scale in a packed activation
DEV = "cuda"


def listed():
    return [
        # training, the widest rows of the dispatch + combine configuration: 16384 tokens of 7168
        dict(name="norm_train", kind="norm_train", T=16384, D=7168, dtype="bf16", wdtype="bf16", residual=True),
        # training, a ragged batch of an odd width, first norm of a block (no residual yet)
        dict(name="norm_train_odd", kind="norm_train", T=1025, D=1003, dtype="f16", wdtype="f32", residual=False),
        # serving a batch of prompts at the benchmark's row width, 8-bit output for the experts
        dict(name="norm_int8", kind="norm_int8", T=4096, D=16384, dtype="bf16", wdtype="bf16", residual=True),
        # one token: norm, 8-bit output and the attention's input projection that reads it
        dict(name="norm_linear_one", kind="norm_linear", T=1, D=7168, N=21504, dtype="bf16", wdtype="bf16",
             residual=True),
        # prompts: 16 x 2048 tokens through a square projection of the 8192-wide preset
        dict(name="linear_prompt", kind="linear", T=32768, D=8192, N=8192, dtype="bf16"),
        # a serving batch of 48 sequences, one token each
        dict(name="linear_batch", kind="linear", T=48, D=7168, N=7168, dtype="bf16"),
        # nothing divides anything, fp32 in and out
        dict(name="linear_odd", kind="linear", T=130, D=1000, N=515, dtype="f32"),
        # prompts through the gate/up product of 32 local experts, about 2048 rows each
        dict(name="experts_prompt", kind="experts", T=8192, top_k=8, E=32, D=7168, N=4096, act="swiglu", dtype="bf16"),
        # eight sequences, one token each, top-8 of 64 local experts
        dict(name="experts_tokens", kind="experts", T=8, top_k=8, E=64, D=7168, N=4096, act="swiglu", dtype="bf16"),
        # a down projection of odd sizes, few experts
        dict(name="experts_odd", kind="experts", T=501, top_k=2, E=7, D=520, N=1001, act="none", dtype="f16"),
        # training: gate/up pre-activations of 65536 routed rows kept in 8 bits, and their gradient
        dict(name="packed_swiglu", kind="packed", T=65536, D=4096, act="swiglu", dtype="bf16"),
        # training: hidden width that ends inside a group, GELU experts
        dict(name="packed_gelu_odd", kind="packed", T=515, D=1000, act="gelu", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_train", "norm_int8", "norm_linear", "linear", "experts", "packed"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm_int8", "norm_linear") and dtype == "f32":
        dtype = "bf16"  # an 8-bit output is asked for where the rows themselves are 16 bits wide
    c = dict(kind=kind, dtype=dtype)
    if kind in ("norm_train", "norm_int8"):
        c["D"] = _log(rng, 64, 16384)
        c["T"] = _log(rng, 1, min(32768, 16384 * 3584 // c["D"]))
    elif kind == "norm_linear":
        c["D"], c["N"] = _log(rng, 64, 8192), _log(rng, 64, 21504)
        c["T"] = _log(rng, 1, 512)
    elif kind == "linear":
        c["D"], c["N"] = _log(rng, 64, 8192), _log(rng, 64, 8192)
        c["T"] = _log(rng, 1, 16384)
    elif kind == "experts":
        c["E"] = _log(rng, 1, 64)
        c["top_k"] = rng.randint(1, min(8, c["E"]))
        c["D"] = _log(rng, 64, 7168)
        c["act"] = rng.choice(["swiglu", "gelu", "none"])
        c["N"] = 2 * _log(rng, 32, 2048) if c["act"] == "swiglu" else _log(rng, 64, 4096)
        c["T"] = _log(rng, 1, 4096)
    else:
        c["act"] = rng.choice(["swiglu", "gelu", "none"])
        c["D"] = 2 * _log(rng, 32, 2048) if c["act"] == "swiglu" else _log(rng, 64, 7168)
        c["T"] = _log(rng, 1, min(32768, 16384 * 3584 // c["D"]))
    if kind.startswith("norm"):
        c["wdtype"] = rng.choice([dtype, "f32"])
        c["residual"] = rng.random() < 0.7
    return c


def _experts_used(case):
    """Experts that a batch reaches on average when every token takes top_k distinct ones."""
    return case["E"] * (1 - (1 - case["top_k"] / case["E"]) ** case["T"])


def work(case):
    k, T, D, e = case["kind"], case["T"], case["D"], 4 if case["dtype"] == "f32" else 2
    if k == "norm_train":
        # x, dy in, y, dx out; with a residual also that, the sum and the sum's gradient
        return {"bytes": T * D * e * (7 if case["residual"] else 4) + 8 * D, "flops": 16 * T * D}
    if k == "norm_int8":
        return {"bytes": T * D * (e * (3 if case["residual"] else 1) + 1) + 4 * D + 4 * T, "flops": 10 * T * D}
    if k == "norm_linear":
        N = case["N"]
        return {"bytes": T * D * e * (3 if case["residual"] else 1) + N * D + 4 * (N + D) + T * N * e,
                "flops": 2 * T * N * D + 10 * T * D}
    if k == "linear":
        N = case["N"]
        return {"bytes": T * D * e + N * D + 4 * N + T * N * e, "flops": 2 * T * N * D}
    if k == "experts":
        N, R = case["N"], T * case["top_k"]
        cols = N // 2 if case["act"] == "swiglu" else N
        return {"bytes": R * D * e + _experts_used(case) * N * (D + 4) + R * cols * e, "flops": 2 * R * N * D}
    cols = D // 2 if case["act"] == "swiglu" else D
    if case["act"] == "none":
        return {"bytes": 2 * T * D * e, "flops": 4 * T * D}
    return {"bytes": T * (D * e + cols * e + D * e + cols * e), "flops": 30 * T * cols}


# ---- inputs -----------------------------------------------------------------------------------
def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _stream(g, T, D, dtype):
    """Rows of a residual stream: unit variance, with one channel in a hundred ten times as large."""
    loud = 1 + 9 * (torch.rand(D, generator=g, device=DEV) < 0.01).float()
    return (torch.randn(T, D, generator=g, device=DEV) * loud).to(dtype)


def _weight8(g, *shape):
    """An int8 weight [.., N, K], rows padded to a multiple of 16 bytes, and its scale per row."""
    K = shape[-1]
    q = torch.zeros(*shape[:-1], -(-K // 16) * 16, dtype=torch.int8, device=DEV)
    q[..., :K] = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
    scale = (0.5 + torch.rand(*shape[:-1], generator=g, device=DEV)) / (73.0 * K**0.5)
    return q[..., :K], scale


def _route(case, g):
    """Rows per expert of T tokens that each take top_k distinct experts, some more popular than others."""
    E, T, K = case["E"], case["T"], case["top_k"]
    popular = torch.randn(E, generator=g, device=DEV) * 0.3
    score = popular - torch.log(-torch.log(torch.rand(T, E, generator=g, device=DEV).clamp(1e-20, 1 - 1e-7)))
    return torch.bincount(score.topk(K, -1).indices.flatten(), minlength=E)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    k, T, D, dt = case["kind"], case["T"], case["D"], DTYPES[case["dtype"]]
    st = {"case": case, "dt": dt}
    if k.startswith("norm"):
        st["x"] = _randn(g, T, D, dtype=dt) if case["residual"] else _stream(g, T, D, dt)
        st["residual"] = _stream(g, T, D, dt) if case["residual"] else None
        st["w"] = (1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(DTYPES[case["wdtype"]])
        if k == "norm_train":
            st["dy"] = _randn(g, T, D, dtype=dt)
            st["dstream"] = _randn(g, T, D, dtype=dt) if case["residual"] else None
            for name in ("x", "residual", "w"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
    if k in ("linear", "packed"):
        st["x"] = _stream(g, T, D, dt) if k == "linear" else _randn(g, T, D, dtype=dt)
    if k in ("norm_linear", "linear"):
        st["wq"], st["ws"] = _weight8(g, case["N"], D)
    if k == "packed" and case["act"] != "none":
        st["grad"] = _randn(g, T, D // 2 if case["act"] == "swiglu" else D, dtype=dt)
    if k == "experts":
        R = T * case["top_k"]
        st["x"] = _stream(g, R, D, dt)
        st["wq"], st["ws"] = _weight8(g, case["E"], case["N"], D)
        counts = _route(case, g)
        st["counts"], st["offsets"] = counts, counts.cumsum(0) - counts
        # for the plain form: the experts that have rows, and where each row lies in their padded blocks
        st["used"] = used = counts.nonzero().flatten()
        st["cap"] = cap = int(counts.max())
        rank = torch.zeros(case["E"], dtype=torch.int64, device=DEV)
        rank[used] = torch.arange(used.numel(), device=DEV)
        st["expert"] = e = torch.repeat_interleave(torch.arange(case["E"], device=DEV), counts)
        st["place"] = rank[e] * cap + torch.arange(R, device=DEV) - st["offsets"][e]
    return st


# ---- the operators in plain torch ---------------------------------------------------------------
def _quantize(y):
    """(whole values in -127..127, scale) of the rows of fp32 `y`: scale = largest magnitude / 127, rounding
    to the nearest, ties to even; a row that holds NaN or infinity has scale NaN. The quotients are taken in
    64 bits: a value next to the border between two whole numbers falls on the side that it lies on."""
    top = y.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    top = torch.where(fine, top, torch.ones_like(top)).clamp_min(TINY)
    q = torch.where(fine, torch.round(y.double() * 127.0 / top.double()).float(), torch.zeros_like(y))
    scale = top / torch.full_like(top, 127.0)  # a tensor: torch divides by a Python number through its reciprocal
    return q, torch.where(fine, scale, torch.full_like(top, math.nan))


def _plain_norm(st):
    """The stream as it is stored, 1 / rms of it (the sum of squares in 64 bits: an 8-bit output sits next to
    the borders between its values) and the normed rows in 32 bits."""
    x = st["x"].detach()
    s = x if st["residual"] is None else (x.float() + st["residual"].detach().float()).to(st["dt"])
    rstd = (1.0 / (s.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    return s, rstd, s.float() * rstd * st["w"].detach().float()


def _activation(h, act):
    if act == "swiglu":
        gate, up = h.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up
    if act == "gelu":
        return 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    return h


def _activation_grad(h, grad, act):
    if act == "swiglu":
        gate, up = h.chunk(2, -1)
        sig = torch.sigmoid(gate)
        return torch.cat([grad * up * sig * (1 + gate * (1 - sig)), grad * gate * sig], -1)
    return grad * (0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi))


def _plain(st):
    case, k, dt = st["case"], st["case"]["kind"], st["dt"]
    if k.startswith("norm"):
        s, rstd, y = _plain_norm(st)
        out = {} if st["residual"] is None else {"stream": s}
        if k == "norm_train":
            hat, dy, w = s.float() * rstd, st["dy"].float(), st["w"].detach()
            g = dy * w.float()
            dx = rstd * (g - hat * (g * hat).mean(-1, keepdim=True))
            if st["residual"] is not None:
                dx = dx + st["dstream"].float()
                out["grad_residual"] = dx.to(dt)
            return out | {"y": y.to(dt), "grad_x": dx.to(dt), "grad_w": (dy * hat).sum(0, dtype=torch.float64).to(w.dtype)}
        q, scale = _quantize(y)
        if k == "norm_int8":
            return out | {"values": (q * scale).to(dt), "scale": scale.flatten()}
        return out | {"out": (q @ st["wq"].float().t() * scale * st["ws"]).to(dt)}
    if k == "linear":
        q, scale = _quantize(st["x"].float())
        return (q @ st["wq"].float().t() * scale * st["ws"]).to(dt)
    if k == "experts":
        q, scale = _quantize(st["x"].float())
        used, cap = st["used"], st["cap"]
        blocks = torch.zeros(used.numel() * cap, case["D"], device=DEV)
        blocks[st["place"]] = q
        h = torch.bmm(blocks.view(used.numel(), cap, -1), st["wq"][used].float().transpose(1, 2))
        h = h.flatten(0, 1)[st["place"]] * scale * st["ws"][st["expert"]]
        return _activation(h, case["act"]).to(dt)
    T, D = st["x"].shape
    h = torch.nn.functional.pad(st["x"].float(), (0, -D % GROUP)).view(T, -1, GROUP)
    q, scale = _quantize(h)
    h = (q * scale).view(T, -1)[:, :D]
    if case["act"] == "none":
        return h.to(dt)
    return {"grad": _activation_grad(h, st["grad"].float(), case["act"]).to(dt),
            "hidden": _activation(h, case["act"]).to(dt)}


def _own(st):
    from fastmoe_b200.kernels import checkpoint, int8, norm

    case, k, dt = st["case"], st["case"]["kind"], st["dt"]
    if k == "norm_train":
        if st["residual"] is None:
            y = norm.rms_norm(st["x"], st["w"], EPS)
            gx, gw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
            return {"y": y, "grad_x": gx, "grad_w": gw}
        y, s = norm.add_rms_norm(st["x"], st["residual"], st["w"], EPS)
        gx, gr, gw = torch.autograd.grad((y, s), (st["x"], st["residual"], st["w"]), (st["dy"], st["dstream"]))
        return {"y": y, "stream": s, "grad_x": gx, "grad_residual": gr, "grad_w": gw}
    if k.startswith("norm"):
        r = norm.rms_norm_int8(st["x"], st["w"], EPS, residual=st["residual"])
        out = {} if st["residual"] is None else {"stream": r.stream}
        if k == "norm_int8":
            return out | {"values": int8.dequantize_rows(r.rows, dt), "scale": r.rows.scale}
        return out | {"out": int8.int8_linear(r.rows, int8.Int8Weight(st["wq"], st["ws"]), out_dtype=dt)}
    if k == "linear":
        return int8.int8_linear(int8.quantize_rows(st["x"]), int8.Int8Weight(st["wq"], st["ws"]), out_dtype=dt)
    if k == "experts":
        from fastmoe_b200.kernels import experts

        act = {"none": experts.ACT_NONE, "swiglu": experts.ACT_SWIGLU, "gelu": experts.ACT_GELU}[case["act"]]
        return int8.grouped_int8_gemm(int8.quantize_rows(st["x"]), int8.Int8Weight(st["wq"], st["ws"]), st["offsets"],
                                      st["counts"], activation=act, covers_all_rows=True, out_dtype=dt)
    packed = checkpoint.pack_activation(st["x"])
    if case["act"] == "none":
        return checkpoint.unpack_activation(packed)
    backward = checkpoint.packed_swiglu_backward if case["act"] == "swiglu" else checkpoint.packed_gelu_backward
    grad, hidden = backward(packed, st["grad"])
    return {"grad": grad, "hidden": hidden}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------
def _eight_bits(v):
    """The whole numbers that rows of `v` are held as in 8 bits, and the step that they count."""
    biggest = torch.maximum(v.abs().max(dim=-1, keepdim=True).values, torch.tensor(TINY, dtype=v.dtype, device=v.device))
    return torch.round(127 * v / biggest), biggest / 127


def exact(case, seed):
    st = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    with torch.no_grad():
        x = st["x"].to(f64)
        if kind.startswith("norm"):
            out = {}
            if st["residual"] is not None:
                # the stream is an output of its own, held in the rows' type; the norm is taken of what is held
                x = out["stream"] = (x + st["residual"].to(f64)).to(st["dt"]).to(f64)
            n = x.shape[1]
            inv = torch.rsqrt(torch.linalg.vecdot(x, x) / n + EPS).unsqueeze(1)
            w = st["w"].to(f64)
            if kind == "norm_train":
                dy = st["dy"].to(f64)
                dyw = dy * w
                dx = inv * dyw - x * inv**3 * (torch.linalg.vecdot(dyw, x) / n).unsqueeze(1)
                if st["residual"] is not None:
                    dx = dx + st["dstream"].to(f64)
                    out["grad_residual"] = dx
                out |= {"y": x * inv * w, "grad_x": dx, "grad_w": torch.einsum("td,td,tz->d", dy, x, inv)}
                return out
            q, step = _eight_bits(x * inv * w)
            if kind == "norm_int8":
                return out | {"values": q * step, "scale": step.squeeze(1)}
            return out | {"out": torch.einsum("tk,nk->tn", q, st["wq"].to(f64)) * step * st["ws"].to(f64)}
        if kind == "packed":
            h = torch.empty_like(x)
            for c in range(0, x.shape[1], GROUP):
                q, step = _eight_bits(x[:, c : c + GROUP])
                h[:, c : c + GROUP] = q * step
            if case["act"] == "none":
                return h
            h.requires_grad_(True)
            with torch.enable_grad():
                if case["act"] == "swiglu":
                    half = h.shape[1] // 2
                    hidden = torch.nn.functional.silu(h[:, :half]) * h[:, half:]
                else:
                    hidden = torch.nn.functional.gelu(h)
            (grad,) = torch.autograd.grad(hidden, h, st["grad"].to(f64))
            return {"grad": grad, "hidden": hidden.detach()}
        q, step = _eight_bits(x)
        if kind == "linear":
            return torch.einsum("tk,nk->tn", q, st["wq"].to(f64)) * step * st["ws"].to(f64)
        rows, first = [], 0
        for e, n in enumerate(st["counts"].tolist()):
            if n == 0:
                continue
            part = slice(first, first + n)
            h = q[part] @ st["wq"][e].to(f64).t() * step[part] * st["ws"][e].to(f64)
            if case["act"] == "swiglu":
                gate, up = h.split(h.shape[1] // 2, dim=1)
                h = torch.nn.functional.silu(gate) * up
            elif case["act"] == "gelu":
                h = torch.nn.functional.gelu(h)
            rows.append(h)
            first += n
        return torch.cat(rows)
