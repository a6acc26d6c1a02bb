"""Workloads of the 8-bit token path: root-mean-square norm, block quantisation, scaled matrix products.

A case names an operator, its sizes and its types.  ``run`` computes it in plain torch operations (32-bit arithmetic,
one rounding at the end) or, where ``own`` is set, through the entry points of ``jigsaw_b200.modules.functional``.

Definitions shared by all cases.  A block of values (1 x 128 along the last axis, or 128 x 128) with the largest
finite magnitude ``a`` has the scale ``s``, the smallest power of two with ``a <= 448 s``, at least 2^-116, and 1 for
a block of zeros; its codes are ``v / s`` rounded to nearest, ties to even, in e4m3.  The norm of a sum is taken of
the sum as it is stored.
"""

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
BLOCK = 128


# ----------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the activations of a single token on their way into an 8-bit product
        {"name": "quantize one token", "op": "quantize", "rows": 1, "cols": 4096, "block": "row", "dtype": "bf16"},
        # a master weight laid out for 8-bit products, sizes that no tile divides
        {"name": "quantize weight, ragged", "op": "quantize", "rows": 11001, "cols": 4100, "block": "square", "dtype": "fp32"},
        # the norm in front of a block of a small image transformer, training, features that no vector divides
        {"name": "norm train, ragged", "op": "norm_train", "rows": 1023, "cols": 1001, "dtype": "fp32", "wdtype": "fp32"},
        # the same in a wide model on a long batch of tokens
        {"name": "norm train, wide", "op": "norm_train", "rows": 16384, "cols": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # residual stream, norm and quantisation of a single token
        {"name": "norm quantize one token", "op": "norm_quantize", "rows": 1, "cols": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # the same over a batch of long sequences
        {"name": "norm quantize batch", "op": "norm_quantize", "rows": 12000, "cols": 5120, "dtype": "bf16", "wdtype": "fp32"},
        # a single token through a prepared weight: bound by reading the weight
        {"name": "matmul one token", "op": "matmul", "rows": 1, "cols": 16384, "inner": 4096, "a": "row", "b": "square", "out": "bf16"},
        # a batch large enough for the tensor cores to be the bound
        {"name": "matmul batch", "op": "matmul", "rows": 8192, "cols": 8192, "inner": 8192, "a": "row", "b": "square", "out": "bf16"},
        # the first MLP layer of the 24 x 1024 image transformer, 4096 tokens, fp32 master weights, training
        {"name": "linear train, image tokens", "op": "linear_train", "rows": 4096, "cols": 4096, "inner": 1024, "bias": True,
         "dtype": "bf16", "wdtype": "fp32"},
        # a short ragged batch, training
        {"name": "linear train, ragged", "op": "linear_train", "rows": 1021, "cols": 2056, "inner": 1000, "bias": True,
         "dtype": "fp16", "wdtype": "fp16"},
        # residual, norm and projection of a few tokens with a prepared weight
        {"name": "norm linear, 7 tokens", "op": "norm_linear", "rows": 7, "cols": 8192, "inner": 4096, "dtype": "bf16", "wdtype": "bf16"},
        # residual, norm and projection of a wide model, training
        {"name": "norm linear train", "op": "norm_linear_train", "rows": 8192, "cols": 11008, "inner": 4096, "bias": False,
         "dtype": "bf16", "wdtype": "bf16"},
    ]


def _size(rng, low, high):
    """A whole number spread over the logarithm of ``low .. high``; one in three a multiple of 128, the others as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v > 128 and rng.random() < 0.34:
        v = v // 128 * 128
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantize", "norm_train", "norm_quantize", "matmul", "linear_train", "norm_linear", "norm_linear_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    half = "fp16" if dtype == "fp16" else "bf16"
    if op == "quantize":
        return {"op": op, "rows": _size(rng, 1, 11000), "cols": _size(rng, 64, 8192), "block": rng.choice(["row", "square"]), "dtype": dtype}
    if op in ("norm_train", "norm_quantize"):
        return {"op": op, "rows": _size(rng, 1, 12000), "cols": _size(rng, 64, 8192), "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"])}
    if op == "matmul":
        return {"op": op, "rows": _size(rng, 1, 8192), "cols": _size(rng, 16, 8192), "inner": _size(rng, 64, 8192),
                "a": rng.choice(["row", "row", "square"]), "b": rng.choice(["row", "square"]), "out": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "linear_train":
        return {"op": op, "rows": _size(rng, 1, 8192), "cols": _size(rng, 16, 8192), "inner": _size(rng, 64, 4096),
                "bias": rng.random() < 0.5, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"])}
    if op == "norm_linear":
        return {"op": op, "rows": _size(rng, 1, 512), "cols": _size(rng, 16, 16384), "inner": _size(rng, 64, 8192),
                "dtype": half, "wdtype": half}
    return {"op": op, "rows": _size(rng, 1, 8192), "cols": _size(rng, 16, 8192), "inner": _size(rng, 64, 4096),
            "bias": rng.random() < 0.5, "dtype": half, "wdtype": half}


# ----------------------------------------------------------------------------------------------- inputs
def _tokens(gen, rows, cols, dtype):
    """Activations: rows of different size and a few features far above the rest."""
    x = torch.randn(rows, cols, generator=gen, device="cuda", dtype=F32)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda", dtype=F32))
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _weight(gen, rows, cols, dtype):
    return (torch.randn(rows, cols, generator=gen, device="cuda", dtype=F32) * cols**-0.5).to(dtype)


def _gain(gen, cols, dtype):
    return (1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda", dtype=F32)).to(dtype)


def _gradient(gen, rows, cols, dtype):
    g = torch.randn(rows, cols, generator=gen, device="cuda", dtype=F32)
    return (g * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda", dtype=F32)) * 2.0**-8).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, M = case["op"], case["rows"]
    s = dict(case)
    if op == "quantize":
        make = _tokens if case["block"] == "row" else _weight
        s["x"] = make(gen, M, case["cols"], DTYPES[case["dtype"]])
        return s
    if op == "matmul":
        N, K = case["cols"], case["inner"]
        s["a_codes"], s["a_scales"] = _quantize(_tokens(gen, M, K, torch.bfloat16), case["a"])
        s["b_codes"], s["b_scales"] = _quantize(_weight(gen, N, K, torch.bfloat16), case["b"])
        return s
    dt, wdt = DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
    train = op.endswith("train")
    K = case["cols"] if op in ("norm_train", "norm_quantize") else case["inner"]
    s["x"] = _tokens(gen, M, K, dt).requires_grad_(train)
    if op != "linear_train":
        s["residual"] = _tokens(gen, M, K, dt).requires_grad_(train)
        s["gain"] = _gain(gen, K, wdt).requires_grad_(train)
    if op in ("norm_train", "norm_quantize"):
        if train:
            s["gy"], s["gsum"] = _gradient(gen, M, K, dt), _gradient(gen, M, K, dt)
        return s
    w = _weight(gen, case["cols"], K, wdt)
    if op == "norm_linear":      # a served model keeps its weight quantised
        s["w_codes"], s["w_scales"] = _quantize(w, "square")
        return s
    s["w"] = w.requires_grad_(True)
    s["bias_value"] = (0.1 * torch.randn(case["cols"], generator=gen, device="cuda")).to(wdt).requires_grad_(True) if case["bias"] else None
    s["gy"] = _gradient(gen, M, case["cols"], dt)
    if op == "norm_linear_train":
        s["gsum"] = _gradient(gen, M, K, dt)
    return s


# ----------------------------------------------------------------------------------------------- plain forms
def _block_shape(block):
    return (1, BLOCK) if block == "row" else (BLOCK, BLOCK)


def _quantize(x, block):
    """(codes, scales) of a matrix."""
    br, bc = _block_shape(block)
    R, C = x.shape
    nr, nc = -(-R // br), -(-C // bc)
    v = torch.nn.functional.pad(x.float(), (0, nc * bc - C, 0, nr * br - R)).view(nr, br, nc, bc)
    mag = v.abs()
    amax = torch.where(mag < math.inf, mag, 0.0).amax(dim=(1, 3))
    m, e = torch.frexp(amax)                                  # amax = m 2^e, 448 = 0.875 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-116)
    e = torch.where(amax == 0, 0, e).to(torch.int32)
    s = ((e + 127) << 23).view(F32)
    codes = (v / s[:, None, :, None]).view(nr * br, nc * bc)[:R, :C].to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(codes, scales, block):
    br, bc = _block_shape(block)
    s = scales.float().repeat_interleave(br, 0)[: codes.shape[0]].repeat_interleave(bc, 1)[:, : codes.shape[1]]
    return codes.float() * s


def _rounded(x, block):
    return _values(*_quantize(x, block), block)


def _along_rows(x):
    """Values of a matrix that is quantised in blocks of 128 x 1."""
    return _rounded(x.t(), "row").t()


def _norm(s, dt):
    """Sum in the type of the input, its scale factor, and the normalised rows in 32 bits."""
    total = (s["x"].detach().float() + s["residual"].detach().float()).to(dt)
    t = total.float()
    rstd = torch.rsqrt(t.square().mean(dim=1, keepdim=True) + EPS)
    return total, rstd, t * rstd * s["gain"].detach().float()


def _norm_backward(g, gsum, total, rstd, gain):
    t, w = total.float(), gain.detach().float()
    gw = g * w
    dx = rstd * gw - t * rstd.pow(3) * (gw * t).mean(dim=1, keepdim=True) + gsum.float()
    return dx, (g * t * rstd).sum(dim=0)


def _linear_backward(x, w, gy):
    dx = _rounded(gy, "row") @ _rounded(w, "square")
    dw = _along_rows(gy.float()).t() @ _along_rows(x)
    return dx, dw


def _plain(s):
    op = s["op"]
    if op == "quantize":
        codes, scales = _quantize(s["x"], s["block"])
        return {"codes": codes, "scales": scales}
    if op == "matmul":
        y = _values(s["a_codes"], s["a_scales"], s["a"]) @ _values(s["b_codes"], s["b_scales"], s["b"]).t()
        return {"y": y.to(DTYPES[s["out"]])}
    dt = DTYPES[s["dtype"]]
    if op == "linear_train":
        x, w, gy = s["x"].detach(), s["w"].detach(), s["gy"]
        y = _rounded(x, "row") @ _rounded(w, "square").t()
        dx, dw = _linear_backward(x.float(), w, gy)
        out = {"dx": dx.to(dt), "dw": dw.to(w.dtype)}
        if s["bias_value"] is not None:
            y = y + s["bias_value"].detach().float()
            out["db"] = gy.float().sum(dim=0).to(w.dtype)
        return {"y": y.to(dt), **out}
    total, rstd, h = _norm(s, dt)
    if op == "norm_train":
        dx, dw = _norm_backward(s["gy"].float(), s["gsum"], total, rstd, s["gain"])
        dx = dx.to(dt)
        return {"y": h.to(dt), "sum": total, "dx": dx, "dresidual": dx, "dgain": dw.to(s["gain"].dtype)}
    if op == "norm_quantize":
        codes, scales = _quantize(h, "row")
        return {"codes": codes, "scales": scales, "sum": total}
    if op == "norm_linear":
        y = _rounded(h, "row") @ _values(s["w_codes"], s["w_scales"], "square").t()
        return {"y": y.to(dt), "sum": total}
    w, gy = s["w"].detach(), s["gy"]
    y = _rounded(h, "row") @ _rounded(w, "square").t()
    out = {}
    if s["bias_value"] is not None:
        y = y + s["bias_value"].detach().float()
        out["db"] = gy.float().sum(dim=0).to(w.dtype)
    dh, dw = _linear_backward(h, w, gy)
    dx, dgain = _norm_backward(dh, s["gsum"], total, rstd, s["gain"])
    dx = dx.to(dt)
    return {"y": y.to(dt), "sum": total, "dx": dx, "dresidual": dx, "dgain": dgain.to(s["gain"].dtype), "dw": dw.to(w.dtype), **out}


# ----------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    from jigsaw_b200.modules import functional as F

    op = s["op"]
    if op == "quantize":
        q = F.quantize_blockwise(s["x"], _block_shape(s["block"]))
        return {"codes": q.codes, "scales": q.scales}
    if op == "matmul":
        a = F.BlockScaled(s["a_codes"], s["a_scales"], _block_shape(s["a"]))
        b = F.BlockScaled(s["b_codes"], s["b_scales"], _block_shape(s["b"]))
        return {"y": F.scaled_matmul(a, b, out_dtype=DTYPES[s["out"]])}
    if op == "norm_quantize":
        q, total = F.rms_norm_quantize(s["x"], s["gain"], eps=EPS, residual=s["residual"])
        return {"codes": q.codes, "scales": q.scales, "sum": total}
    if op == "norm_linear":
        w = F.BlockScaled(s["w_codes"], s["w_scales"], (BLOCK, BLOCK))
        y, total = F.rms_norm_linear(s["x"], s["gain"], w, eps=EPS, residual=s["residual"])
        return {"y": y, "sum": total}
    if op == "norm_train":
        y, total = F.distributed_rms_norm(s["x"], s["gain"], eps=EPS, residual=s["residual"])
        dx, dr, dw = torch.autograd.grad((y, total), (s["x"], s["residual"], s["gain"]), (s["gy"], s["gsum"]))
        return {"y": y, "sum": total, "dx": dx, "dresidual": dr, "dgain": dw}
    leaves = [s["x"], s["w"]] + ([s["bias_value"]] if s["bias_value"] is not None else [])
    if op == "linear_train":
        y = F.scaled_linear(s["x"], s["w"], s["bias_value"])
        dx, dw, *db = torch.autograd.grad(y, leaves, s["gy"])
        return {"y": y, "dx": dx, "dw": dw, **({"db": db[0]} if db else {})}
    y, total = F.rms_norm_linear(s["x"], s["gain"], s["w"], s["bias_value"], eps=EPS, residual=s["residual"])
    dx, dw, *rest = torch.autograd.grad((y, total), leaves + [s["residual"], s["gain"]], (s["gy"], s["gsum"]))
    out = {"y": y, "sum": total, "dx": dx, "dresidual": rest[-2], "dgain": rest[-1], "dw": dw}
    if len(rest) == 3:
        out["db"] = rest[0]
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------------------------- work
def work(case):
    op, M, C = case["op"], case["rows"], case["cols"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if op == "quantize":
        return {"bytes": M * C * (size[case["dtype"]] + 1), "flops": 3 * M * C}
    if op == "matmul":
        K = case["inner"]
        return {"bytes": (M + C) * K + M * C * size[case["out"]], "flops": 2 * M * C * K}
    d, w = size[case["dtype"]], size[case["wdtype"]]
    if op == "norm_train":         # x, residual, two gradients in; y, the sum and the gradient out
        return {"bytes": 7 * M * C * d + 2 * C * w, "flops": 16 * M * C}
    if op == "norm_quantize":
        return {"bytes": M * C * (3 * d + 1) + C * w, "flops": 8 * M * C}
    K = case["inner"]
    if op == "norm_linear":
        return {"bytes": 3 * M * K * d + C * K + M * C * d + K * w, "flops": 2 * M * C * K}
    bias = 2 * C * w if case["bias"] else 0
    if op == "linear_train":
        return {"bytes": 2 * M * K * d + 2 * M * C * d + 2 * C * K * w + bias, "flops": 6 * M * C * K}
    return {"bytes": 5 * M * K * d + 2 * M * C * d + 2 * C * K * w + 2 * K * w + bias, "flops": 6 * M * C * K}


# ----------------------------------------------------------------------------------------------- 64 bits
def _grid64(v):
    """To the nearest e4m3 value, ties to even: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _codes64(x, block):
    """(code values, scales) of a matrix of 64-bit numbers."""
    x = x.double()
    R, C = x.shape
    br, bc = (1 if block == "row" else 128), 128
    rows, cols = torch.arange(R, device=x.device) // br, torch.arange(C, device=x.device) // bc
    nr, nc = int(rows[-1]) + 1, int(cols[-1]) + 1
    top = torch.zeros(R, nc, dtype=F64, device=x.device).scatter_reduce_(1, cols.expand(R, C), x.abs(), "amax")
    top = torch.zeros(nr, nc, dtype=F64, device=x.device).scatter_reduce_(0, rows[:, None].expand(R, nc), top, "amax")
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0))
    for shift in (-1.0, 1.0):                                # the logarithm may be off by a step next to a power of two
        fits = top <= 448.0 * torch.exp2(e + min(shift, 0.0))
        e = torch.where(fits if shift < 0 else ~fits, e + shift, e)
    s = torch.where(top > 0, torch.exp2(e.clamp(min=-116.0)), 1.0)
    return _grid64(x / s[rows][:, cols]), s


def _through64(x, block):
    c, s = _codes64(x, block)
    br = 1 if block == "row" else 128
    return c * s[torch.arange(c.shape[0], device=c.device) // br][:, torch.arange(c.shape[1], device=c.device) // 128]


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and "codes" not in k and "scales" not in k}
    op = case["op"]
    if op == "quantize":
        c, e = _codes64(d["x"], case["block"])
        return {"codes": c, "scales": e}
    if op == "matmul":
        def full(codes, scales, block):
            r = torch.arange(codes.shape[0], device=codes.device) // (1 if block == "row" else 128)
            c = torch.arange(codes.shape[1], device=codes.device) // 128
            return codes.to(F64) * scales.to(F64)[r][:, c]

        return {"y": full(s["a_codes"], s["a_scales"], case["a"]) @ full(s["b_codes"], s["b_scales"], case["b"]).T}
    out = {}
    if op == "linear_train":
        h = d["x"]
    else:
        total = (d["x"] + d["residual"]).to(DTYPES[case["dtype"]]).double()       # the stored sum is what is normalised
        r = 1.0 / torch.sqrt((total * total).sum(1, keepdim=True) / total.shape[1] + EPS)
        h = total * r * d["gain"]
        out["sum"] = d["x"] + d["residual"]
    if op == "norm_quantize":
        c, e = _codes64(h, "row")
        return {"codes": c, "scales": e, **out}
    if op == "norm_train":
        out["y"], g = h, d["gy"]
    else:
        if op == "norm_linear":
            r8, c8 = (torch.arange(n, device="cuda") // 128 for n in s["w_codes"].shape)
            wq = s["w_codes"].to(F64) * s["w_scales"].to(F64)[r8][:, c8]
        else:
            wq = _through64(d["w"], "square")
        y = _through64(h, "row") @ wq.T
        if op == "norm_linear":
            return {"y": y, **out}
        out["y"] = y + d["bias_value"] if case["bias"] else y
        if case["bias"]:
            out["db"] = d["gy"].sum(0)
        g = _through64(d["gy"], "row") @ wq
        out["dw"] = _through64(d["gy"].T, "row") @ _through64(h.T, "row").T
        if op == "linear_train":
            return {**out, "dx": g}
    # y_i = t_i r w_i with r = (mean t^2 + eps)^(-1/2):  dL/dt_k = r w_k g_k - r^3 t_k / n sum_i g_i w_i t_i
    inner = (g * d["gain"] * total).sum(1, keepdim=True) / total.shape[1]
    dx = r * (d["gain"] * g - r * r * inner * total) + d["gsum"]
    return {**out, "dx": dx, "dresidual": dx, "dgain": (g * total * r).sum(0)}
