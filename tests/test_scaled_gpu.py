"""The 8-bit kernels on one GPU against oracles in 64 bits: every form of the product, ragged and strided operands, values that
are not numbers, gradients, streams, captured graphs, and rows past 32-bit offsets."""

import pytest
import torch

import scaled_oracle as O

pytestmark = pytest.mark.gpu

ROW, SQUARE = (1, 128), (128, 128)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _strict():
    from jigsaw_b200.ops import _lib, symm

    with _lib.strict_fused():
        yield
    torch.cuda.synchronize()
    symm.arena(torch.device("cuda", 0)).check_status()


def _F():
    from jigsaw_b200.modules import functional

    return functional


def _tensor(*shape, dtype=torch.float32, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))).to(dtype)


def _same(q, x, square, what):
    codes, scales = O.quantize(x, square)
    assert torch.equal(q.scales.double(), scales), f"{what}: scales"
    assert torch.equal(q.codes.double().nan_to_num(0.25), codes.nan_to_num(0.25)), f"{what}: codes"


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 100), (33, 129), (128, 128), (130, 260), (257, 1000), (40, 1023)])
def test_quantize(shape, dtype):
    from jigsaw_b200.modules.linear._scaled import _quantize_2d

    x = _tensor(*shape, dtype=dtype)
    for block in (ROW, SQUARE):
        _same(_F().quantize_blockwise(x, block), x, block == SQUARE, f"{block}")
        rows, cols, sums = _quantize_2d(x, block, cols=True, colsum=torch.float32)
        _same(rows, x, block == SQUARE, f"{block} rows")
        _same(cols, x.t(), block == SQUARE, f"{block} columns")
        ref = x.double().sum(0)
        O.assert_within(sums, ref, (shape[0] + 8) * 2.0**-24 * x.double().abs().sum(0), "column sums")
        only = _quantize_2d(x, block, rows=False, cols=True)[1]
        assert torch.equal(only.codes.view(torch.uint8), cols.codes.view(torch.uint8))


def test_quantize_norm_factors():
    """Codes of x * r * gain, in the transposed layout that the weight gradient reads."""
    from jigsaw_b200.modules.linear._scaled import _quantize_2d

    for dtype in TYPES:
        x, r, gain = _tensor(200, 300, dtype=dtype), _tensor(1, 200, seed=1)[0].abs(), _tensor(1, 300, seed=2)[0].to(dtype)
        cols = _quantize_2d(x, ROW, rows=False, cols=True, rstd=r, gain=gain)[1]
        _same(cols, ((x.float() * r[:, None]) * gain.float()).t(), False, "columns")


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_values_that_are_not_numbers(dtype):
    x = _tensor(140, 300, dtype=dtype)
    x[0] = 0.0
    x[1, 7], x[2, 140], x[3, 3] = float("inf"), float("-inf"), float("nan")
    x[4] = float("nan")
    x[5] = torch.finfo(dtype).min
    x[6] = torch.finfo(dtype).smallest_normal / 4
    x[:, 17] = float("inf")
    from jigsaw_b200.modules.linear._scaled import _quantize_2d

    for block in (ROW, SQUARE):
        for cols in (False, True):
            rows, turned, _ = _quantize_2d(x, block, cols=cols)
            _same(rows, x, block == SQUARE, "rows")
            if cols:
                _same(turned, x.t(), block == SQUARE, "columns")


def test_quantize_strided_and_unaligned_inputs():
    F = _F()
    base = _tensor(70, 520, dtype=torch.bfloat16)
    for view in (base[:, :256], base[:, 1:257], base[::2, 3:400], base.t(), base[3:4], base[:, 5:6]):
        for block in (ROW, SQUARE):
            _same(F.quantize_blockwise(view, block), view, block == SQUARE, f"{tuple(view.shape)} {view.stride()}")
    x = base.view(7, 10, 520)
    q = F.quantize_blockwise(x)
    assert q.shape == x.shape and torch.equal(q.dequantize(torch.float64).view(70, 520), O.values(base))
    _same(F.quantize_blockwise(base[:1].expand(5, 520)), base[:1].expand(5, 520), False, "expanded")


# ----------------------------------------------------------------------------- products
#: one size at least for each form of the kernel: few rows (one CTA a tile and shared tiles), narrow, shared narrow, wide,
#: pairs; one value on each axis, ends inside a tile, a k-block or a scale word
SIZES = [(1, 1, 1), (1, 4096, 1024), (3, 130, 700), (16, 20000, 272), (17, 300, 2560), (33, 64, 128), (64, 1000, 4112),
         (65, 33, 16), (128, 128, 128), (130, 140, 5), (300, 700, 5008), (129, 257, 4099), (1000, 2056, 1000), (2048, 2048, 640),
         (2047, 4099, 1040), (4200, 2600, 2176), (8200, 2300, 2064),
         (1000, 1021, 5136), (700, 1096, 5200)]


@pytest.mark.parametrize("M, N, K", SIZES)
def test_scaled_matmul(M, N, K):
    F = _F()
    a, b, bias = _tensor(M, K), _tensor(N, K, seed=1, spread=0.2), _tensor(1, N, seed=2)[0]
    for k, (ab, bb, out, use_bias) in enumerate([(ROW, SQUARE, torch.bfloat16, True), (ROW, ROW, torch.float32, False),
                                                 (SQUARE, ROW, torch.float16, True), (SQUARE, SQUARE, torch.float32, True)]):
        qa, qb = F.quantize_blockwise(a, ab), F.quantize_blockwise(b, bb)
        bt = bias.to([torch.float32, torch.float32, torch.float16, torch.bfloat16][k]) if use_bias else None
        y = F.scaled_matmul(qa, qb, bt, out)
        va, vb = qa.dequantize(torch.float64), qb.dequantize(torch.float64)
        want = va @ vb.t() + (0 if bt is None else bt.double())
        extra = 0 if bt is None else 2.0**-23 * (want.abs() + bt.double().abs())
        assert y.dtype == out and y.is_contiguous()
        # fp16 overflows to infinity where the value does
        fits = want.abs() <= 65000 if out == torch.float16 else torch.ones_like(want, dtype=torch.bool)
        O.assert_within(y[fits], want[fits], (O.product_bound(va, vb, want, out) + extra)[fits], f"{ab} {bb} {out}")


def test_scaled_matmul_is_reproducible_and_close_to_fp32_sums():
    """The same bits on every run (parts of a tile are added in a fixed order), and fp32 results as good as an fp32 sum of
    2048 terms, however long the row: truncation of each of 64 additions in TMEM (2^-23 each, in one direction) against the
    root mean square of the terms."""
    F = _F()
    for M, N, K in ((5, 700, 8192), (200, 300, 8192), (3000, 3000, 8192)):
        a, b = F.quantize_blockwise(_tensor(M, K, spread=0.0)), F.quantize_blockwise(_tensor(N, K, seed=1, spread=0.0))
        y = F.scaled_matmul(a, b, out_dtype=torch.float32)
        want = a.dequantize(torch.float64) @ b.dequantize(torch.float64).t()
        assert float((y.double() - want).norm() / want.norm()) < 64 * 2.0**-23 * 2048**0.5 / 8192**0.5
        for _ in range(3):
            assert torch.equal(y, F.scaled_matmul(a, b, out_dtype=torch.float32))


def test_scaled_matmul_operands_in_any_layout():
    """Codes and scales that a user made: contiguous with rows of any length, transposed scales, views with gaps, odd addresses."""
    F = _F()
    M, N, K = 70, 90, 1000
    qa, qb = F.quantize_blockwise(_tensor(M, K)), F.quantize_blockwise(_tensor(N, K, seed=1), SQUARE)
    want = F.scaled_matmul(qa, qb, out_dtype=torch.float32)

    def layouts(q):
        c, s, blk = q.codes, q.scales, q.block
        yield F.BlockScaled(c.clone(memory_format=torch.contiguous_format), s.contiguous(), blk)
        wide = torch.zeros(c.shape[0], 1040, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        wide[:, 16:1016].view(torch.uint8).copy_(c.view(torch.uint8))
        yield F.BlockScaled(wide[:, 16:1016], s, blk)
        wide[:, 3:1003].view(torch.uint8).copy_(c.view(torch.uint8))
        yield F.BlockScaled(wide[:, 3:1003], s.t().contiguous().t(), blk)
        yield F.BlockScaled(c.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn) if c.dim() == 2 else c, s, blk)

    for a in layouts(qa):
        assert torch.equal(F.scaled_matmul(a, qb, out_dtype=torch.float32), want)
    for b in layouts(qb):
        assert torch.equal(F.scaled_matmul(qa, b, out_dtype=torch.float32), want)
    bias = _tensor(1, 2 * N, seed=3)[0]
    assert torch.equal(F.scaled_matmul(qa, qb, bias[::2], torch.float32), F.scaled_matmul(qa, qb, bias[::2].contiguous(), torch.float32))


def test_scaled_matmul_not_a_number_stays_in_its_row():
    F = _F()
    for M, N in ((4, 200), (200, 300), (3000, 3000)):
        x, w = _tensor(M, 512), _tensor(N, 512, seed=1)
        clean = F.scaled_matmul(F.quantize_blockwise(x), F.quantize_blockwise(w), out_dtype=torch.float32)
        x[M // 2, 77] = float("inf")
        w[N // 3, 300] = float("nan")
        y = F.scaled_matmul(F.quantize_blockwise(x), F.quantize_blockwise(w), out_dtype=torch.float32)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[M // 2], bad[:, N // 3] = True, True
        assert torch.equal(y.isnan(), bad) and torch.equal(y[~bad], clean[~bad])


def test_empty_operands_on_cuda():
    F = _F()
    q = lambda *s: F.quantize_blockwise(torch.empty(s, device="cuda"))  # noqa: E731
    assert F.scaled_matmul(q(0, 8), q(4, 8)).shape == (0, 4) and F.scaled_matmul(q(3, 8), q(0, 8)).shape == (3, 0)
    assert torch.equal(F.scaled_matmul(q(3, 0), q(4, 0), torch.ones(4, device="cuda")).float(), torch.ones(3, 4, device="cuda"))
    x, w = torch.empty(0, 8, device="cuda", requires_grad=True), torch.ones(4, 8, device="cuda", requires_grad=True)
    F.scaled_linear(x, w).sum().backward()
    assert x.grad.shape == (0, 8) and not w.grad.any()
    y, t = F.rms_norm_linear(x.detach(), None, w.detach(), residual=x.detach())
    assert y.shape == (0, 4) and t.shape == (0, 8) and F.distributed_rms_norm(x.detach()).shape == (0, 8)


def test_rows_past_32_bit_offsets():
    """2.3e9 elements: the last rows of codes, scales and products are those of the last rows alone."""
    F = _F()
    R, C = 70016, 33024
    x = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    x[:-40].fill_(1.0)
    x[-40:] = _tensor(40, C, dtype=torch.bfloat16)
    q = F.quantize_blockwise(x)
    _same(F.BlockScaled(q.codes[-40:], q.scales[-40:], ROW), x[-40:], False, "rows")
    y, t = F.distributed_rms_norm(x[:, :32768], residual=x[:, :32768])
    want, rt, _ = O.norm(x[-40:, :32768], x[-40:, :32768], None, 1e-6)
    assert torch.equal(t[-40:].double(), rt)
    O.assert_within(y[-40:], want, (2.0**-18 + O.half_step(torch.bfloat16)) * want.abs() + 1e-30, "norm")
    del y, t
    w = F.quantize_blockwise(_tensor(33024, 128, seed=1), SQUARE)
    a = F.BlockScaled(q.codes[:, :128], q.scales[:, :1], ROW)
    out = F.scaled_matmul(a, w)
    tail = F.scaled_matmul(F.BlockScaled(q.codes[-256:, :128], q.scales[-256:, :1], ROW), w)
    assert torch.equal(out[-256:], tail)


@pytest.mark.parametrize("M, N", [(5, 300), (130, 140), (1100, 9700)])
def test_scaled_matmul_long_rows_of_one_sign(M, N):
    """Additions into TMEM truncate, each by up to 2^-23 of the sum so far and all in one direction: at most 512 of them (16384
    terms, 32 at a time) before the parts are added with rounding, at most 8 parts here, so 2^-14 + 8 * 2^-24 of the result, and
    one rounding of the result.  Summed in one go the 4096 additions could lose 2^-11, a whole half step of fp16."""
    F = _F()
    K = 131072 if M < 1000 else 32768
    g = torch.Generator(device="cuda").manual_seed(0)
    a = F.quantize_blockwise(torch.rand(M, K, generator=g, device="cuda") * 2.0**-8 + 2.0**-8)
    b = F.quantize_blockwise(torch.rand(N, K, generator=g, device="cuda") + 1.0, SQUARE)
    want = torch.cat([a.dequantize(torch.float64) @ part.t() for part in b.dequantize(torch.float64).split(2048)], dim=1)
    for out in (torch.float16, torch.bfloat16):
        y = F.scaled_matmul(a, b, out_dtype=out)
        O.assert_within(y, want, (2.0**-14 + 2.0**-21 + O.half_step(out) * (1 + 2.0**-13)) * want, str(out))


# ----------------------------------------------------------------------------- linear layer
@pytest.mark.parametrize("dtype, wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float16)])
@pytest.mark.parametrize("M, N, K, bias", [(1, 1, 1, True), (1, 4096, 512, False), (200, 130, 140, True), (1021, 2056, 1000, True),
                                           (4096, 1024, 512, False)])
def test_scaled_linear_and_its_gradients(M, N, K, bias, dtype, wdtype):
    F = _F()
    x, w = _tensor(M, K, dtype=dtype).requires_grad_(), _tensor(N, K, dtype=wdtype, seed=1, spread=0.1).requires_grad_()
    b = _tensor(1, N, seed=2)[0].to(wdtype).requires_grad_() if bias else None
    g = (_tensor(M, N, seed=3) / 64).to(dtype)
    y = F.scaled_linear(x, w, b)
    y.backward(g)
    xd, wd = x.detach(), w.detach()
    vx, vw, vg, cx, cg = O.values(xd), O.values(wd, True), O.values(g), O.values_along_rows(xd), O.values_along_rows(g)
    bd = 0.0 if b is None else b.detach().double()
    ry = vx @ vw.t() + bd
    O.assert_within(y, ry, O.product_bound(vx, vw, ry, dtype) + 2.0**-23 * (ry.abs() + abs(bd)), "y")
    rx, rw = vg @ vw, cg.t() @ cx
    O.assert_within(x.grad, rx, O.product_bound(vg, vw.t(), rx, dtype), "dx")
    O.assert_within(w.grad, rw, O.product_bound(cg.t(), cx.t(), rw, wdtype), "dw")
    if bias:
        rb = g.double().sum(0)
        O.assert_within(b.grad, rb, (M + 8) * 2.0**-24 * g.double().abs().sum(0) + O.half_step(wdtype) * rb.abs() + 2.0**-25, "db")


def test_scaled_linear_gradients_are_differences():
    F = _F()
    g = torch.Generator().manual_seed(0)

    def whole(*s):
        t = torch.randint(-7, 8, s, generator=g).float()
        t[:, 0], t[0] = 448.0, 448.0
        return t.cuda()

    x, w, go, b = whole(6, 9), whole(5, 9), whole(6, 5), torch.zeros(5, device="cuda")
    loss = lambda x, w, b: (F.scaled_linear(x, w, b).double() * go.double()).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    with torch.no_grad():
        for k, t in enumerate((x, w, b)):
            for _ in range(6):
                at = tuple(int(torch.randint(1, n, (1,), generator=g)) for n in t.shape)
                hi = [v.clone() for v in (x, w, b)]
                hi[k][at] += 1.0
                assert float(loss(*hi) - loss(x, w, b)) == float(grads[k][at]), (k, at)


def test_scaled_linear_forms_and_dispatch():
    from jigsaw_b200.ops import _lib

    F = _F()
    x, w, b = _tensor(2, 3, 256, dtype=torch.bfloat16), _tensor(64, 256, seed=1), _tensor(1, 64, seed=2)[0]
    _lib.dispatch_counts(reset=True)
    before = _lib.LAUNCHES
    y = F.scaled_linear(x, w, b)
    assert _lib.LAUNCHES == before + 3 and y.shape == (2, 3, 64) and y.dtype == torch.bfloat16
    with torch.autocast("cuda", dtype=torch.float16):
        assert F.scaled_linear(x, w, b).dtype == torch.float16
    with torch.no_grad():
        prepared = F.quantize_blockwise(w, SQUARE)
        before = _lib.LAUNCHES
        assert torch.equal(F.scaled_linear(x, prepared, b), y) and _lib.LAUNCHES == before + 2
    strided = _tensor(6, 512, dtype=torch.bfloat16)[:, ::2]
    assert torch.equal(F.scaled_linear(strided, w, b), F.scaled_linear(strided.contiguous(), w, b))
    # gradients of a broadcast input and of a weight that two layers share
    xe = _tensor(1, 256, dtype=torch.float32).requires_grad_()
    wr = w.clone().requires_grad_()
    out = F.scaled_linear(xe.expand(4, 256), wr, b)
    out = F.scaled_linear(torch.cat((out,) * 4, dim=1), wr)
    out.sum().backward()
    assert xe.grad.shape == (1, 256) and bool(wr.grad.isfinite().all())
    (gx,) = torch.autograd.grad(F.scaled_linear(xe, w, b).sum(), xe, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    # weight only, input only, bias only
    for k in range(3):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x.float(), w, b))]
        F.scaled_linear(*leaves).sum().backward()
        assert [v.grad is not None for v in leaves] == [i == k for i in range(3)]
    counts = _lib.dispatch_counts()
    assert counts["scaled_linear"]["fused"] > 5 and all(v["fallback"] == 0 for v in counts.values())
    with pytest.raises(_lib.FusedPathDeclined):
        F.rms_norm_quantize(torch.ones(2, 40000, device="cuda"))
    with _lib.strict_fused(False):                # longer rows than the norm kernels hold: torch operations
        q = F.rms_norm_quantize(torch.ones(2, 40000, device="cuda"))
        assert torch.equal(q.dequantize(), torch.ones(2, 40000, device="cuda"))
        xl = torch.ones(2, 40000, device="cuda", requires_grad=True)
        F.rms_norm_linear(xl, None, torch.ones(3, 40000, device="cuda")).sum().backward()
        assert xl.grad is not None


# ----------------------------------------------------------------------------- norm
def _check_norm(R, C, dtype, wdtype, residual, make=None):
    F = _F()
    x = (make or _tensor)(R, C, dtype=dtype).requires_grad_()
    r = (make or _tensor)(R, C, dtype=dtype, seed=1).requires_grad_() if residual else None
    w = (_tensor(1, C, seed=2)[0] + 1).to(wdtype).requires_grad_() if wdtype is not None else None
    g, gs = _tensor(R, C, dtype=dtype, seed=3), _tensor(R, C, dtype=dtype, seed=4)
    out = F.distributed_rms_norm(x, w, eps=1e-5, residual=r)
    leaves = [t for t in (x, r, w) if t is not None]
    grads = dict(zip("xrw" if residual else "xw", torch.autograd.grad(out if residual else (out,), leaves, (g, gs) if residual else (g,))))
    y = out[0] if residual else out
    ry, rt, rr = O.norm(x.detach(), None if r is None else r.detach(), None if w is None else w.detach(), 1e-5)
    rx, rw = O.norm_backward(g, gs if residual else None, rt, rr, None if w is None else w.detach())
    u, h, tiny = 2.0**-24, O.half_step(dtype), torch.finfo(dtype).smallest_normal
    # squares: 32 fp32 additions a thread, the rest in fp64; then r, two products, one rounding
    O.assert_within(y, ry, (40 * u + h) * ry.abs() + tiny, f"y {R} {C} {dtype}")
    wg = g.double().abs() * (1.0 if w is None else w.detach().double().abs())
    mag = rr * (wg + rt.abs() * rr.square() * (wg * rt.abs()).mean(1, keepdim=True))
    O.assert_within(grads["x"], rx, 100 * u * mag + 4 * u * (gs.double().abs() if residual else 0) + h * rx.abs() + tiny, f"dx {R} {C} {dtype}")
    if residual:
        assert torch.equal(out[1].double(), rt) and torch.equal(grads["x"], grads["r"])
    if w is not None:
        bound = (R + 40) * u * (g.double() * rt * rr).abs().sum(0) + O.half_step(wdtype) * rw.abs()
        O.assert_within(grads["w"], rw, bound + tiny, f"dw {R} {C} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R, C", [(1, 1), (1, 4096), (3, 7), (5, 64), (9, 513), (700, 256), (300, 512), (1023, 1001), (130, 1024), (200, 1030),
                                  (2, 8192), (310, 4096), (5, 8200), (3, 16384), (2, 20000), (2, 32768)])
def test_rms_norm(R, C, dtype):
    _check_norm(R, C, dtype, dtype, True)
    _check_norm(R, C, dtype, torch.float32, False)
    _check_norm(R, C, dtype, None, True)


def test_rms_norm_strided_and_unaligned_inputs():
    def view(step, shift):
        def make(R, C, dtype, seed=0):
            return _tensor(R * step, C + 9, dtype=dtype, seed=seed)[::step, shift:shift + C]
        return make

    for step, shift in ((1, 8), (2, 8), (1, 1), (3, 5)):
        for R, C in ((40, 256), (300, 1280), (1, 4096)):
            _check_norm(R, C, torch.bfloat16, torch.bfloat16, True, view(step, shift))
    F = _F()
    t = _tensor(60, 40).t()
    torch.testing.assert_close(F.distributed_rms_norm(t), F.distributed_rms_norm(t.contiguous()))


def test_rms_norm_not_a_number_and_zero_rows():
    F = _F()
    x = _tensor(300, 768, dtype=torch.bfloat16)
    x[3], x[5, 100], x[7, 2] = 0.0, float("inf"), float("nan")
    y = F.distributed_rms_norm(x, eps=1e-6)
    ref = x.float() * (x.float().square().mean(1, keepdim=True) + 1e-6).rsqrt()
    assert torch.equal(y.isnan(), ref.isnan()) and not y[3].any()
    q = F.rms_norm_quantize(x, eps=1e-6)
    assert torch.equal(q.codes.float().isnan(), ref.isnan()) and torch.equal(q.scales[3].float(), torch.ones(6, device="cuda"))
    assert not F.distributed_rms_norm(torch.zeros(2, 64, device="cuda"), eps=0.0).isnan().logical_not().any(), "0 / 0"


@pytest.mark.parametrize("R, C", [(1, 4096), (1, 100), (7, 8192), (200, 300), (1000, 1000), (150, 5120), (2, 20000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm_quantize(R, C, dtype):
    F = _F()
    x, r, w = _tensor(R, C, dtype=dtype), _tensor(R, C, dtype=dtype, seed=1), _tensor(1, C, seed=2)[0]
    q, t = F.rms_norm_quantize(x, w, 1e-6, r)
    want, rt, _ = O.norm(x, r, w, 1e-6)
    assert torch.equal(t.double(), rt)
    codes, scales = O.quantize(want)
    # the kernel's norm is within 40 2^-24 of the 64-bit one: a code differs only where that crosses a rounding border, and
    # then by one step
    step = 2.0**-3 * want.abs() + 2.0**-9 * scales.repeat_interleave(128, 1)[:, :C]
    values = codes * scales.repeat_interleave(128, 1)[:, :C]
    off = (q.dequantize(torch.float64) - values).abs()
    assert bool((off <= step * 1.01).all()) and float((off > 0).double().mean()) < 1e-4
    assert isinstance(F.rms_norm_quantize(x, w), F.BlockScaled)


@pytest.mark.parametrize("residual, bias", [(True, True), (False, False)])
@pytest.mark.parametrize("M, N, K", [(1, 128, 64), (150, 96, 200), (1030, 512, 1024)])
def test_rms_norm_linear_is_norm_then_linear(M, N, K, residual, bias):
    F = _F()
    x = _tensor(M, K).requires_grad_()
    r = _tensor(M, K, seed=1).requires_grad_() if residual else None
    w, n = _tensor(N, K, seed=2).requires_grad_(), (_tensor(1, K, seed=3)[0] + 1).requires_grad_()
    b = _tensor(1, N, seed=4)[0].requires_grad_() if bias else None
    g, gs = _tensor(M, N, seed=5), _tensor(M, K, seed=6)
    leaves = [t for t in (x, n, w, r, b) if t is not None]

    def run(fused):
        if fused:
            out = F.rms_norm_linear(x, n, w, b, 1e-6, r)
            y, t = out if residual else (out, None)
        else:
            out = F.distributed_rms_norm(x, n, None, 1e-6, r)
            h, t = out if residual else (out, None)
            y = F.scaled_linear(h, w, b)
        return y, torch.autograd.grad((y, t) if residual else (y,), leaves, (g, gs) if residual else (g,))

    (y1, g1), (y2, g2) = run(True), run(False)
    # in fp32 both quantise the same rows in the forward pass, and their gradients meet the same kernels
    assert torch.equal(y1, y2) and all(torch.equal(a, c) for a, c in zip(g1, g2))
    with torch.no_grad():
        out = F.rms_norm_linear(x, n, F.quantize_blockwise(w, SQUARE), b, 1e-6, r)
        assert torch.equal(out[0] if residual else out, y1)


def test_rms_norm_linear_partial_gradients():
    F = _F()
    x, r, n, w, b = _tensor(6, 20), _tensor(6, 20, seed=1), torch.ones(20, device="cuda"), _tensor(4, 20, seed=2), torch.zeros(4, device="cuda")
    for k in range(5):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, r, n, w, b))]
        y, t = F.rms_norm_linear(leaves[0], leaves[2], leaves[3], leaves[4], residual=leaves[1])
        y.sum().backward()
        assert all((v.grad is not None) == (i == k) for i, v in enumerate(leaves)), k
    leaves = [t.clone().requires_grad_() for t in (x, r, n, w)]
    y, t = F.rms_norm_linear(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    t.sum().backward()
    assert torch.equal(leaves[0].grad, torch.ones_like(x)) and (leaves[3].grad is None or not leaves[3].grad.any())
    # no weight of the norm, no residual
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    F.rms_norm_linear(xr, None, wr, b).sum().backward()
    assert bool(xr.grad.isfinite().all()) and bool(wr.grad.isfinite().all())


# ----------------------------------------------------------------------------- streams, graphs, layers
def _step(F, x, r, n, w, b, g, gs):
    y, t = F.rms_norm_linear(x, n, w, b, residual=r)
    return (y, t, *torch.autograd.grad((y, t), (x, r, n, w, b), (g, gs)))


def _step_inputs(seed=0):
    leaves = [_tensor(300, 256, dtype=torch.bfloat16, seed=seed), _tensor(300, 256, dtype=torch.bfloat16, seed=seed + 1),
              _tensor(1, 256, seed=seed + 2)[0], _tensor(384, 256, seed=seed + 3), _tensor(1, 384, seed=seed + 4)[0]]
    return [t.requires_grad_() for t in leaves] + [_tensor(300, 384, dtype=torch.bfloat16, seed=seed + 5), _tensor(300, 256, dtype=torch.bfloat16, seed=seed + 6)]


def test_steps_on_two_streams_at_once():
    F = _F()
    ins = [_step_inputs(0), _step_inputs(50)]
    want = [_step(F, *i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(_step(F, *ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


def test_captured_steps():
    """Forward and backward in two graphs that share nothing: each replays on new inputs, in any order."""
    F = _F()
    steps = []
    for seed in (0, 50):
        ins = _step_inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                _step(F, *ins)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(F, *ins)
        steps.append((ins, graph, out))
    for k in (0, 1, 1, 0):
        ins, graph, out = steps[k]
        with torch.no_grad():
            for t in ins:
                t.copy_(t * 1.25)
        graph.replay()
        want = _step(F, *ins)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    del steps


def test_layers_and_model():
    import jigsaw_b200 as jb
    from jigsaw_b200.ops import _lib

    norm = jb.modules.DistributedRMSNorm(256, None, torch.device("cuda", 0), None, None)
    x = _tensor(4, 33, 256, dtype=torch.bfloat16)
    before = _lib.LAUNCHES
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = norm(x)
    assert _lib.LAUNCHES == before + 1 and y.dtype == torch.float32
    ref = torch.nn.RMSNorm(256, device="cuda")
    want = torch.nn.functional.rms_norm(x.float(), (256,), ref.weight, torch.finfo(torch.bfloat16).eps)
    torch.testing.assert_close(y, want, rtol=1e-5, atol=1e-5)


def test_calls_inside_other_machinery():
    """Inference mode, recomputation, batched gradients, forward mode, lazily negated inputs."""
    import torch.autograd.forward_ad as fw
    from torch.utils.checkpoint import checkpoint

    F = _F()
    x, w, n = _tensor(40, 256, dtype=torch.bfloat16), _tensor(64, 256, seed=1), _tensor(1, 256, seed=2)[0]
    prepared = F.quantize_blockwise(w, SQUARE)
    with torch.inference_mode():
        assert torch.equal(F.scaled_linear(x, w), F.scaled_linear(x, prepared))
        assert torch.equal(F.rms_norm_linear(x, n, w, residual=x)[0], F.rms_norm_linear(x, n, prepared, residual=x)[0])
        assert F.distributed_rms_norm(x, n).is_inference()
    grads = []
    for again in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, n, w)]
        f = lambda x, n, w: F.rms_norm_linear(x, n, w, residual=x)  # noqa: E731
        y, t = checkpoint(f, *leaves, use_reentrant=False) if again else f(*leaves)
        (y.float().sum() + t.float().sum()).backward()
        grads.append([v.grad for v in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    for f in (lambda x: F.scaled_linear(x, w), lambda x: F.distributed_rms_norm(x, n), lambda x: F.rms_norm_linear(x, n, w)):
        leaf = x.float().requires_grad_()
        y = f(leaf)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, torch.ones(3, *y.shape, device="cuda"), is_grads_batched=True)
    with fw.dual_level():
        dual = fw.make_dual(x.float(), torch.ones(40, 256, device="cuda"))
        for f in (lambda: F.scaled_linear(dual, prepared), lambda: F.rms_norm_linear(dual, n, prepared), lambda: F.rms_norm_quantize(dual)):
            with pytest.raises(ValueError):
                f()
        for f in (lambda: F.scaled_linear(dual, w), lambda: F.rms_norm_linear(dual, n, w), lambda: F.distributed_rms_norm(dual, n)):
            with pytest.raises(RuntimeError):
                f()
    z = torch.complex(_tensor(40, 1), _tensor(40, 1, seed=4)).conj().imag
    assert z.is_neg()
    with pytest.raises(Exception, match="outside the coverage"):
        F.quantize_blockwise(z)
    from jigsaw_b200.ops import _lib

    with _lib.strict_fused(False):
        _same(F.quantize_blockwise(z), z.resolve_neg(), False, "negated")


def test_quantize_few_very_long_rows():
    """More block columns than the grid of the kernel for few rows holds."""
    F = _F()
    C = 65535 * 1024 + 300
    x = torch.zeros(2, C, dtype=torch.bfloat16, device="cuda")
    x[:, -400:] = _tensor(2, 400, dtype=torch.bfloat16)
    q = F.quantize_blockwise(x)
    at = (C - 400) // 128 * 128
    tail = F.BlockScaled(q.codes[:, at:], q.scales[:, at // 128:], ROW)
    _same(tail, x[:, at:], False, "tail")
    assert not q.codes[:, :at].view(torch.uint8).any() and bool((q.scales[:, : at // 128].view(torch.uint8) == 127).all())
