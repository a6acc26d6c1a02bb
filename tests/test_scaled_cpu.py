"""The 8-bit token path on CPU: quantisation against an exhaustive search of the e4m3 grid, products and gradients against
64 bits and against differences, root-mean-square norm, refusals, empty operands, the layers on two and four ranks."""

import pytest
import torch

import scaled_oracle as O
from dist_utils import all_ok, assert_close, run_distributed, split
from jigsaw_b200.modules import functional as F
from jigsaw_b200.modules import scaled

ROW, SQUARE = (1, 128), (128, 128)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tensor(*shape, dtype=torch.float32, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype)


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("block", [ROW, SQUARE])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (5, 127), (3, 129), (130, 300), (257, 16)])
def test_codes_and_scales_follow_the_definition(shape, dtype, block):
    x = _tensor(*shape, dtype=dtype)
    q = F.quantize_blockwise(x, block)
    codes, scales = O.quantize(x, block == SQUARE)
    assert q.codes.dtype == torch.float8_e4m3fn and q.scales.dtype == torch.float8_e8m0fnu
    assert torch.equal(q.codes.double(), codes) and torch.equal(q.scales.double(), scales)
    assert torch.equal(q.dequantize(torch.float64), O.values(x, block == SQUARE))
    assert torch.equal(q.dequantize(torch.bfloat16).double(), q.dequantize(torch.float64)), "bf16 holds the values exactly"


def test_every_rounding_border_and_scale_border():
    grid = O.e4m3_grid()
    mid = (grid[1:] + grid[:-1]) / 2
    v = torch.cat((grid, mid, mid * (1 + 2**-20), mid * (1 - 2**-20), torch.tensor([448.0]))).float()
    v = torch.cat((v, -v))
    for k in range(0, v.numel(), 127):                           # 448 in every block: scale 1
        part = torch.cat((v[k:k + 127], torch.tensor([448.0])))
        assert torch.equal(F.quantize_blockwise(part[None]).dequantize(torch.float64)[0], O.round_e4m3(part.double()))
    top = torch.tensor([448.0, 448.0 * (1 + 2**-23), 449.0, 896.0, 897.0, 2.0**-100, 1.75 * 2.0**-120, 2.0**-130, 1e-45, 3.0e38])
    x = torch.zeros(len(top), 128)
    x[:, 5] = top
    assert torch.equal(F.quantize_blockwise(x).scales.double(), O.quantize(x)[1])


def test_not_a_number_zero_and_extremes():
    x = _tensor(6, 300)
    x[0] = 0.0
    x[1, 7], x[1, 140] = float("inf"), float("-inf")
    x[2, 3] = float("nan")
    x[3] = float("nan")
    x[4] = torch.finfo(torch.float32).min
    x[5] = 1e-44
    for block in (ROW, SQUARE):
        q = F.quantize_blockwise(x, block)
        codes, scales = O.quantize(x, block == SQUARE)
        assert torch.equal(q.scales.double(), scales)
        assert torch.equal(q.codes.double().isnan(), codes.isnan())
        assert torch.equal(q.codes.double().nan_to_num(0.5), codes.nan_to_num(0.5))


def test_quantize_shapes_strides_and_empties():
    x = _tensor(3, 4, 200)
    q = F.quantize_blockwise(x)
    assert q.shape == x.shape and q.scales.shape == (3, 4, 2)
    assert torch.equal(q.dequantize(), O.values(x.reshape(12, 200)).view(3, 4, 200).float())
    v = F.quantize_blockwise(x[0, 0])
    assert v.shape == (200,) and v.scales.shape == (2,) and torch.equal(v.dequantize(), q.dequantize()[0, 0])
    t = _tensor(200, 60).t()
    assert torch.equal(F.quantize_blockwise(t).dequantize(torch.float64), O.values(t))
    for shape in ((0, 100), (4, 0), (2, 0, 128)):
        e = F.quantize_blockwise(torch.empty(shape))
        assert e.shape == shape and e.scales.shape == (*shape[:-1], -(-shape[-1] // 128))
    assert F.quantize_blockwise(torch.empty(0, 5), SQUARE).scales.shape == (0, 1)
    assert not F.quantize_blockwise(torch.randn(2, 128, requires_grad=True)).scales.requires_grad


@pytest.mark.parametrize("call, error", [
    (lambda: F.quantize_blockwise(torch.zeros(2, 4, dtype=torch.int32)), TypeError),
    (lambda: F.quantize_blockwise(torch.zeros(2, 4).to(torch.float8_e4m3fn)), TypeError),
    (lambda: F.quantize_blockwise(torch.zeros(2, 4), (1, 64)), ValueError),
    (lambda: F.quantize_blockwise(torch.zeros(2, 3, 4), SQUARE), ValueError),
    (lambda: F.quantize_blockwise(torch.tensor(1.0)), ValueError),
    (lambda: F.BlockScaled(torch.zeros(2, 4), torch.zeros(2, 1), ROW), TypeError),
    (lambda: F.BlockScaled(torch.zeros(2, 300).to(torch.float8_e4m3fn), torch.ones(2, 2).to(torch.float8_e8m0fnu)), ValueError),
    (lambda: torch.vmap(lambda t: F.quantize_blockwise(t).codes)(torch.zeros(2, 3, 128)), NotImplementedError),
])
def test_quantize_refuses(call, error):
    with pytest.raises(error):
        call()


# ----------------------------------------------------------------------------- products
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("a_block, b_block", [(ROW, SQUARE), (ROW, ROW), (SQUARE, ROW)])
@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (7, 130, 300), (129, 16, 128)])
def test_scaled_matmul(M, N, K, a_block, b_block, out):
    a, b, bias = _tensor(M, K), _tensor(N, K, seed=1), _tensor(1, N, seed=2)[0]
    y = F.scaled_matmul(F.quantize_blockwise(a, a_block), F.quantize_blockwise(b, b_block), bias, out)
    va, vb = O.values(a, a_block == SQUARE), O.values(b, b_block == SQUARE)
    want = va @ vb.t() + bias.double()
    assert y.dtype == out
    O.assert_within(y, want, O.product_bound(va, vb, want, out) + 2.0**-23 * (want.abs() + bias.double().abs()), "product")


def test_scaled_matmul_leading_dimensions_and_empties():
    a, b = F.quantize_blockwise(_tensor(2, 3, 200)), F.quantize_blockwise(_tensor(5, 200, seed=1), SQUARE)
    assert torch.equal(F.scaled_matmul(a, b, out_dtype=torch.float32).view(6, 5),
                       F.scaled_matmul(F.quantize_blockwise(_tensor(2, 3, 200).view(6, 200)), b, out_dtype=torch.float32))
    q = lambda *s: F.quantize_blockwise(torch.empty(s))  # noqa: E731
    assert F.scaled_matmul(q(0, 8), q(4, 8)).shape == (0, 4)
    assert F.scaled_matmul(q(3, 8), q(0, 8)).shape == (3, 0)
    bias = torch.arange(4.0)
    assert torch.equal(F.scaled_matmul(q(3, 0), q(4, 0), bias, torch.float32), bias.expand(3, 4))


@pytest.mark.parametrize("call, error", [
    (lambda q: F.scaled_matmul(torch.zeros(2, 4), q(2, 4)), TypeError),
    (lambda q: F.scaled_matmul(q(2, 4), q(2, 5)), ValueError),
    (lambda q: F.scaled_matmul(q(2, 4), q(2, 2, 4)), ValueError),
    (lambda q: F.scaled_matmul(q(2, 4), q(3, 4), torch.zeros(2)), ValueError),
    (lambda q: F.scaled_matmul(q(2, 4), q(3, 4), out_dtype=torch.float64), TypeError),
])
def test_scaled_matmul_refuses(call, error):
    with pytest.raises(error):
        call(lambda *s: F.quantize_blockwise(torch.ones(s)))


# ----------------------------------------------------------------------------- linear layer
def _linear_oracle(x, w, b, g):
    vx, vw, vg = O.values(x), O.values(w, True), O.values(g)
    cx, cg = O.values_along_rows(x), O.values_along_rows(g)
    y = vx @ vw.t() + (0 if b is None else b.double())
    return (y, O.product_bound(vx, vw, y, x.dtype)), (vg @ vw, O.product_bound(vg, vw.t(), vg @ vw, x.dtype)), \
        (cg.t() @ cx, O.product_bound(cg.t(), cx.t(), cg.t() @ cx, w.dtype)), g.double().sum(0)


@pytest.mark.parametrize("dtype, wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("M, N, K, bias", [(1, 3, 5, True), (200, 130, 140, False), (130, 64, 257, True)])
def test_scaled_linear_and_its_gradients(M, N, K, bias, dtype, wdtype):
    x, w = _tensor(M, K, dtype=dtype).requires_grad_(), _tensor(N, K, dtype=wdtype, seed=1, spread=0.1).requires_grad_()
    b = _tensor(1, N, seed=2)[0].to(wdtype).requires_grad_() if bias else None
    g = _tensor(M, N, dtype=dtype, seed=3)
    y = F.scaled_linear(x, w, b)
    y.backward(g)
    (ry, by), (rx, bx), (rw, bw), rb = _linear_oracle(x.detach(), w.detach(), None if b is None else b.detach(), g)
    assert y.dtype == dtype and x.grad.dtype == dtype and w.grad.dtype == wdtype
    O.assert_within(y, ry, by + (2.0**-23 * (ry.abs() + (0 if b is None else b.double().abs()))), "y")
    O.assert_within(x.grad, rx, bx, "dx")
    O.assert_within(w.grad, rw, bw, "dw")
    if bias:
        O.assert_within(b.grad, rb, (M + 8) * 2.0**-23 * g.double().abs().sum(0) + O.half_step(wdtype) * rb.abs() + 1e-7, "db")


def test_scaled_linear_gradients_are_differences():
    """On inputs that the codes hold exactly (whole numbers up to 8, a 448 in every block fixes the scales) the layer is
    linear in each argument, so differences over whole steps are the gradients exactly."""
    g = torch.Generator().manual_seed(0)

    def whole(*s):
        t = torch.randint(-7, 8, s, generator=g).float()
        t[:, 0], t[0] = 448.0, 448.0
        return t

    x, w, go = whole(6, 9), whole(5, 9), whole(6, 5)
    loss = lambda x, w, b: (F.scaled_linear(x, w, b).double() * go.double()).sum()  # noqa: E731
    b = torch.zeros(5)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    with torch.no_grad():
        for k, t in enumerate((x, w, b)):
            for _ in range(10):
                at = tuple(int(torch.randint(1, n, (1,), generator=g)) for n in t.shape)
                hi = [v.clone() for v in (x, w, b)]
                hi[k][at] += 1.0
                assert float(loss(*hi) - loss(x, w, b)) == float(grads[k][at]), (k, at)


def test_scaled_linear_forms():
    x, w = _tensor(2, 3, 40), _tensor(8, 40, seed=1)
    y = F.scaled_linear(x, w)
    assert y.shape == (2, 3, 8) and torch.equal(y.view(6, 8), F.scaled_linear(x.view(6, 40), w))
    assert torch.equal(F.scaled_linear(x[0, 0], w), y[0, 0])
    with torch.no_grad():
        assert torch.equal(F.scaled_linear(x, F.quantize_blockwise(w, SQUARE)), y)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert F.scaled_linear(x, w).dtype == torch.bfloat16
    for shape in ((0, 40), (2, 0, 40)):
        e = torch.empty(shape, requires_grad=True)
        F.scaled_linear(e, w.requires_grad_()).sum().backward()
        assert e.grad.shape == shape and not w.grad.any()
        w = w.detach()
    assert torch.equal(F.scaled_linear(torch.empty(2, 0), torch.empty(3, 0), torch.ones(3)), torch.ones(2, 3))
    # only what wants a gradient gets one, and a second differentiation is refused
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert F.scaled_linear(x, w).requires_grad is False
    F.scaled_linear(x, wr).sum().backward()
    assert wr.grad is not None and x.grad is None
    (gx,) = torch.autograd.grad(F.scaled_linear(xr, w).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.parametrize("call, error", [
    (lambda x, w: F.scaled_linear(x, w[:, :5]), ValueError),
    (lambda x, w: F.scaled_linear(x, w[0]), ValueError),
    (lambda x, w: F.scaled_linear(x, w, torch.zeros(3)), ValueError),
    (lambda x, w: F.scaled_linear(x.double(), w), TypeError),
    (lambda x, w: F.scaled_linear(x, w.double()), TypeError),
    (lambda x, w: F.scaled_linear(x.requires_grad_(), F.quantize_blockwise(w, SQUARE)), ValueError),
    (lambda x, w: torch.vmap(lambda t: F.scaled_linear(t, w))(x[None]), NotImplementedError),
])
def test_scaled_linear_refuses(call, error):
    with pytest.raises(error):
        call(torch.ones(2, 6), torch.ones(4, 6))


# ----------------------------------------------------------------------------- norm
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("dtype", TYPES + [torch.float64])
def test_rms_norm_against_64_bits(dtype, affine, residual):
    R, C = 9, 70
    x = _tensor(R, C, dtype=dtype).requires_grad_()
    r = _tensor(R, C, dtype=dtype, seed=1).requires_grad_() if residual else None
    w = (_tensor(1, C, seed=2)[0] + 1).requires_grad_() if affine else None
    g, gs = _tensor(R, C, dtype=dtype, seed=3), _tensor(R, C, dtype=dtype, seed=4)
    out = F.distributed_rms_norm(x, w, eps=1e-5, residual=r)
    y, t = out if residual else (out, None)
    (y.double() * g.double()).sum().add((t.double() * gs.double()).sum() if residual else 0).backward()
    ry, rt, rr = O.norm(x.detach(), None if r is None else r.detach(), None if w is None else w.detach(), 1e-5)
    rx, rw = O.norm_backward(g, gs if residual else None, rt, rr, None if w is None else w.detach())
    u = 2.0**-24
    assert y.dtype == dtype
    O.assert_within(y, ry, (C + 8) * u * ry.abs() + O.half_step(dtype) * ry.abs() + 1e-7, "y")
    mag = rr * (1.0 if w is None else w.detach().double().abs()) * g.double().abs()
    mag = mag + rt.abs() * rr**3 * (mag / rr * rt.abs()).mean(1, keepdim=True)
    # the plain path rounds the gradient twice in 16 bits (through the norm, and where it meets that of the sum)
    slack = O.half_step(dtype) * (rx.abs() + (rx - (gs.double() if residual else 0)).abs())
    O.assert_within(x.grad, rx, 4 * (C + 8) * u * mag + slack + 1e-7, "dx")
    if residual:
        assert torch.equal(t.double(), rt) and torch.equal(x.grad, r.grad)
    if affine:
        O.assert_within(w.grad, rw, (R + C + 16) * 2 * u * (g.double() * rt * rr).abs().sum(0) + O.half_step(w.dtype) * rw.abs() + 1e-7, "dw")


def test_rms_norm_gradients_are_differences():
    x, r, w = (_tensor(3, 6, dtype=torch.float64, seed=k).requires_grad_() for k in (0, 1, 2))
    w = w.detach()[0].clone().requires_grad_()
    assert torch.autograd.gradcheck(lambda x, r, w: F.distributed_rms_norm(x, w, eps=1e-3, residual=r), (x, r, w))


def test_rms_norm_matches_torch_and_handles_edges():
    x = _tensor(4, 5, 32)
    ref = torch.nn.RMSNorm(32, eps=1e-6)
    torch.testing.assert_close(F.distributed_rms_norm(x, ref.weight), ref(x))
    assert torch.equal(F.distributed_rms_norm(torch.zeros(2, 8), eps=0.5), torch.zeros(2, 8))
    y, t = F.distributed_rms_norm(x.bfloat16(), residual=x)
    assert y.dtype == t.dtype == torch.float32, "the common type of input and residual"
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y, t = F.distributed_rms_norm(x.bfloat16(), residual=x.bfloat16())
    assert y.dtype == torch.float32 and t.dtype == torch.bfloat16
    assert F.distributed_rms_norm(torch.empty(0, 8)).shape == (0, 8)
    torch.testing.assert_close(torch.vmap(F.distributed_rms_norm)(x), F.distributed_rms_norm(x))


@pytest.mark.parametrize("call, error", [
    (lambda x: F.distributed_rms_norm(x, torch.ones(5)), ValueError),
    (lambda x: F.distributed_rms_norm(x, residual=torch.ones(6)), ValueError),
    (lambda x: F.distributed_rms_norm(x, eps=-1.0), ValueError),
    (lambda x: F.distributed_rms_norm(x, eps=float("nan")), ValueError),
    (lambda x: F.distributed_rms_norm(x.long()), TypeError),
    (lambda x: F.distributed_rms_norm(torch.tensor(1.0)), ValueError),
    (lambda x: F.rms_norm_quantize(x.requires_grad_()), ValueError),
    (lambda x: F.rms_norm_linear(x, torch.ones(5), torch.ones(4, 6)), ValueError),
    (lambda x: F.rms_norm_linear(x, torch.ones(6, dtype=torch.float64), torch.ones(4, 6)), TypeError),
    (lambda x: F.rms_norm_linear(x, torch.ones(6, requires_grad=True), F.quantize_blockwise(torch.ones(4, 6), SQUARE)), ValueError),
    (lambda x: torch.vmap(F.rms_norm_quantize)(x[None]).codes, NotImplementedError),
])
def test_norms_refuse(call, error):
    with pytest.raises(error):
        call(torch.ones(2, 6))


def test_rms_norm_quantize():
    x, r, w = _tensor(5, 3, 300, dtype=torch.bfloat16), _tensor(5, 3, 300, dtype=torch.bfloat16, seed=1), _tensor(1, 300, seed=2)[0]
    q, t = F.rms_norm_quantize(x, w, 1e-6, r)
    want, rt, _ = O.norm(x, r, w, 1e-6)
    assert torch.equal(t.double(), rt) and q.shape == x.shape and q.scales.shape == (5, 3, 3)
    # the norm is within 2^-18 of the 64-bit one, so a code is at most one step (2^-3 of its value, or 2^-9 scales) off
    scale = q.scales.double().repeat_interleave(128, -1)[..., :300]
    O.assert_within(q.dequantize(), want, 2.0**-4 * want.abs() * (1 + 2.0**-10) + 2.0**-10 * scale * (1 + 2.0**-10), "values")
    assert isinstance(F.rms_norm_quantize(x, w), F.BlockScaled)
    e, t = F.rms_norm_quantize(torch.empty(0, 200), residual=torch.empty(0, 200))
    assert e.scales.shape == (0, 2) and t.shape == (0, 200)


# ----------------------------------------------------------------------------- norm and linear layer in one
@pytest.mark.parametrize("residual, bias", [(True, True), (False, False)])
def test_rms_norm_linear_is_norm_then_linear(residual, bias):
    M, K, N = 150, 200, 96
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
        loss = (y * g).sum() + ((t * gs).sum() if residual else 0)
        return y, torch.autograd.grad(loss, leaves)

    (y1, g1), (y2, g2) = run(True), run(False)
    assert torch.equal(y1, y2)                    # in fp32 both quantise the same normalised rows
    for a, c in zip(g1, g2):
        torch.testing.assert_close(a, c, rtol=2e-5, atol=2e-5 * float(c.abs().max()))   # two orders of fp32 sums of 200 terms
    with torch.no_grad():
        out = F.rms_norm_linear(x, n, F.quantize_blockwise(w, SQUARE), b, 1e-6, r)
        assert torch.equal(out[0] if residual else out, y1)


def test_rms_norm_linear_partial_gradients_and_empties():
    x, r, n, w, b = _tensor(6, 20), _tensor(6, 20, seed=1), torch.ones(20), _tensor(4, 20, seed=2), torch.zeros(4)
    for k in range(5):
        leaves = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, r, n, w, b))]
        y, t = F.rms_norm_linear(leaves[0], leaves[2], leaves[3], leaves[4], residual=leaves[1])
        y.sum().backward()
        assert all((v.grad is not None) == (i == k) for i, v in enumerate(leaves)), k
    leaves = [t.clone().requires_grad_() for t in (x, r, n, w)]
    y, t = F.rms_norm_linear(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    t.sum().backward()                             # only the sum was used
    assert torch.equal(leaves[0].grad, torch.ones_like(x)) and (leaves[3].grad is None or not leaves[3].grad.any())
    y, t = F.rms_norm_linear(torch.empty(0, 20), n, w, residual=torch.empty(0, 20))
    assert y.shape == (0, 4) and t.shape == (0, 20)


# ----------------------------------------------------------------------------- layers
def _worker_layers(rank, world):
    import jigsaw_b200 as jb

    M = jb.modules
    mesh = jb.make_process_mesh({"row": 2, "col": 2} if world == 4 else {"row": 1, "col": 2})
    row, col = mesh["row"], mesh["col"]
    for eps, affine in ((1e-3, True), (None, False)):
        ref = torch.nn.RMSNorm(8, eps=eps, elementwise_affine=affine, dtype=torch.float64)
        torch.manual_seed(0)
        if affine:
            torch.nn.init.uniform_(ref.weight, 0.5, 2.0)
        layer = jb.convert.convert_to_jigsaw(torch.nn.Sequential(ref), mesh, "cpu")[0]
        assert isinstance(layer, M.DistributedRMSNorm) and all_ok(layer.local_dim == 8 // col.size() and layer.eps == eps)
        x, g = torch.randn(4, 5, 8, dtype=torch.float64), torch.randn(4, 5, 8, dtype=torch.float64)
        cuts = {0: row, 2: col}
        xl, xr = split(x, cuts).requires_grad_(), x.clone().requires_grad_()
        y, yr = layer(xl), ref(xr)
        y.backward(split(g, cuts))
        yr.backward(g)
        assert_close(y, split(yr.detach(), cuts), "forward", 1e-10, 1e-10)
        assert_close(xl.grad, split(xr.grad, cuts), "input gradient", 1e-10, 1e-10)
        if affine:
            assert_close(layer.weight.grad, split(ref.weight.grad, {0: col}), "weight gradient", 1e-10, 1e-10)
            assert layer.get_parameter_count() == 8 and layer.shard_spec()["weight"][0][1] is col
        s, t = layer(xl.detach(), residual=xl.detach())
        assert_close(s, split(ref(2 * x).detach(), cuts), "with a residual", 1e-10, 1e-10)
        assert torch.equal(t, 2 * xl.detach())
        back = layer.convert_to_torch(mesh)
        assert all_ok(back.eps == eps and all(torch.equal(back.state_dict()[k], v) for k, v in ref.state_dict().items()))
        other = jb.make_process_mesh({"row": 4, "col": 1} if world == 4 else {"row": 2, "col": 1})
        layer.reshard_parameters(mesh, other)
        assert_close(layer(split(x, {0: other["row"]})), split(ref(x).detach(), {0: other["row"]}), "re-sharded", 1e-10, 1e-10)
    # an 8-bit linear layer on a cut mesh is the undivided one: codes and scales do not depend on the cut
    ref = torch.nn.Linear(256, 64)
    torch.manual_seed(1)
    torch.nn.init.normal_(ref.weight)
    torch.nn.init.normal_(ref.bias)
    layer = M.DistributedLinear.convert_to_jigsaw(ref, mesh, "cpu", precision="fp8")
    assert "precision=fp8" in repr(layer)
    x = torch.randn(8, 256)
    want = M.scaled.scaled_linear(x, ref.weight.detach(), ref.bias.detach())
    cuts = {0: row, 1: col}
    xl = split(x, cuts).requires_grad_()
    y = layer(xl)
    assert_close(y, split(want, cuts), "8-bit linear", 1e-5, 1e-4)
    y.sum().backward()
    assert all_ok(xl.grad is not None and layer.weight.grad is not None and bool(layer.weight.grad.isfinite().all()))
    layer.reshard_parameters(mesh, mesh)
    assert layer.config.precision == "fp8"
    # norm in front of the layer, features cut: falls back to norm, then layer
    norm = M.DistributedRMSNorm(256, None, "cpu", row, col, eps=1e-6)
    h, t = norm.forward_linear(xl.detach(), layer, residual=xl.detach())
    assert_close(h, layer(norm(2 * xl.detach())), "norm in front of a cut layer", 1e-6, 1e-6)


@pytest.mark.parametrize("world", [2, 4])
def test_layers_on_a_mesh(world):
    run_distributed(_worker_layers, world)


def _worker_vit(rank, world):
    import jigsaw_b200 as jb
    from jigsaw_b200.models import ViT, ViTConfig

    mesh = jb.make_process_mesh({"row": 2, "col": 1})
    torch.manual_seed(0)
    cfg = ViTConfig(depth=2, norm="rms", linear_precision="fp8")
    model = ViT(mesh, "cpu", cfg)
    x = torch.randn(1, cfg.in_channels, *cfg.image_size, generator=torch.Generator().manual_seed(3))
    xl = split(x, {3: mesh["row"]})
    out = model(xl)
    out.square().mean().backward()
    assert all_ok(bool(out.isfinite().all()) and all(p.grad is not None and bool(p.grad.isfinite().all()) for p in model.parameters()))
    # the fused call inside the blocks is norm, then layer
    blk = model.blocks[0]
    t = torch.randn(1, 8, cfg.dim)
    h, s = blk.norm2.forward_linear(t, blk.fc1, residual=t)
    assert_close(h, blk.fc1(blk.norm2(2 * t)), "fused block", 1e-5, 1e-4)
    for bad in (dict(norm="batch"), dict(linear_precision="int8")):
        try:
            ViT(mesh, "cpu", ViTConfig(**bad))
        except ValueError:
            continue
        raise AssertionError(bad)


def test_vit_with_rms_norm_and_8_bit_products():
    run_distributed(_worker_vit, 2)


def test_names():
    import jigsaw_b200.modules as M

    for name in scaled.__all__:
        assert hasattr(scaled, name) and getattr(scaled, name).__module__ == "jigsaw_b200.modules.scaled"
    assert M.DistributedRMSNorm is scaled.DistributedRMSNorm and F.scaled_linear is scaled.scaled_linear


def test_forward_mode_is_refused():
    """A tangent would be lost without a word: the forms that have no derivative refuse it like a gradient, the others have no
    forward mode."""
    import torch.autograd.forward_ad as fw

    w = torch.ones(4, 6)
    prepared = F.quantize_blockwise(w, SQUARE)
    with fw.dual_level():
        x = fw.make_dual(torch.ones(2, 6), torch.ones(2, 6))
        gain = fw.make_dual(torch.ones(6), torch.ones(6))
        plain = torch.ones(2, 6)
        for call in (lambda: F.scaled_linear(x, prepared), lambda: F.rms_norm_linear(x, None, prepared),
                     lambda: F.rms_norm_linear(plain, gain, prepared), lambda: F.rms_norm_linear(plain, None, prepared, residual=x),
                     lambda: F.rms_norm_quantize(x), lambda: F.rms_norm_quantize(plain, gain)):
            with pytest.raises(ValueError):
                call()
        for call in (lambda: F.scaled_linear(x, w), lambda: F.rms_norm_linear(x, None, w)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
