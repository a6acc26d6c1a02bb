"""Gradients of the norm and of the 8-bit linear layers on the kernels, in the forms in which autograd hands them over."""

import pytest
import torch

import scaled_oracle as O
from dist_utils import run_distributed

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.fixture(autouse=True)
def _strict():
    from jigsaw_b200.ops import _lib, symm

    with _lib.strict_fused():
        yield
    torch.cuda.synchronize()
    symm.arena(torch.device("cuda", 0)).check_status()


def _F():
    from jigsaw_b200.modules import functional as F

    return F


def _tensor(*shape, dtype=torch.float32, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda") * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))
    return x.to(dtype)


def _calls(columns):
    """The three operators with gradients, their outputs ``[40, columns]`` (the second also gives the sum)."""
    F = _F()
    x, r, w, n, b = (_tensor(*s, seed=k) for k, s in enumerate(((40, 64), (40, 64), (columns, 64), (64,), (columns,))))
    t = _tensor(40, columns, seed=7)
    return {
        "linear": ((x, w, b), lambda x, w, b: (F.scaled_linear(x, w, b),)),
        "norm linear": ((x, n, w, b, r), lambda x, n, w, b, r: F.rms_norm_linear(x, n, w, b, residual=r)),
        "norm": ((t, t + 1, w[:, 0].clone()), lambda t, r, w: F.distributed_rms_norm(t, w, eps=0.1, residual=r)),
    }


@pytest.mark.parametrize("columns", [1, 24])
@pytest.mark.parametrize("name", ["linear", "norm linear", "norm"])
def test_lazily_negated_gradients(name, columns):
    """The gradient of an output that becomes the imaginary part of a conjugated number arrives with its sign in a flag; with
    one column its memory is read in place."""
    inputs, f = _calls(columns)[name]
    leaves = [t.clone().requires_grad_() for t in inputs]

    def grads(conjugate):
        loss = 0.0
        for k, y in enumerate(f(*leaves)):
            z = torch.complex(torch.zeros_like(y), y)
            z = z.conj().imag if conjugate else -z.imag
            loss = loss + (z * _tensor(*y.shape, seed=20 + k)).sum()
        return torch.autograd.grad(loss, leaves)

    for got, want in zip(grads(True), grads(False)):
        assert bool(want.any()) and torch.equal(got, want)
    # a negated gradient that lies in memory like an ordinary one
    outs = f(*leaves)
    gs = [_tensor(*y.shape, seed=20 + k) for k, y in enumerate(outs)]
    got = torch.autograd.grad(outs, leaves, [torch._neg_view(g) for g in gs], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(outs, leaves, [-g for g in gs])))


@pytest.mark.parametrize("name", ["linear", "norm linear", "norm"])
def test_gradients_that_are_zeros_without_memory(name):
    inputs, f = _calls(24)[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    outs = f(*leaves)
    grads = torch.autograd.grad(outs, leaves, [torch._efficientzerotensor(y.shape, dtype=y.dtype, device=y.device) for y in outs])
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))


class _Wrapped(torch.Tensor):
    """A tensor whose values are in another one, and which has no memory of its own."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.t = t

    @classmethod
    def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
        return f(*[a.t if isinstance(a, cls) else a for a in args], **(kwargs or {}))


@pytest.mark.parametrize("name", ["linear", "norm linear", "norm"])
def test_wrapped_gradients_are_refused(name):
    inputs, f = _calls(24)[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    outs = f(*leaves)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(outs, leaves, [_Wrapped(torch.ones_like(y)) for y in outs], retain_graph=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(outs, leaves, [torch.ones(3, *y.shape, device="cuda") for y in outs], is_grads_batched=True)


@pytest.mark.parametrize("name", ["linear", "norm linear"])
def test_the_status_word_may_be_reset_between_forward_and_backward(name):
    """``check_status`` clears it after an error that some other kernel recorded; the graph of a sound step is not part of that."""
    from jigsaw_b200.ops import symm

    inputs, f = _calls(24)[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    gs = [_tensor(*y.shape, seed=20 + k) for k, y in enumerate(f(*inputs))]
    want = torch.autograd.grad(f(*leaves), leaves, gs)
    outs = f(*leaves)
    status = symm.arena(outs[0].device)
    status.status[0] = 1
    with pytest.raises(RuntimeError, match="kernel error 1"):
        status.check_status()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(outs, leaves, gs), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [64, 65, 5000])
def test_sums_and_outputs_below_the_normal_range(C, dtype):
    """The stored sum is the rounded sum of the two tensors at every size, and the norm is of that sum: values below 2^-126 are
    not flushed to zero on the way in."""
    F = _F()
    g = torch.Generator(device="cuda").manual_seed(0)
    step = 2.0**-149 if dtype == torch.float32 else 2.0**-133
    x, r = (torch.randint(-(2**6), 2**6, (7, C), generator=g, device="cuda").double() * step for _ in range(2))
    x[:, 0], r[:, 0] = 2.0**-126, -(2.0**-126) + step
    x, r = x.to(dtype), r.to(dtype)
    gain = torch.full((C,), 2.0**20, device="cuda")
    want = x.double() + r.double()
    y, t = F.distributed_rms_norm(x, gain, eps=2.0**-40, residual=r)
    assert torch.equal(t.double(), want) and bool(want.any())
    # r = 2^20 exactly, and two products by powers of two: one rounding to the type
    assert torch.equal(y, (want * 2.0**40).to(dtype))
    assert torch.equal(F.rms_norm_quantize(x, gain, 2.0**-40, r)[1].double(), want)


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M, N, K", [(5, 300, 131072), (130, 140, 131072), (1100, 9700, 32768)])
def test_scaled_matmul_long_rows_that_cancel(M, N, K, out):
    """The loss of the truncating additions is relative to the sum of magnitudes S: 16-bit results take at most 512 of them in a
    row (fp32: 64), each up to 2^-23 S, then K / 16384 (fp32: K / 2048) rounded additions of what was drained and at most 16 of
    parts (two accumulators, eight CTAs), and one rounding."""
    F = _F()
    g = torch.Generator(device="cuda").manual_seed(0)
    a = torch.rand(M, K, generator=g, device="cuda") + 1.0
    sign = torch.ones(K, device="cuda")
    sign[K // 2:] = -1.0                         # what the first half of a row adds up, the second takes away
    a = F.quantize_blockwise(a * sign * 2.0**-8)
    b = F.quantize_blockwise(torch.rand(N, K, generator=g, device="cuda") + 1.0, (128, 128))
    va = a.dequantize(torch.float64)
    parts = b.dequantize().split(1024)
    want = torch.cat([va @ p.double().t() for p in parts], dim=1)
    total = torch.cat([va.abs() @ p.double().abs().t() for p in parts], dim=1)
    assert float(want.abs().median()) < 0.02 * float(total.median()), "the sums cancel"
    chunk = 2048 if out == torch.float32 else 16384
    bound = (chunk // 32 * 2.0**-23 + (K // chunk + 16) * 2.0**-24) * total
    half = torch.finfo(out).eps / 2
    y = F.scaled_matmul(a, b, out_dtype=out).double()
    assert bool(((y - want).abs() <= bound * (1 + half) + half * want.abs() + 2.0**-25).all())


# ----------------------------------------------------------------------------- gradients against 64 bits
def _span(h, quantised):
    """Values of the quantised ``h`` in 64 bits, and how far they move if ``h`` is off by 40 2^-24 of itself (the error of the
    kernels' norm): a code changes only where that crosses a rounding border."""
    low, high = quantised(h * (1 - 40 * U)), quantised(h * (1 + 40 * U))
    return quantised(h), (high - low).abs()


def _check_norm_linear(M, N, K, dtype, wdtype, residual, bias):
    F = _F()
    x = _tensor(M, K, dtype=dtype).requires_grad_()
    r = _tensor(M, K, dtype=dtype, seed=1).requires_grad_() if residual else None
    n = (_tensor(1, K, seed=2, spread=0.0)[0] * 0.2 + 1).to(wdtype).requires_grad_()
    w = (_tensor(N, K, seed=3, spread=0.1) * K**-0.5).to(wdtype).requires_grad_()
    b = _tensor(1, N, seed=4)[0].to(wdtype).requires_grad_() if bias else None
    g, gs = (_tensor(M, N, seed=5) / 64).to(dtype), (_tensor(M, K, seed=6) / 64).to(dtype)
    leaves = {k: t for k, t in dict(x=x, r=r, n=n, w=w, b=b).items() if t is not None}
    out = F.rms_norm_linear(x, n, w, b, 1e-5, r)
    y, t = out if residual else (out, x)
    got = dict(zip(leaves, torch.autograd.grad((y, t) if residual else (y,), list(leaves.values()), (g, gs) if residual else (g,))))

    h, rt, rr = O.norm(x.detach(), None if r is None else r.detach(), n.detach(), 1e-5)
    vw, vg, cg = O.values(w.detach(), True), O.values(g), O.values_along_rows(g)
    (vh, dh_codes), (ch, dc_codes) = _span(h, O.values), _span(h, O.values_along_rows)
    bd = 0.0 if b is None else b.detach().double()
    ry = vh @ vw.t() + bd
    O.assert_within(y, ry, O.product_bound(vh, vw, ry, dtype) + dh_codes @ vw.abs().t() + 2.0**-23 * (ry.abs() + abs(bd)), "y")
    assert torch.equal(t.double(), rt) and y.dtype == dtype
    rw = cg.t() @ ch
    O.assert_within(got["w"], rw, O.product_bound(cg.t(), ch.t(), rw, wdtype) + cg.abs().t() @ dc_codes, "dw")
    if bias:
        rb = g.double().sum(0)
        O.assert_within(got["b"], rb, (M + 8) * U * g.double().abs().sum(0) + O.half_step(wdtype) * rb.abs() + 2.0**-25, "db")
    # the gradient of the normalised rows is an fp32 product, whose error goes through the norm's own backward pass
    rh = vg @ vw
    off = O.product_bound(vg, vw.t(), rh, torch.float32)
    rx, rn = O.norm_backward(rh, gs if residual else None, rt, rr, n.detach())
    gain = n.detach().double().abs()

    def through(m):
        return rr * (gain * m + rt.abs() * rr.square() * (gain * m * rt.abs()).mean(1, keepdim=True))

    tiny = torch.finfo(dtype).smallest_normal
    bound = through(off) + 100 * U * through(rh.abs()) + 4 * U * (gs.double().abs() if residual else 0) + O.half_step(dtype) * rx.abs() + tiny
    O.assert_within(got["x"], rx, bound * (1 + O.half_step(dtype)), "dx")
    if residual:
        assert torch.equal(got["x"], got["r"])
    bound = (off * rt.abs() * rr).sum(0) + (M + 40) * U * (rh * rt * rr).abs().sum(0) + O.half_step(wdtype) * rn.abs() + tiny
    O.assert_within(got["n"], rn, bound * (1 + O.half_step(wdtype)), "dgain")


@pytest.mark.parametrize("dtype, wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                           (torch.float32, torch.float32)])
@pytest.mark.parametrize("M, N, K", [(1, 24, 64), (300, 384, 512), (257, 130, 1001), (1030, 96, 1024), (5, 40, 8200), (3, 33, 8201), (150, 64, 5120),
                                     (2, 17, 20000)])
def test_rms_norm_linear_and_its_gradients(M, N, K, dtype, wdtype):
    _check_norm_linear(M, N, K, dtype, wdtype, True, True)
    _check_norm_linear(M, N, K, dtype, wdtype, False, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, C", [(1, 1), (3, 7), (300, 512), (700, 256), (1023, 1001), (310, 4096), (5, 8200), (3, 8201), (2, 16392), (2, 20000)])
def test_norm_of_16_bit_rows_with_a_gradient_in_fp32(R, C, dtype):
    """Under autocast the norm's output, and so its gradient, is fp32 while the sum stays in 16 bits."""
    F = _F()
    x, r = (_tensor(R, C, dtype=dtype, seed=k).requires_grad_() for k in (0, 1))
    w = (_tensor(1, C, seed=2)[0] + 1).requires_grad_()
    g, gs = _tensor(R, C, seed=3), _tensor(R, C, dtype=dtype, seed=4)
    with torch.autocast("cuda", dtype=dtype):
        y, t = F.distributed_rms_norm(x, w, eps=1e-5, residual=r)
    assert y.dtype == torch.float32 and t.dtype == dtype
    dx, dr, dw = torch.autograd.grad((y, t), (x, r, w), (g, gs))
    ry, rt, rr = O.norm(x.detach(), r.detach(), w.detach(), 1e-5)
    rx, rw = O.norm_backward(g, gs, rt, rr, w.detach())
    tiny = torch.finfo(dtype).smallest_normal
    assert torch.equal(t.double(), rt) and torch.equal(dx, dr)
    O.assert_within(y, ry, 41 * U * ry.abs() + 2.0**-126, "y")
    wg = g.double().abs() * w.detach().double().abs()
    mag = rr * (wg + rt.abs() * rr.square() * (wg * rt.abs()).mean(1, keepdim=True))
    O.assert_within(dx, rx, 100 * U * mag + 4 * U * gs.double().abs() + O.half_step(dtype) * rx.abs() + tiny, "dx")
    O.assert_within(dw, rw, (R + 40) * U * (g.double() * rt * rr).abs().sum(0) + U * rw.abs() + tiny, "dw")


# ----------------------------------------------------------------------------- layers
def _worker_layers(rank, world):
    import jigsaw_b200 as jb
    from jigsaw_b200.ops import _lib

    dev = torch.device("cuda", 0)
    mesh = jb.make_process_mesh({"row": 1, "col": 1})
    row, col, model = mesh["row"], mesh["col"], mesh["model"]
    with _lib.strict_fused():
        for dtype in (torch.float32, torch.bfloat16):
            norm = jb.modules.DistributedRMSNorm(200, None, dev, row, col, dtype=dtype)
            cfg = jb.modules.LinearConfig(model, linear_layer=True, device=dev, precision="fp8")
            fc = jb.modules.DistributedLinear(200, 72, dev, model, row, col, config=cfg, dtype=dtype)
            with torch.no_grad():
                norm.weight.copy_(1 + 0.2 * _tensor(1, 200, seed=9)[0])
            x, g = _tensor(3, 50, 200, dtype=dtype).requires_grad_(), _tensor(3, 50, 72, dtype=dtype, seed=1)
            y = fc(x)
            dx, dw, db = torch.autograd.grad(y, (x, fc.weight, fc.bias), g)
            x2, g2 = x.detach().view(150, 200), g.view(150, 72)
            wd, bd = fc.weight.detach(), fc.bias.detach().double()
            vx, vw, vg, cx, cg = O.values(x2), O.values(wd, True), O.values(g2), O.values_along_rows(x2), O.values_along_rows(g2)
            ry = vx @ vw.t() + bd
            O.assert_within(y.view(150, 72), ry, O.product_bound(vx, vw, ry, dtype) + 2.0**-23 * (ry.abs() + bd.abs()), "layer")
            O.assert_within(dx.view(150, 200), vg @ vw, O.product_bound(vg, vw.t(), vg @ vw, dtype), "dx")
            O.assert_within(dw, cg.t() @ cx, O.product_bound(cg.t(), cx.t(), cg.t() @ cx, dtype), "dw")
            rb = g2.double().sum(0)
            O.assert_within(db, rb, 158 * U * g2.double().abs().sum(0) + O.half_step(dtype) * rb.abs(), "db")
            # norm and layer in one: three launches, and the function of its parts
            r = _tensor(3, 50, 200, dtype=dtype, seed=2)
            before = _lib.LAUNCHES
            h, t = norm.forward_linear(x.detach(), fc, r)
            assert _lib.LAUNCHES == before + 3
            want, rt = jb.modules.functional.rms_norm_linear(x.detach(), norm.weight, fc.weight, fc.bias, 2.0**-23, r)
            assert torch.equal(h, want) and torch.equal(t, rt) and torch.equal(t, x.detach() + r)
            if dtype == torch.float32:                     # nothing is rounded between the modules
                handle = fc.register_forward_hook(lambda *a: None)
                assert torch.equal(norm.forward_linear(x.detach(), fc, r)[0], h)
                handle.remove()
        # the default eps, from the kernels, against torch on small rows
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            z = (_tensor(40, 256, seed=3, spread=0.0) * 0.003).to(dtype)
            ref = torch.nn.RMSNorm(256, device=dev, dtype=dtype)
            layer = jb.convert.convert_to_jigsaw(torch.nn.Sequential(ref), mesh, dev)[0]
            want = z.double() * (z.double().square().mean(1, keepdim=True) + 2.0**-23).rsqrt()
            tiny = torch.finfo(dtype).smallest_normal
            O.assert_within(layer(z), want, (40 * U + O.half_step(dtype)) * want.abs() + tiny, "default eps")
            O.assert_within(ref(z), want, (300 * U + 2 * O.half_step(dtype)) * want.abs() + tiny, "torch")
            with torch.autocast("cuda", dtype=torch.bfloat16):
                y = layer(z)
            assert y.dtype == torch.float32
            O.assert_within(y, want, 41 * U * want.abs() + 2.0**-126, "default eps under autocast")


def test_layers():
    run_distributed(_worker_layers, 1, backend="nccl")


def _worker_vit(rank, world):
    import jigsaw_b200 as jb
    from jigsaw_b200.models import ViT, ViTConfig
    from jigsaw_b200.ops import _lib

    dev = torch.device("cuda", 0)
    mesh = jb.make_process_mesh({"row": 1, "col": 1})
    torch.manual_seed(0)
    model = ViT(mesh, dev, ViTConfig(depth=2, norm="rms", linear_precision="fp8"))
    cfg = ViTConfig()
    x = torch.randn(1, cfg.in_channels, *cfg.image_size, device=dev)

    def step():
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = model(x)
        out.float().square().mean().backward()
        return out.detach(), [p.grad for p in model.parameters()]

    _lib.dispatch_counts(reset=True)
    out, grads = step()
    counts = _lib.dispatch_counts()
    assert counts["rms_norm_linear"] == {**counts["rms_norm_linear"], "fused": 2, "fallback": 0}
    assert counts["scaled_linear"]["fused"] == 2 and counts["scaled_linear"]["fallback"] == 0
    assert bool(out.isfinite().all()) and all(g is not None and bool(g.isfinite().all()) for g in grads)
    # each block is what its modules do one after the other
    blk = model.blocks[0]
    t = _tensor(1, 40, cfg.dim, seed=5)
    with torch.no_grad():
        a = blk.attn(blk.norm1(t))
        h, s = jb.modules.functional.distributed_rms_norm(a, blk.norm2.weight, eps=2.0**-23, residual=t)
        want = s + blk.fc2(blk.act(blk.fc1(h)))
        torch.testing.assert_close(blk(t), want, rtol=1e-5, atol=1e-5 * float(want.abs().max()))


def test_vit_with_rms_norms_and_8_bit_products():
    run_distributed(_worker_vit, 1, backend="nccl")


# ----------------------------------------------------------------------------- saved-tensor hooks
def _spread(t):
    """The same values at other strides: every second row of a wider buffer."""
    if t.dim() == 0:
        return t
    raw = t.contiguous().view(torch.uint8) if t.element_size() == 1 else t.contiguous()
    buffer = raw.new_zeros(*(2 * n for n in raw.shape))
    view = buffer[tuple(slice(0, n) for n in raw.shape)] if t.dim() > 1 else buffer[::2]
    view.copy_(raw)
    return view.view(t.dtype) if t.element_size() == 1 else view


@pytest.mark.parametrize("name", ["linear", "norm linear", "norm"])
def test_what_saved_tensor_hooks_give_back(name):
    """Copies at other strides give the same gradients; a tensor on another device, of another type or shape is refused."""
    hooks = torch.autograd.graph.saved_tensors_hooks
    inputs, f = _calls(130)[name]
    leaves = [t.clone().requires_grad_() for t in inputs]
    gs = [_tensor(*y.shape, seed=20 + k) for k, y in enumerate(f(*inputs))]
    want = torch.autograd.grad(f(*leaves), leaves, gs)

    def grads(unpack):
        with hooks(lambda t: t.clone(), unpack):
            outs = f(*leaves)
        return torch.autograd.grad(outs, leaves, gs)

    for unpack in (lambda t: t, _spread):
        assert all(torch.equal(a, b) for a, b in zip(grads(unpack), want))
    with torch.autograd.graph.save_on_cpu():
        outs = f(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(outs, leaves, gs), want))
    for unpack in (lambda t: t.cpu(), lambda t: t.view(torch.uint8), lambda t: t[..., :-1], lambda t: t[:1], lambda t: t.double()):
        with pytest.raises(RuntimeError):
            grads(unpack)
