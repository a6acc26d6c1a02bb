"""Gradients of the norm and of the 8-bit linear layers on the kernels, in the forms in which autograd hands them over."""

import pytest
import torch

pytestmark = pytest.mark.gpu


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
