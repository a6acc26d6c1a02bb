"""``DistributedRMSNorm`` against ``torch.nn.RMSNorm``: the default eps."""

import pytest
import torch

from jigsaw_b200.modules import DistributedRMSNorm

TYPES = [torch.bfloat16, torch.float16, torch.float32, torch.float64]


def _rows(*shape, dtype, size, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * size).to(dtype)


def _want(t, eps):
    t = t.double()
    return t * (t.square().mean(-1, keepdim=True) + eps).rsqrt()


def _bound(want, dtype):
    # fp32 sums of 64 squares, a root and a product, then one rounding; torch rounds the product to the type once more
    u = torch.finfo(torch.promote_types(dtype, torch.float32)).eps / 2
    return (64 + 8) * u * want.abs() + torch.finfo(dtype).eps * want.abs() + torch.finfo(dtype).smallest_normal


# ----------------------------------------------------------------------------- default eps
@pytest.mark.parametrize("size", [0.003, 0.03, 1.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_default_eps_is_that_of_torch(dtype, size):
    """Without an eps the norm takes the machine epsilon of the type that it computes in: fp32 for 16-bit inputs."""
    x = _rows(5, 64, dtype=dtype, size=size)
    layer, ref = DistributedRMSNorm(64, None, "cpu", None, None, dtype=dtype), torch.nn.RMSNorm(64, dtype=dtype)
    want = _want(x, 2.0**-52 if dtype == torch.float64 else 2.0**-23)
    for got in (layer(x), ref(x)):
        assert bool(((got.double() - want).abs() <= _bound(want, dtype)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_default_eps_in_front_of_a_linear_layer(dtype):
    x = _rows(5, 64, dtype=dtype, size=0.003)
    layer, eye = DistributedRMSNorm(64, None, "cpu", None, None, dtype=dtype), torch.nn.Identity()
    want = _want(x, 2.0**-23)
    assert bool(((layer.forward_linear(x, eye).double() - want).abs() <= _bound(want, dtype)).all())


@pytest.mark.parametrize("dtypes", [(torch.float32, torch.float64), (torch.float64, torch.float32), (torch.bfloat16, torch.float64),
                                    (torch.bfloat16, torch.float32)])
def test_default_eps_is_that_of_the_sum(dtypes):
    """What is normalised is the sum in the common type of input and residual: the order of the two changes nothing, and the norm is
    that of the sum alone."""
    x, r = _rows(5, 64, dtype=dtypes[0], size=2e-7), _rows(5, 64, dtype=dtypes[1], size=2e-7, seed=1)
    common = torch.promote_types(*dtypes)
    layer = DistributedRMSNorm(64, None, "cpu", None, None, dtype=common)
    y, t = layer(x, r)
    assert t.dtype == y.dtype == common
    want = _want(t, 2.0**-52 if common == torch.float64 else 2.0**-23)
    for got in (y, layer(r, x)[0], layer(t), layer.forward_linear(x, torch.nn.Identity(), r)[0], torch.nn.functional.rms_norm(t, (64,))):
        assert bool(((got.double() - want).abs() <= _bound(want, common)).all())
