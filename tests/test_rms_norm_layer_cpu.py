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


# ----------------------------------------------------------------------------- conversion
class _Group:
    def __init__(self, n):
        self.n = n

    def size(self):
        return self.n


@pytest.mark.parametrize("shape, col, options", [((4, 8), 1, {}), ((8,), 3, {}), ((8,), 1, {"convert_layer_norm": False}),
                                                 ((8,), 2, {"convert_layer_norm": False})])
def test_norms_that_the_layer_cannot_take_are_left_to_non_safe(shape, col, options):
    """Over several axes, over features that the column ranks cannot share, or not to be converted: refused before anything is
    changed, and kept as plain torch with ``non_safe=True``."""
    from jigsaw_b200 import convert

    mesh = {"row": _Group(1), "col": _Group(col), "model": _Group(col)}
    inner = torch.nn.Sequential(torch.nn.RMSNorm(shape))
    model = torch.nn.Sequential(torch.nn.GELU(), inner)
    with pytest.raises(ValueError, match=r"1\.0: non-elementwise module RMSNorm"):
        convert.convert_to_jigsaw(model, mesh, "cpu", **options)
    with pytest.warns(UserWarning, match=r"1\.0: non-elementwise module RMSNorm"):
        out = convert.convert_to_jigsaw(model, mesh, "cpu", non_safe=True, **options)
    assert out is model and type(inner[0]) is torch.nn.RMSNorm


def test_a_default_half_precision_norm_keeps_its_function_through_conversion():
    from dist_utils import run_distributed

    run_distributed(_worker_convert, 2)


def _worker_convert(rank, world):
    import jigsaw_b200 as jb
    from dist_utils import all_ok

    mesh = jb.make_process_mesh({"row": 2, "col": 1})
    for dtype in (torch.bfloat16, torch.float16):
        ref = torch.nn.RMSNorm(64, dtype=dtype)
        torch.manual_seed(0)
        torch.nn.init.uniform_(ref.weight, 0.5, 2.0)
        x = _rows(5, 64, dtype=dtype, size=0.01)
        want = _want(x, 2.0**-23) * ref.weight.detach().double()
        layer = jb.convert.convert_to_jigsaw(torch.nn.Sequential(ref), mesh, "cpu")[0]
        assert isinstance(layer, DistributedRMSNorm)
        for m in (layer, ref, layer.convert_to_torch(mesh)):
            assert all_ok(bool(((m(x).detach().double() - want).abs() <= 2 * _bound(want, dtype)).all()))


@pytest.mark.parametrize("kind", [torch.nn.LayerNorm, torch.nn.RMSNorm])
def test_norms_convert_without_groups(kind):
    """A mesh whose axes have no group is a single process: nothing is cut."""
    from jigsaw_b200 import convert

    layer = convert.convert_to_jigsaw(kind(8), {"row": None, "col": None, "model": None}, "cpu")
    assert type(layer).__name__ == f"Distributed{kind.__name__}" and layer.local_dim == 8
    x = _rows(3, 8, dtype=torch.float32, size=1.0)
    torch.testing.assert_close(layer(x), kind(8)(x))
