"""``DistributedRMSNorm.forward_linear`` in front of an 8-bit linear layer, when something watches or replaces module calls."""

import pytest
import torch

from dist_utils import all_ok, assert_close, run_distributed


def _layers(jb, mesh):
    row, col, model = mesh["row"], mesh["col"], mesh["model"]
    torch.manual_seed(0)
    norm = jb.modules.DistributedRMSNorm(64, None, "cpu", row, col, eps=1e-6)
    cfg = jb.modules.LinearConfig(model, linear_layer=True, device="cpu", precision="fp8")
    fc = jb.modules.DistributedLinear(64, 32, "cpu", model, row, col, config=cfg)
    return norm, fc


def _worker_hooks(rank, world):
    import jigsaw_b200 as jb

    mesh = jb.make_process_mesh({"row": 1, "col": 1})
    norm, fc = _layers(jb, mesh)
    x, r = torch.randn(5, 64, generator=torch.Generator().manual_seed(1)), torch.randn(5, 64, generator=torch.Generator().manual_seed(2))
    want, total = norm.forward_linear(x, fc, r)
    register = {
        "forward": lambda m, f: m.register_forward_hook(lambda mod, a, out: f(mod)),
        "forward pre": lambda m, f: m.register_forward_pre_hook(lambda mod, a: f(mod)),
        "backward": lambda m, f: m.register_full_backward_hook(lambda mod, gi, go: f(mod)),
        "backward pre": lambda m, f: m.register_full_backward_pre_hook(lambda mod, go: f(mod)),
        "every module": lambda m, f: torch.nn.modules.module.register_module_forward_hook(lambda mod, a, out: f(mod) if mod is m else None),
    }
    for kind, put in register.items():
        for watched in (norm, fc):
            seen = []
            handle = put(watched, lambda m: seen.append(m))
            y, t = norm.forward_linear(x.clone().requires_grad_(), fc, r.clone().requires_grad_())
            y.sum().backward()
            handle.remove()
            assert all_ok(seen == [watched]), (kind, type(watched), len(seen))
            assert_close(y, want, kind, 1e-6, 1e-6)
            assert torch.equal(t, total)
    # the gradient of a hook on the output counts
    handle = fc.register_forward_hook(lambda mod, a, out: out * 2)
    assert_close(norm.forward_linear(x, fc, r)[0], 2 * want, "changed output", 1e-6, 1e-6)
    handle.remove()
    # a module whose forward was replaced, and a subclass with a forward of its own
    fc.forward = lambda h: type(fc).forward(fc, h) + 1
    assert_close(norm.forward_linear(x, fc, r)[0], want + 1, "replaced forward", 1e-6, 1e-6)
    del fc.forward

    class Plus(jb.modules.DistributedLinear):
        def forward(self, h):
            return super().forward(h) + 3

    class Twice(jb.modules.DistributedRMSNorm):
        def forward(self, x, residual=None):
            y, t = super().forward(x, residual)
            return 2 * y, t

    fc.__class__ = Plus
    assert_close(norm.forward_linear(x, fc, r)[0], want + 3, "subclass of the linear layer", 1e-6, 1e-6)
    fc.__class__ = jb.modules.DistributedLinear
    norm.__class__ = Twice
    assert_close(norm.forward_linear(x, fc, r)[0] - fc.bias, 2 * (want - fc.bias), "subclass of the norm", 1e-5, 1e-5)


def test_hooks_and_replaced_forwards_are_not_passed_by():
    run_distributed(_worker_hooks, 1)


def _worker_vit(rank, world):
    import jigsaw_b200 as jb
    from jigsaw_b200.models import ViT, ViTConfig

    mesh = jb.make_process_mesh({"row": 1, "col": 1})
    cfg = ViTConfig(depth=1, norm="rms", linear_precision="fp8")
    model = ViT(mesh, "cpu", cfg)
    seen = []
    for name, m in model.named_modules():
        if name:
            m.register_forward_hook(lambda mod, a, out, name=name: seen.append(name))
    model(torch.randn(1, cfg.in_channels, *cfg.image_size))
    assert all_ok({"blocks.0.norm1", "blocks.0.norm2", "blocks.0.fc1", "blocks.0.fc2"} <= set(seen)), seen


def test_every_layer_of_the_vit_is_seen_by_hooks():
    run_distributed(_worker_vit, 1)
