"""``DistributedRMSNorm``: root-mean-square norm over a feature dimension split across ``col_group``, with the residual's
addition in the same call.

The weight holds the local ``C / col`` slice, is replicated (marked, broadcast) over ``row_group`` and gets its gradient
summed over it by ``sync_grad``.  Only a single trailing normalised dimension is supported.  The reference has no such
layer; this one follows its LayerNorm (jigsaw/modules/normalization/_layer_norm.py:15-368) in constructor, conversion and
re-sharding.
"""

from __future__ import annotations

from typing import Any

import torch
import torch.distributed as dist

from ... import parallel
from ..._core.placement import check_divisible, gather_dim
from ..._core.shard_repr import shard_repr
from ..linear._linear import DistributedLinear
from ._rms_functional import distributed_rms_norm, rms_norm_linear


def _called_plainly(module: torch.nn.Module, kind: type) -> bool:
    """A call of ``module`` runs ``kind.forward`` and nothing else: no hook, no forward of a subclass or of the instance."""
    return (type(module).forward is kind.forward and "forward" not in vars(module)
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


class DistributedRMSNorm(torch.nn.Module):
    def __init__(
        self,
        normalized_dim: int,
        local_rank: int | None,
        device: torch.device | str,
        row_group: dist.ProcessGroup | None,
        col_group: dist.ProcessGroup | None,
        eps: float | None = None,
        elementwise_affine: bool = True,
        dtype: torch.dtype | None = None,
    ) -> None:
        super().__init__()
        if not isinstance(normalized_dim, int):
            if len(tuple(normalized_dim)) != 1:
                raise NotImplementedError("DistributedRMSNorm normalizes a single trailing dimension only")
            normalized_dim = int(tuple(normalized_dim)[0])
        self.normalized_dim = normalized_dim
        self.local_rank = local_rank                      # kept as given; the layer takes its place from the groups
        self.device = torch.device(device)
        self.row_group, self.col_group = row_group, col_group
        self.eps = eps                                    # None: see _eps
        self.elementwise_affine = elementwise_affine
        local = check_divisible(normalized_dim, 1 if col_group is None else col_group.size(), "normalized_dim")
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.ones(local, device=self.device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        self._mark()

    @property
    def spatial_group(self) -> dist.ProcessGroup | None:
        return self.row_group

    @property
    def channel_group(self) -> dist.ProcessGroup | None:
        return self.col_group

    @property
    def local_dim(self) -> int:
        """Features of the normalised axis held by this rank."""
        return self.normalized_dim // (1 if self.col_group is None else self.col_group.size())

    def _mark(self) -> None:
        for p in self.parameters():
            if not parallel.replica_groups(p):
                parallel.mark_replicated(p, [self.row_group])
        with torch.no_grad():
            if self.row_group is not None and self.row_group.size() > 1:
                for p in self.parameters():
                    dist.broadcast(p.data, group_src=0, group=self.row_group)

    def _eps(self, x: torch.Tensor, residual: torch.Tensor | None) -> float:
        """Without an eps: the machine epsilon of the type that the norm of the sum computes in, as in ``torch.nn.RMSNorm``
        (2^-52 where one of the two is fp64, else 2^-23)."""
        if self.eps is not None:
            return self.eps
        wide = x.dtype == torch.float64 or (residual is not None and residual.dtype == torch.float64)
        return torch.finfo(torch.float64 if wide else torch.float32).eps

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> Any:
        """``y``, or ``(y, x + residual)`` with a residual."""
        (w,) = parallel.sync_grad(self.weight)
        return distributed_rms_norm(x, w, self.col_group, self._eps(x, residual), residual)

    def forward_linear(self, x: torch.Tensor, linear: torch.nn.Module, residual: torch.Tensor | None = None) -> Any:
        """``linear(self(x, residual))``, and the sum if there is a residual.  With an 8-bit ``DistributedLinear`` whose
        input features are whole on this rank, the norm's output goes into the product as 8-bit codes, unless something
        watches or replaces a call of one of the two (hooks, an own ``forward``): then both modules are called, and the norm's
        output is rounded to its type in between."""
        if (_called_plainly(self, DistributedRMSNorm) and isinstance(linear, DistributedLinear) and _called_plainly(linear, DistributedLinear)
                and linear.config.precision == "fp8" and linear.col_group.size() == 1
                and not torch.nn.modules.module._has_any_global_hook()):
            g, w, b = parallel.sync_grad(self.weight, linear.weight, linear.bias)
            return rms_norm_linear(x, g, linear._out_block_weight(w), b, self._eps(x, residual), residual)
        out = self(x, residual)
        return linear(out) if residual is None else (linear(out[0]), out[1])

    # ------------------------------------------------------------------ conversion
    @classmethod
    def convert_to_jigsaw(
        cls, model: torch.nn.RMSNorm, process_mesh_dict: dict, device: torch.device | str, row_kw: str = "row",
        col_kw: str = "col", model_kw: str = "model", **kwargs: Any,
    ) -> "DistributedRMSNorm":
        if len(model.normalized_shape) != 1:
            raise NotImplementedError("DistributedRMSNorm normalizes a single trailing dimension only")
        layer = cls(
            model.normalized_shape[0], None, device, process_mesh_dict[row_kw], process_mesh_dict[col_kw], eps=model.eps,
            elementwise_affine=model.elementwise_affine, dtype=None if model.weight is None else model.weight.dtype,
        )
        layer._load_global(model.weight)
        return layer

    def _load_global(self, weight: torch.Tensor | None) -> None:
        r = 0 if self.col_group is None else self.col_group.rank()
        n = self.local_dim
        with torch.no_grad():
            if weight is not None and self.weight is not None:
                self.weight.data = weight.detach()[r * n : (r + 1) * n].clone().to(self.device)

    def merge_weights(self, from_process_mesh: dict, row_kw: str = "row", col_kw: str = "col",
                      model_kw: str = "model") -> torch.Tensor | None:
        """All-gather the slices over the column group (``row_kw`` and ``model_kw`` are accepted for a uniform
        signature: the weight is not cut over them)."""
        with torch.no_grad():
            return None if self.weight is None else gather_dim(self.weight.detach(), from_process_mesh[col_kw], 0)

    def convert_to_torch(self, process_mesh_dict: dict, row_kw: str = "row", col_kw: str = "col", model_kw: str = "model") -> torch.nn.RMSNorm:
        w = self.merge_weights(process_mesh_dict, col_kw=col_kw)
        layer = torch.nn.RMSNorm(self.normalized_dim, eps=self.eps, elementwise_affine=self.elementwise_affine, device=self.device)
        if w is not None:
            layer.weight.data = w
        return layer

    def reshard_parameters(self, from_process_mesh: dict, to_process_mesh: dict, pm_row_key: str = "row",
                           pm_col_key: str = "col", pm_model_key: str = "model") -> None:
        new_col = to_process_mesh[pm_col_key]
        check_divisible(self.normalized_dim, new_col.size(), "normalized_dim")
        w = self.merge_weights(from_process_mesh, col_kw=pm_col_key)
        self.row_group, self.col_group = to_process_mesh[pm_row_key], new_col
        if self.weight is not None and w is not None:
            self.weight = torch.nn.Parameter(torch.empty(0, device=self.device, dtype=w.dtype))
        self._load_global(w)
        self._mark()

    def shard_spec(self) -> dict:
        """Which dimension of which parameter is cut over which group (sharded checkpoints)."""
        return {"weight": () if self.col_group is None else ((0, self.col_group),)}

    def get_parameter_count(self) -> int:
        return self.normalized_dim if self.elementwise_affine else 0

    def extra_repr(self) -> str:
        return (f"({self.normalized_dim},), eps={self.eps}, elementwise_affine={self.elementwise_affine}, "
                + shard_repr(row=self.row_group, col=self.col_group))
