"""Root-mean-square norm with the residual's addition, in the input's type, in 8 bits, and fused in front of an 8-bit
linear layer.

    t = x + residual            (rounded to the type of x: the sum is stored, and the norm is of the stored sum)
    y = t * r * weight,         r = (mean(t^2) + eps)^(-1/2)

    dt_k = r (w_k g_k - r^2 t_k mean(w g t)) + gradient that reaches the sum on its own,    dw = sum over rows of g t r

The feature axis may be cut over a column group: the sum of squares is then added over the group (a differentiable
all-reduce, whose adjoint is the backward pass's).
"""

from __future__ import annotations

import math
from typing import Any

import torch
import torch.distributed as dist
from torch.autograd.function import once_differentiable

from ..._core.autocast import autocast_dtype
from ..._core.collectives import all_reduce_sum
from ...ops import scaled_fused
from ..linear._scaled import (
    _HALF,
    ROW,
    SQUARE,
    BlockScaled,
    _check_linear,
    _grads,
    _made,
    _out_dtype,
    _product,
    _quantize_2d,
    _refuse_vmap,
    _traced,
    quantize_blockwise,
)


def _check(name: str, x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None, eps: float) -> None:
    if not x.is_floating_point() or x.element_size() == 1:
        raise TypeError(f"{name} takes fp64, fp32, bf16 or fp16 tensors, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError(f"{name} needs at least one dimension")
    if weight is not None and weight.shape != (x.shape[-1],):
        raise ValueError(f"{name}: weight of shape {tuple(weight.shape)} for {x.shape[-1]} features")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{name}: residual of shape {tuple(residual.shape)}, input of shape {tuple(x.shape)}")
    dev = x.device
    if (weight is not None and weight.device != dev) or (residual is not None and residual.device != dev):
        raise ValueError(f"{name}: input on {dev}, weight or residual on another device")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"{name}: eps must be finite and not negative, got {eps}")


def _same_type(x: torch.Tensor, residual: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor | None]:
    if residual is None or residual.dtype == x.dtype:
        return x, residual
    dt = torch.promote_types(x.dtype, residual.dtype)
    return x.to(dt), residual.to(dt)


def _plain(x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None, col_group: Any, eps: float) -> tuple:
    """``(normalised rows in fp32 or wider, sum, r)`` in torch operations."""
    t = x if residual is None else x + residual
    wide = t.to(torch.promote_types(t.dtype, torch.float32))
    parts = 1 if col_group is None else col_group.size()
    sq = (wide * wide).sum(dim=-1, keepdim=True)
    if parts > 1:
        sq = all_reduce_sum(sq, col_group)
    r = torch.rsqrt(sq / (wide.shape[-1] * parts) + eps)
    y = wide * r
    return (y if weight is None else y * weight.to(torch.promote_types(weight.dtype, wide.dtype))), t, r


def _norm_backward(t: torch.Tensor, weight: torch.Tensor | None, rstd: torch.Tensor, g: torch.Tensor | None,
                   gsum: torch.Tensor | None, want_w: bool) -> tuple:
    """Gradients of the sum and of the weight; ``rstd [R]`` as the forward pass computed it."""
    want_w = want_w and weight is not None
    if g is None:                                 # only the sum was used
        return (None if gsum is None else gsum.to(t.dtype)), (torch.zeros_like(weight) if want_w and weight is not None else None)
    tw, gw, r = t.float(), g.float(), rstd[:, None]
    gy = gw if weight is None else gw * weight.float()
    dx = r * (gy - tw * (r * r * (gy * tw).mean(dim=1, keepdim=True)))
    if gsum is not None:
        dx = dx + gsum.float()
    return dx.to(t.dtype), (gw * tw * r).sum(dim=0).to(weight.dtype) if want_w and weight is not None else None


def distributed_rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, col_group: dist.ProcessGroup | None = None,
                         eps: float = 1e-6, residual: torch.Tensor | None = None) -> Any:
    """Root-mean-square norm of the last axis of ``x`` (cut over ``col_group``), times ``weight``.

    With ``residual`` (same shape) the norm is of ``x + residual``, and ``(y, x + residual)`` is returned: the sum, in the
    common type of the two, is the residual of the next block.  Statistics are fp32 or wider; ``y`` is fp32 under autocast
    and has the type of the sum otherwise.  Differentiable in every tensor.  On CUDA with the whole feature axis on one
    rank, fp32, bf16 and fp16 run as one kernel per direction (plus one that adds up the weight's gradient)."""
    whole = col_group is None or col_group.size() == 1
    if x.is_cuda and whole:
        out = scaled_fused.rms_norm(x, weight, residual, eps)
        if out is not None:
            return out[0] if residual is None else out
    _check("distributed_rms_norm", x, weight, residual, eps)
    if residual is not None and residual.dtype != x.dtype:
        x, residual = _same_type(x, residual)
        return distributed_rms_norm(x, weight, col_group, eps, residual)
    if x.is_cuda and whole and x.numel() > 0:
        scaled_fused.declined("rms_norm", "under torch.vmap, in 64 bits, or rows longer than the kernel keeps in registers")
    out_dtype = x.dtype if autocast_dtype(x.device.type) is None else torch.promote_types(x.dtype, torch.float32)
    y, t, _ = _plain(x, weight, residual, col_group, eps)
    y = y.to(out_dtype)
    return y if residual is None else (y, t)


def _norm_to_codes(x: torch.Tensor, weight: torch.Tensor | None, eps: float, residual: torch.Tensor | None,
                   keep_rstd: bool) -> tuple[BlockScaled, torch.Tensor, torch.Tensor | None]:
    """``(codes, sum, r)``; ``r`` per row."""
    if x.is_cuda:
        out = scaled_fused.rms_norm_quantize(x, weight, eps, residual, keep_rstd)
        if out is not None:
            return _made(out[0], out[1], ROW), (x if out[2] is None else out[2]), out[3]
        scaled_fused.declined("rms_norm_quantize", "in 64 bits, or rows longer than the kernel keeps in registers")
    y, t, r = _plain(x, weight, residual, None, eps)
    return quantize_blockwise(y), t, r.reshape(-1)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6,
                      residual: torch.Tensor | None = None) -> Any:
    """Root-mean-square norm with the output in 8 bits (blocks of 128 features, quantised from the unrounded fp32 value):
    a :class:`BlockScaled`, or ``(BlockScaled, x + residual)`` with a residual.  For inference: not differentiable
    (:func:`rms_norm_linear` is), so tensors that want gradients are refused."""
    if x.is_cuda and not _traced(x, weight, residual):
        out = scaled_fused.rms_norm_quantize(x, weight, eps, residual, False)
        if out is not None:
            q = _made(out[0], out[1], ROW)
            return q if residual is None else (q, out[2])
    _check("rms_norm_quantize", x, weight, residual, eps)
    _refuse_vmap("rms_norm_quantize", x, weight, residual)
    if _traced(x, weight, residual):
        raise ValueError("rms_norm_quantize has no gradient; use rms_norm_linear, or call it under torch.no_grad()")
    if residual is not None and residual.dtype != x.dtype:
        x, residual = _same_type(x, residual)
        return rms_norm_quantize(x, weight, eps, residual)
    if x.numel() == 0:
        empty = BlockScaled(x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
                            x.new_empty((*x.shape[:-1], -(-x.shape[-1] // 128)), dtype=torch.float8_e8m0fnu), ROW)
        return empty if residual is None else (empty, x + residual)
    q, t, _ = _norm_to_codes(x.detach(), weight, eps, None if residual is None else residual.detach(), False)
    return q if residual is None else (q, t)


class _RmsNormLinear(torch.autograd.Function):
    """The normalised rows exist only as codes.  The backward pass recomputes them from the stored sum, in the column blocks
    that the weight gradient wants, and keeps the gradient of the normalised rows in fp32 between the product and the norm.
    (CUDA calls take the native form of the same function.)"""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, gain: torch.Tensor | None, w: torch.Tensor, b: torch.Tensor | None, eps: float,
                residual: torch.Tensor | None, out_dtype: torch.dtype, need_h: bool, need_w: bool) -> Any:
        q, t, r = _norm_to_codes(x, gain, eps, residual, need_h or need_w)
        wr, wc, _ = _quantize_2d(w, SQUARE, cols=need_h)
        ctx.set_materialize_grads(False)
        ctx.need_w, ctx.has_residual = need_w, residual is not None
        ctx.types = (w.dtype, None if b is None else b.dtype)
        if need_h or need_w:
            ctx.save_for_backward(t, r, gain, *((wc.codes, wc.scales) if wc is not None else (None, None)))
        y = _product(q, wr, b, out_dtype)
        return y if residual is None else (y, t)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, g: torch.Tensor | None, gsum: torch.Tensor | None = None) -> tuple:
        want_b = ctx.needs_input_grad[3] and ctx.types[1] is not None
        if not ctx.saved_tensors:                 # only the bias wants a gradient
            db = g.sum(dim=0, dtype=torch.float32).to(ctx.types[1]) if g is not None and want_b else None
            return (None, None, None, db) + (None,) * 5
        t, r, gain, wc, ws = ctx.saved_tensors
        dh = dw = db = None
        if g is not None:
            gr, gc, db = _quantize_2d(g, ROW, rows=wc is not None, cols=ctx.need_w, colsum=ctx.types[1] if want_b else None)
            if wc is not None:
                dh = _product(gr, BlockScaled(wc, ws, SQUARE), None, torch.float32)
            if ctx.need_w:
                hc = _quantize_2d(t, ROW, rows=False, cols=True, rstd=r, gain=gain)[1]
                dw = _product(gc, hc, None, ctx.types[0])
        dx, dgain = _norm_backward(t, gain, r, dh, gsum, ctx.needs_input_grad[1])
        return dx, dgain, dw, db, None, dx if ctx.has_residual else None, None, None, None


def rms_norm_linear(x: torch.Tensor, norm_weight: torch.Tensor | None, weight: "torch.Tensor | BlockScaled",
                    bias: torch.Tensor | None = None, eps: float = 1e-6, residual: torch.Tensor | None = None) -> Any:
    """``scaled_linear(rms_norm(x + residual) , weight, bias)`` with the norm's output in 8 bits from the start: the
    normalised rows are quantised from their unrounded fp32 values and never stored otherwise.  Returns ``y``, or
    ``(y, x + residual)`` with a residual.  Differentiable like :func:`scaled_linear`; a prepared ``weight`` serves
    inference."""
    prepared = isinstance(weight, BlockScaled)
    if x.is_cuda:
        run = scaled_fused.prepared_norm_linear if prepared else scaled_fused.rms_norm_linear
        out = run(x, norm_weight, weight, bias, residual, eps)
        if out is not None:
            return out[0] if residual is None else out
    K, N, prepared = _check_linear("rms_norm_linear", x, weight, bias)
    _check("rms_norm_linear", x, norm_weight, residual, eps)
    _refuse_vmap("rms_norm_linear", norm_weight, residual)
    if (norm_weight is not None and norm_weight.dtype not in _HALF) or (residual is not None and residual.dtype not in _HALF):
        raise TypeError("rms_norm_linear takes fp32, bf16 or fp16 tensors")
    if prepared and _traced(norm_weight, residual):
        raise ValueError("rms_norm_linear: a prepared weight (BlockScaled) serves inference only; call it under torch.no_grad()")
    if residual is not None and residual.dtype != x.dtype:
        x, residual = _same_type(x, residual)
        return rms_norm_linear(x, norm_weight, weight, bias, eps, residual)
    out_dtype = _out_dtype(x)
    M = math.prod(x.shape[:-1])
    if M == 0 or N == 0 or K == 0:
        h, t, _ = _plain(x, norm_weight, residual, None, eps)
        w = weight.dequantize() if prepared else weight.float()
        y = torch.nn.functional.linear(h.float(), w, None if bias is None else bias.float()).to(out_dtype)
        return y if residual is None else (y, t)
    if prepared:
        q, t, _ = _norm_to_codes(x.detach(), norm_weight, eps, None if residual is None else residual.detach(), False)
        y = _product(q, weight, None if bias is None else bias.detach(), out_dtype)
        return y if residual is None else (y, t)
    gx, gn, gw, gr = _grads(x, norm_weight, weight, residual)
    out = _RmsNormLinear.apply(x.reshape(M, K), norm_weight, weight, bias, eps, None if residual is None else residual.reshape(M, K),
                               out_dtype, gx or gn or gr, gw)
    if residual is None:
        return out.view(*x.shape[:-1], N)
    return out[0].view(*x.shape[:-1], N), out[1].view(x.shape)
