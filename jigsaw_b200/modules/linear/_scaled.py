"""8-bit matrix products with block scales: quantisation, product, differentiable linear layer.

A matrix is held as e4m3 codes with one power-of-two scale per block, either 1 x 128 along the last axis (activations,
gradients) or 128 x 128 (weights, whose transpose then shares the scales).  The scale of a block whose largest finite
magnitude is ``A`` is the smallest power of two ``s`` with ``A <= 448 s`` (448 is the largest e4m3 value), at least
2^-116, and 1 for a block of zeros; a code is ``v / s`` rounded to nearest even.  Infinities and NaN become NaN codes
and do not count towards ``A``.

Because the scales are powers of two, dividing by them is exact, the codes are determined by the definition alone (the
CUDA kernels and the torch operations below give the same bits), and the tensor cores apply them inside the product.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..._core.autocast import autocast_dtype
from ...ops import scaled_fused

BLOCK = 128
ROW, SQUARE = (1, BLOCK), (BLOCK, BLOCK)
_HALF = (torch.float32, torch.bfloat16, torch.float16)
_batched = torch._C._functorch.is_batchedtensor


@dataclass(frozen=True, eq=False)
class BlockScaled:
    """A matrix in 8 bits: ``codes`` (``float8_e4m3fn``, ``[..., C]``), ``scales`` (``float8_e8m0fnu``) and the ``block`` that
    shares a scale, ``(1, 128)`` (scales ``[..., ceil(C / 128)]``) or ``(128, 128)`` (two dimensions, scales
    ``[ceil(R / 128), ceil(C / 128)]``).  Its values are ``codes * scales``; it carries no gradient."""

    codes: torch.Tensor
    scales: torch.Tensor
    block: tuple[int, int] = ROW

    def __post_init__(self) -> None:
        c, s = self.codes, self.scales
        if c.dtype != torch.float8_e4m3fn or s.dtype != torch.float8_e8m0fnu:
            raise TypeError(f"BlockScaled holds float8_e4m3fn codes and float8_e8m0fnu scales, got {c.dtype} and {s.dtype}")
        if c.dim() == 0:
            raise ValueError("codes need at least one dimension")
        want = _scale_shape(c.shape, self.block)
        if tuple(s.shape) != want:
            raise ValueError(f"codes of shape {tuple(c.shape)} in blocks of {self.block} need scales of shape {want}, got {tuple(s.shape)}")
        if c.device != s.device:
            raise ValueError(f"codes on {c.device}, scales on {s.device}")

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, rounded to ``dtype`` (fp32 and bf16 hold them exactly)."""
        return _values(self.codes, self.scales, self.block).to(dtype)


def _made(codes: torch.Tensor, scales: torch.Tensor, block: tuple[int, int]) -> BlockScaled:
    """A ``BlockScaled`` of parts that belong together (no checks)."""
    q = object.__new__(BlockScaled)
    put = object.__setattr__
    put(q, "codes", codes)
    put(q, "scales", scales)
    put(q, "block", block)
    return q


def _check_block(block: tuple[int, int]) -> tuple[int, int]:
    if block == ROW or block == SQUARE:
        return block
    block = tuple(block)
    if block not in (ROW, SQUARE):
        raise ValueError(f"blocks are (1, 128) or (128, 128), got {block}")
    return block


def _scale_shape(shape: torch.Size, block: tuple[int, int]) -> tuple[int, ...]:
    nb = -(-shape[-1] // BLOCK)
    if _check_block(block) == ROW:
        return (*shape[:-1], nb)
    if len(shape) != 2:
        raise ValueError(f"blocks of (128, 128) need a matrix, got {len(shape)} dimensions")
    return (-(-shape[0] // BLOCK), nb)


# ----------------------------------------------------------------------------- the definition, in torch operations
def _quantize_plain(x: torch.Tensor, block: tuple[int, int]) -> tuple[torch.Tensor, torch.Tensor]:
    R, C = x.shape
    br, bc = block
    nr, nc = -(-R // br), -(-C // bc)
    v = torch.nn.functional.pad(x.float(), (0, nc * bc - C, 0, nr * br - R)).view(nr, br, nc, bc)
    if v.numel() == 0:
        return x.new_empty(R, C, dtype=torch.float8_e4m3fn), x.new_empty(nr, nc, dtype=torch.float8_e8m0fnu)
    mag = v.abs()
    amax = torch.where(mag < math.inf, mag, 0.0).amax(dim=(1, 3))
    m, e = torch.frexp(amax)                                    # amax = m 2^e with m in [.5, 1), and 448 = .875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-116)
    e = torch.where(amax == 0, 0, e).to(torch.int32) + 127
    q = v / (e << 23).view(torch.float32)[:, None, :, None]
    q = torch.where(mag < math.inf, q, math.nan)                # infinities become NaN
    codes = q.reshape(nr * br, nc * bc)[:R, :C].to(torch.float8_e4m3fn)
    return codes, e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(codes: torch.Tensor, scales: torch.Tensor, block: tuple[int, int]) -> torch.Tensor:
    C = codes.shape[-1]
    s = scales.float()
    if block[0] > 1:
        s = s.repeat_interleave(BLOCK, 0)[: codes.shape[0]]
    return codes.float() * s.repeat_interleave(BLOCK, -1)[..., :C]


# ----------------------------------------------------------------------------- kernels or definition
def _quantize_2d(x: torch.Tensor, block: tuple[int, int], rows: bool = True, cols: bool = False,
                 rstd: torch.Tensor | None = None, gain: torch.Tensor | None = None,
                 colsum: torch.dtype | None = None) -> tuple[BlockScaled | None, BlockScaled | None, torch.Tensor | None]:
    """``x [R, C]`` (times ``rstd`` per row and ``gain`` per column) in blocks along its rows, its transpose in blocks along the
    columns of ``x``, and the column sums of the values."""
    if x.is_cuda:
        out = scaled_fused.quantize_both(x, block == SQUARE, rows, cols, rstd, gain, colsum)
        if out is not None:
            c, s, ct, st, sums = out
            return (None if c is None else _made(c, s, block)), (None if ct is None else _made(ct, st, block)), sums
        scaled_fused.declined("quantize", "outside the coverage of the kernel")
    v = x
    if rstd is not None:
        v = v.float() * rstd[:, None]
        v = v if gain is None else v * gain.float()
    return (
        BlockScaled(*_quantize_plain(v, block), block) if rows else None,
        BlockScaled(*_quantize_plain(v.t(), block), block) if cols else None,
        None if colsum is None else v.sum(dim=0, dtype=torch.promote_types(v.dtype, torch.float32)).to(colsum),
    )


def _product(a: BlockScaled, b: BlockScaled, bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    """``a [..., K] b [N, K]^T + bias``."""
    if a.codes.is_cuda:
        out = scaled_fused.scaled_matmul(a, b, bias, out_dtype)
        if out is not None:
            return out
        scaled_fused.declined("scaled_matmul", "outside the coverage of the kernel")
    y = a.dequantize() @ b.dequantize().t()
    if bias is not None:
        y = y + bias.float()
    return y.to(out_dtype)


# ----------------------------------------------------------------------------- public functions
def _refuse_vmap(name: str, *tensors: Any) -> None:
    for t in tensors:
        if t is not None and _batched(t):
            raise NotImplementedError(f"{name} has no batching rule for torch.vmap; give it the members as leading dimensions")


def quantize_blockwise(x: torch.Tensor, block: tuple[int, int] = ROW) -> BlockScaled:
    """``x`` in e4m3 codes with one power-of-two scale per ``block``: ``(1, 128)`` along the last axis of a tensor of any number
    of dimensions, or ``(128, 128)`` of a matrix.  Blocks at the end of an axis may be shorter.  fp32, bf16 and fp16 run on
    one kernel launch on CUDA; other floating types are converted to fp32 first.  The result carries no gradient."""
    block = _check_block(block)
    if x.is_cuda:
        out = scaled_fused.quantize(x, block is SQUARE or block == SQUARE)
        if out is not None:
            return _made(out[0], out[1], block)
    _refuse_vmap("quantize_blockwise", x)
    if not x.is_floating_point() or x.element_size() == 1:
        raise TypeError(f"quantize_blockwise takes fp64, fp32, bf16 or fp16 tensors, got {x.dtype}")
    dims = x.dim()
    if dims == 0:
        raise ValueError("quantize_blockwise needs at least one dimension")
    if dims != 2 and block == SQUARE:
        raise ValueError(f"blocks of (128, 128) need a matrix, got {dims} dimensions")
    if x.dtype == torch.float64:
        return quantize_blockwise(x.float(), block)
    if x.numel() == 0:
        shape = _scale_shape(x.shape, block)
        return _made(x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(shape, dtype=torch.float8_e8m0fnu), block)
    if x.is_cuda:
        scaled_fused.declined("quantize", "outside the coverage of the kernel")
    if dims == 2:
        return _made(*_quantize_plain(x.detach(), block), block)
    codes, scales = _quantize_plain(x.detach().reshape(-1, x.shape[-1]), block)
    return _made(codes.view(x.shape), scales.view(*x.shape[:-1], scales.shape[-1]), block)


def _check_bias(bias: torch.Tensor | None, n: int, device: torch.device) -> None:
    if bias is None:
        return
    if bias.shape != (n,):
        raise ValueError(f"bias of shape {tuple(bias.shape)} for {n} output features")
    if bias.device != device:
        raise ValueError(f"bias on {bias.device}, operands on {device}")


def scaled_matmul(a: BlockScaled, b: BlockScaled, bias: torch.Tensor | None = None,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T + bias`` of two matrices in 8 bits, ``a [..., K]`` and ``b [N, K]`` (weights keep the layout of
    ``torch.nn.Linear``), each with scales per row or per square of 128.  Products and sums are those of the values
    ``codes * scales`` with fp32 accumulation; the result is rounded once, to ``out_dtype`` (fp32, bf16 or fp16).  Not
    differentiable: :func:`scaled_linear` is the form with gradients."""
    if not isinstance(a, BlockScaled) or not isinstance(b, BlockScaled):
        raise TypeError("scaled_matmul takes BlockScaled operands (see quantize_blockwise)")
    if a.codes.is_cuda and out_dtype in _HALF:
        out = scaled_fused.scaled_matmul(a, b, bias, out_dtype)
        if out is not None:
            return out
    _refuse_vmap("scaled_matmul", a.codes, a.scales, b.codes, b.scales, bias)
    sa, sb = a.codes.shape, b.codes.shape
    if len(sb) != 2:
        raise ValueError(f"b needs two dimensions, got {len(sb)}")
    if sa[-1] != sb[1]:
        raise ValueError(f"reduction sizes differ: {sa[-1]} vs {sb[1]}")
    if a.codes.device != b.codes.device:
        raise ValueError(f"operands on {a.codes.device} and {b.codes.device}")
    if out_dtype not in _HALF:
        raise TypeError(f"out_dtype is fp32, bf16 or fp16, got {out_dtype}")
    n = sb[0]
    if bias is not None:
        _check_bias(bias, n, a.codes.device)
    if a.codes.numel() == 0 or n == 0:
        y = torch.zeros(*sa[:-1], n, dtype=torch.float32, device=a.codes.device)
        return (y if bias is None else y + bias.detach().float()).to(out_dtype)
    return _product(a, b, None if bias is None else bias.detach(), out_dtype)


class _ScaledLinear(torch.autograd.Function):
    """``y = q(x) q(w)^T + b`` and its gradients as two more 8-bit products: ``dx = q(g) q(w)`` with blocks of ``g`` along the
    output features, ``dw = q(g^T) q(x^T)^T`` with blocks of both along the tokens.  (CUDA calls take the native form of the
    same function.)"""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None, out_dtype: torch.dtype, need_x: bool,
                need_w: bool) -> torch.Tensor:
        xr, xc, _ = _quantize_2d(x, ROW, cols=need_w)
        wr, wc, _ = _quantize_2d(w, SQUARE, cols=need_x)
        ctx.save_for_backward(*((xc.codes, xc.scales) if xc is not None else (None, None)),
                              *((wc.codes, wc.scales) if wc is not None else (None, None)))
        ctx.types = (x.dtype, w.dtype, None if b is None else b.dtype)
        return _product(xr, wr, b, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, g: torch.Tensor) -> tuple:
        xc, xs, wc, ws = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        want_x, want_w = want_x and wc is not None, want_w and xc is not None
        tx, tw, tb = ctx.types
        want_b = want_b and tb is not None
        dx = dw = db = None
        if want_x or want_w:
            gr, gc, db = _quantize_2d(g, ROW, rows=want_x, cols=want_w, colsum=tb if want_b else None)
            if want_x:
                dx = _product(gr, BlockScaled(wc, ws, SQUARE), None, tx)
            if want_w:
                dw = _product(gc, BlockScaled(xc, xs, ROW), None, tw)
        elif want_b:
            db = g.sum(dim=0, dtype=torch.float32).to(tb)
        return dx, dw, db, None, None, None


def _check_linear(name: str, x: torch.Tensor, weight: "torch.Tensor | BlockScaled", bias: torch.Tensor | None) -> tuple:
    """Checks of the linear entry points; returns ``(K, N, prepared)``."""
    prepared = isinstance(weight, BlockScaled)
    wc = weight.codes if prepared else weight
    _refuse_vmap(name, x, wc, bias)
    if wc.dim() != 2:
        raise ValueError(f"{name}: weight needs two dimensions [out, in], got {wc.dim()}")
    N, K = wc.shape
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"{name}: input of shape {tuple(x.shape)} for a weight of shape {tuple(wc.shape)}")
    if x.dtype not in _HALF or (not prepared and wc.dtype not in _HALF) or (bias is not None and bias.dtype not in _HALF):
        raise TypeError(f"{name} takes fp32, bf16 or fp16 tensors")
    if x.device != wc.device:
        raise ValueError(f"{name}: input on {x.device}, weight on {wc.device}")
    _check_bias(bias, N, x.device)
    if prepared and _traced(x, bias):
        raise ValueError(f"{name}: a prepared weight (BlockScaled) serves inference only; call it under torch.no_grad()")
    return K, N, prepared


def _grads(*tensors: torch.Tensor | None) -> tuple[bool, ...]:
    on = torch.is_grad_enabled()
    return tuple(on and t is not None and t.requires_grad for t in tensors)


def _traced(*tensors: torch.Tensor | None) -> bool:
    """A derivative is asked for: a gradient, or a tangent of forward mode."""
    if any(_grads(*tensors)):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def scaled_linear(x: torch.Tensor, weight: "torch.Tensor | BlockScaled", bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` with all matrix products in 8 bits: ``x [..., K]`` is quantised per row and 128 features,
    ``weight [N, K]`` per 128 x 128.  Differentiable: the two gradient products are 8-bit products of the same kind, with
    the output gradient (and, for the weight gradient, ``x``) quantised along the axis that is summed; the bias gradient is
    the fp32 sum.  Sums are fp32; the output has the autocast type or that of ``x``, gradients the types of their tensors.

    ``weight`` may be prepared once with ``quantize_blockwise(weight, (128, 128))`` for inference."""
    prepared = isinstance(weight, BlockScaled)
    if x.is_cuda:
        out = scaled_fused.prepared_linear(x, weight, bias) if prepared else scaled_fused.scaled_linear(x, weight, bias)
        if out is not None:
            return out
    K, N, prepared = _check_linear("scaled_linear", x, weight, bias)
    out_dtype = _out_dtype(x)
    M = math.prod(x.shape[:-1])
    if M == 0 or N == 0 or K == 0:
        w = weight.dequantize(x.dtype) if prepared else weight.to(x.dtype)
        return torch.nn.functional.linear(x, w, None if bias is None else bias.to(x.dtype)).to(out_dtype)
    if prepared:
        return _product(quantize_blockwise(x), weight, None if bias is None else bias.detach(), out_dtype)
    need_x, need_w = _grads(x, weight)
    y = _ScaledLinear.apply(x.reshape(M, K), weight, bias, out_dtype, need_x, need_w)
    return y.view(*x.shape[:-1], N)


def _out_dtype(x: torch.Tensor) -> torch.dtype:
    """The autocast type, or that of ``x``."""
    dt = autocast_dtype(x.device.type)
    return dt if dt in _HALF else x.dtype
