"""The 8-bit kernels: block quantisation and root-mean-square norm (``csrc/scaled_quant.cu``), matrix product with block
scales (``csrc/scaled_gemm.cu``), and the layers made of them.

Buffers, launches and backward passes are driven by the native torch binding (``csrc/torch_binding.cpp``): a training step
of one layer is seven launches, which from Python take several times as long as the kernels on a short batch.  The functions
here decide whether the kernels cover a call (``None`` otherwise); shapes are checked by the callers in
``jigsaw_b200.modules``.  Nothing is kept between calls: every buffer comes from torch's allocator for the call, so calls on
several streams and captured graphs share nothing.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Any

import torch

from . import _build, _lib, symm

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ENTRY = ("jb_scaled_gemm", "jb_quantize", "jb_column_sum", "jb_rms_norm_fwd", "jb_rms_bwd_parts", "jb_rms_norm_bwd")


@lru_cache(maxsize=1)
def native() -> Any:
    """The torch binding, with the entry points of the kernel library; raises if either is missing."""
    import ctypes

    m = _build.load_binding()
    L = _lib.lib()
    m.init({name: ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRY})
    _lib.add_launch_counter(m.launches)
    return m


_max_cols = 0


def max_cols() -> int:
    """Longest row that the norm kernels keep in registers."""
    global _max_cols
    if not _max_cols:
        _max_cols = int(_lib.lib().jb_rms_max_cols())
    return _max_cols


def _status(t: torch.Tensor) -> torch.Tensor:
    return symm.arena(t.device).status


def _ran(name: str, out: Any) -> Any:
    _lib.record(name, True)
    return out


def _declined(name: str, why: str) -> None:
    _lib.decline(why)
    _lib.record(name, False)
    return None


def _norm_covers(x: torch.Tensor) -> bool:
    return x.shape[-1] <= max_cols()


@_lib.traced("jb.quantize")
def maybe_fused_quantize(x: torch.Tensor, square: bool, rows: bool = True, cols: bool = False, rstd: torch.Tensor | None = None,
                         gain: torch.Tensor | None = None, colsum: torch.dtype | None = None) -> tuple | None:
    """Codes and scales of the rows of ``x`` (of ``x * rstd[:, None] * gain`` when ``rstd`` is given), read once.

    Returns ``(codes, scales, codes_t, scales_t, column sums)``: the first pair for blocks along the rows (``rows``), the
    second for the transposed matrix in blocks along the columns (``cols``); ``square`` uses one scale per 128 x 128 for
    both.  The column sums of the unquantised values come in the type ``colsum``."""
    if x.dtype not in TYPES or x.numel() == 0:
        return _declined("quantize", "needs a non-empty tensor in fp32, bf16 or fp16")
    return _ran("quantize", native().quantize(x, square, rows, cols, rstd, gain, -1 if colsum is None else TYPES[colsum]))


@_lib.traced("jb.scaled_matmul")
def maybe_fused_scaled_matmul(a: Any, b: Any, bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor | None:
    """``A B^T + bias`` for ``A [..., K]`` and ``B [N, K]`` in e4m3 codes with e8m0 block scales."""
    if a.codes.numel() == 0 or b.codes.numel() == 0 or out_dtype not in TYPES or (bias is not None and bias.dtype not in TYPES):
        return _declined("scaled_matmul", "needs non-empty operands and fp32, bf16 or fp16 bias and output")
    return _ran("scaled_matmul", native().scaled_matmul(a.codes, a.scales, a.block[0] > 1, b.codes, b.scales, b.block[0] > 1, bias,
                                                        TYPES[out_dtype], _status(a.codes)))


@_lib.traced("jb.scaled_linear")
def maybe_fused_scaled_linear(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None, out_dtype: torch.dtype, need_x: bool,
                              need_w: bool) -> torch.Tensor | None:
    """Differentiable 8-bit linear layer; ``need_x`` / ``need_w``: the input / the weight will want a gradient."""
    return _ran("scaled_linear", native().scaled_linear(x, w, b, TYPES[out_dtype], need_x, need_w, _status(x)))


def prepared_linear(x: torch.Tensor, w: Any, b: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor:
    """Inference with a prepared weight."""
    return _ran("scaled_linear", native().linear_prepared(x, w.codes, w.scales, w.block[0] > 1, b, TYPES[out_dtype], _status(x)))


@_lib.traced("jb.rms_norm")
def maybe_fused_rms_norm(x: torch.Tensor, gain: torch.Tensor | None, residual: torch.Tensor | None, eps: float,
                         out_dtype: torch.dtype, need: bool) -> tuple | None:
    """Differentiable ``(y, x + residual)``; ``need``: some tensor will want a gradient."""
    if not _norm_covers(x) or out_dtype not in (torch.float32, x.dtype):
        return _declined("rms_norm", "rows longer than the kernel keeps in registers, or another output type")
    return _ran("rms_norm", native().rms_norm(x, gain, residual, eps, TYPES[out_dtype], need))


@_lib.traced("jb.rms_norm_quantize")
def maybe_fused_rms_quantize(x: torch.Tensor, gain: torch.Tensor | None, eps: float, residual: torch.Tensor | None,
                             keep_rstd: bool) -> tuple | None:
    """``(codes, scales, x + residual, r)`` with a scale per row and 128 columns."""
    if not _norm_covers(x):
        return _declined("rms_norm_quantize", "rows longer than the kernel keeps in registers")
    return _ran("rms_norm_quantize", native().rms_quantize(x, gain, eps, residual, keep_rstd))


@_lib.traced("jb.rms_norm_linear")
def maybe_fused_rms_norm_linear(x: torch.Tensor, gain: torch.Tensor | None, w: torch.Tensor, b: torch.Tensor | None,
                                residual: torch.Tensor | None, eps: float, out_dtype: torch.dtype, need_h: bool,
                                need_w: bool) -> tuple | None:
    """Differentiable ``(y, x + residual)``; ``need_h``: something in front of the product will want a gradient."""
    if not _norm_covers(x):
        return _declined("rms_norm_linear", "rows longer than the kernel keeps in registers")
    return _ran("rms_norm_linear", native().rms_norm_linear(x, gain, w, b, residual, eps, TYPES[out_dtype], need_h, need_w, _status(x)))


def maybe_prepared_norm_linear(x: torch.Tensor, gain: torch.Tensor | None, w: Any, b: torch.Tensor | None,
                               residual: torch.Tensor | None, eps: float, out_dtype: torch.dtype) -> tuple | None:
    """Inference with a prepared weight: ``(y, x + residual)`` in two launches."""
    if not _norm_covers(x):
        return _declined("rms_norm_linear", "rows longer than the kernel keeps in registers")
    return _ran("rms_norm_linear", native().norm_linear_prepared(x, gain, eps, residual, w.codes, w.scales, w.block[0] > 1, b,
                                                                 TYPES[out_dtype], _status(x)))
