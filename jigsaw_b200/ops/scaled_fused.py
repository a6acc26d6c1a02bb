"""The 8-bit kernels: block quantisation and root-mean-square norm (``csrc/scaled_quant.cu``), matrix product with block
scales (``csrc/scaled_gemm.cu``), and the layers made of them.

Buffers, launches and backward passes are driven by the native torch binding (``csrc/torch_binding.cpp``): a training step
of one layer is seven launches, which from Python take several times as long as the kernels on a short batch.  A function
here answers ``None`` to a call that the kernels do not cover or whose arguments do not fit; the callers in
``jigsaw_b200.modules`` then raise the error, or compute the call in torch operations and say so to :func:`declined`.
Nothing is kept between calls: every buffer comes from torch's allocator for the call, so calls on
several streams and captured graphs share nothing.
"""

from __future__ import annotations

from typing import Any

import torch

from . import _build, _lib, symm

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ENTRY = ("jb_scaled_gemm", "jb_quantize", "jb_column_sum", "jb_rms_max_cols", "jb_rms_norm_fwd", "jb_rms_bwd_parts", "jb_rms_norm_bwd")


_native: Any = None


def native() -> Any:
    """The torch binding, with the entry points of the kernel library; raises if either is missing."""
    global _native
    if _native is None:
        import ctypes

        m = _build.load_binding()
        L = _lib.lib()
        m.init({name: ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in _ENTRY})
        _lib.add_launch_counter(m.launches)
        _native = m
    return _native


_status_known: set[int] = set()


def _on(t: torch.Tensor) -> Any:
    """The binding, ready for the device of ``t``."""
    m = _native or native()
    idx = t.get_device()
    if idx not in _status_known:
        m.set_status(idx, symm.arena(t.device).status)
        _status_known.add(idx)
    return m


def _answer(name: str, out: Any) -> Any:
    """Counts a call that ran on the kernels; ``None`` (not covered) goes back to the caller."""
    if out is not None:
        _lib.record(name, True)
    return out


def declined(name: str, why: str) -> None:
    """Counts a call on CUDA tensors that torch operations compute; raises under strict dispatch."""
    _lib.decline(why)
    _lib.record(name, False)


@_lib.traced("jb.quantize")
def quantize(x: torch.Tensor, square: bool) -> tuple | None:
    """``(codes, scales)`` of a tensor in blocks along its last axis, or of a matrix in squares."""
    return _answer("quantize", (_native or native()).quantize_any(x, square))


@_lib.traced("jb.quantize")
def quantize_both(x: torch.Tensor, square: bool, rows: bool = True, cols: bool = False, rstd: torch.Tensor | None = None,
                  gain: torch.Tensor | None = None, colsum: torch.dtype | None = None) -> tuple | None:
    """Codes and scales of a matrix (of ``x * rstd[:, None] * gain`` when ``rstd`` is given), read once.

    Returns ``(codes, scales, codes_t, scales_t, column sums)``: the first pair for blocks along the rows (``rows``), the
    second for the transposed matrix in blocks along the columns (``cols``); ``square`` uses one scale per 128 x 128 for
    both.  The column sums of the unquantised values come in the type ``colsum``."""
    return _answer("quantize", (_native or native()).quantize(x, square, rows, cols, rstd, gain, -1 if colsum is None else TYPES[colsum]))


@_lib.traced("jb.scaled_matmul")
def scaled_matmul(a: Any, b: Any, bias: torch.Tensor | None, out_dtype: torch.dtype) -> torch.Tensor | None:
    """``A B^T + bias`` for ``A [..., K]`` and ``B [N, K]`` in e4m3 codes with e8m0 block scales."""
    return _answer("scaled_matmul", _on(a.codes).scaled_matmul(a.codes, a.scales, a.block[0] > 1, b.codes, b.scales, b.block[0] > 1,
                                                               bias, TYPES[out_dtype]))


@_lib.traced("jb.scaled_linear")
def scaled_linear(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None) -> torch.Tensor | None:
    """Differentiable 8-bit linear layer."""
    return _answer("scaled_linear", _on(x).scaled_linear(x, w, b))


@_lib.traced("jb.scaled_linear")
def prepared_linear(x: torch.Tensor, w: Any, b: torch.Tensor | None) -> torch.Tensor | None:
    """Inference with a prepared weight; not covered where a gradient is wanted."""
    return _answer("scaled_linear", _on(x).linear_prepared(x, w.codes, w.scales, w.block[0] > 1, b))


@_lib.traced("jb.rms_norm")
def rms_norm(x: torch.Tensor, gain: torch.Tensor | None, residual: torch.Tensor | None, eps: float) -> tuple | None:
    """Differentiable ``(y, x + residual)``."""
    return _answer("rms_norm", _on(x).rms_norm(x, gain, residual, eps))


@_lib.traced("jb.rms_norm_quantize")
def rms_norm_quantize(x: torch.Tensor, gain: torch.Tensor | None, eps: float, residual: torch.Tensor | None,
                      keep_rstd: bool) -> tuple | None:
    """``(codes, scales, x + residual, r)`` with a scale per row and 128 columns."""
    return _answer("rms_norm_quantize", (_native or native()).rms_quantize(x, gain, eps, residual, keep_rstd))


@_lib.traced("jb.rms_norm_linear")
def rms_norm_linear(x: torch.Tensor, gain: torch.Tensor | None, w: torch.Tensor, b: torch.Tensor | None,
                    residual: torch.Tensor | None, eps: float) -> tuple | None:
    """Differentiable ``(y, x + residual)``."""
    return _answer("rms_norm_linear", _on(x).rms_norm_linear(x, gain, w, b, residual, eps))


@_lib.traced("jb.rms_norm_linear")
def prepared_norm_linear(x: torch.Tensor, gain: torch.Tensor | None, w: Any, b: torch.Tensor | None,
                         residual: torch.Tensor | None, eps: float) -> tuple | None:
    """Inference with a prepared weight: ``(y, x + residual)`` in two launches; not covered where a gradient is wanted."""
    return _answer("rms_norm_linear", _on(x).norm_linear_prepared(x, gain, eps, residual, w.codes, w.scales, w.block[0] > 1, b))
