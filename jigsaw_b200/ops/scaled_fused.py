"""Bindings of the 8-bit kernels: block quantisation and root-mean-square norm (``csrc/scaled_quant.cu``), matrix product
with block scales (``csrc/scaled_gemm.cu``).

The functions take two-dimensional CUDA tensors and return ``None`` (with a reason) where the kernels do not cover a call;
shapes and types are checked by the callers in ``jigsaw_b200.modules``.  Nothing is cached between calls: every buffer is
allocated for the call by torch, so calls on several streams and captured graphs share nothing.
"""

from __future__ import annotations

import ctypes
from typing import Any

import torch

from . import _lib, symm

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _call(fn: Any, dev: torch.device, *args: Any) -> None:
    """Launch on the current stream of the tensors' device, which need not be the current device."""
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc != 0:
        raise RuntimeError(f"jigsaw_b200 kernel launcher {fn.__name__} failed with code {rc}")


def _pitch(n: int) -> int:
    return (n + 15) // 16 * 16


def _new_codes(rows: int, cols: int, dev: torch.device) -> torch.Tensor:
    """``[rows, cols]`` codes whose rows start on 16-byte boundaries (the tensor memory accelerator's rule)."""
    t = torch.empty(rows, _pitch(cols), dtype=CODES, device=dev)
    return t if cols % 16 == 0 else t[:, :cols]


def _new_scales(rows: int, blocks: int, dev: torch.device) -> torch.Tensor:
    """``[rows, blocks]`` scales, rows contiguous: a warp of the product reads the scales of 32 rows in one request."""
    return torch.empty(blocks, rows, dtype=SCALES, device=dev).t()


def _rows_contiguous(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _covers(*tensors: torch.Tensor | None) -> bool:
    if not all(t is None or (t.is_cuda and t.dtype in TYPES) for t in tensors):
        return False
    if not _lib.available():
        raise RuntimeError("jigsaw_b200: the sm_100a kernel library is missing on a CUDA machine")
    return True


@_lib.traced("jb.maybe_fused_quantize")
@_lib.audited("quantize")
def maybe_fused_quantize(x: torch.Tensor, square: bool, rows: bool = True, cols: bool = False, rstd: torch.Tensor | None = None,
                         gain: torch.Tensor | None = None, colsum: torch.dtype | None = None) -> tuple | None:
    """Codes and scales of ``x [R, C]`` (of ``x * rstd[:, None] * gain`` when ``rstd`` is given), read once.

    Returns ``(codes, scales, codes_t, scales_t, column sums)``: the first pair for blocks along the rows (``rows``), the
    second for the transposed matrix in blocks along the columns (``cols``); ``square`` uses one scale per 128 x 128 for
    both.  The column sums of the unquantised values come in the type ``colsum``."""
    if not _covers(x, gain) or x.dim() != 2 or x.numel() == 0:
        return _lib.decline("needs a non-empty matrix in fp32, bf16 or fp16")
    if colsum is not None and colsum not in TYPES:
        return _lib.decline("column sums come in fp32, bf16 or fp16")
    x = _rows_contiguous(x)
    R, C, dev = x.shape[0], x.shape[1], x.device
    rb, cb = (R + 127) // 128, (C + 127) // 128
    L = _lib.lib()
    q = _lib.JbQuant()
    q.x, q.ldx, q.rows, q.cols, q.type, q.square = x.data_ptr(), x.stride(0), R, C, TYPES[x.dtype], int(square)
    codes = scales = codes_t = scales_t = part = None
    if square:
        scales = torch.empty(rb, cb, dtype=SCALES, device=dev)
        q.scales, q.scale_row, q.scale_k = scales.data_ptr(), cb, 1
        scales_t = scales.t()
    if rows:
        codes = _new_codes(R, C, dev)
        q.codes, q.pitch = codes.data_ptr(), codes.stride(0) if R > 1 else _pitch(C)
        if not square:
            scales = _new_scales(R, cb, dev)
            q.scales, q.scale_row, q.scale_k = scales.data_ptr(), 1, R
    if cols:
        codes_t = _new_codes(C, R, dev)
        q.codes_t, q.pitch_t = codes_t.data_ptr(), codes_t.stride(0) if C > 1 else _pitch(R)
        if not square:
            scales_t = _new_scales(C, rb, dev)
            q.scales_t, q.scale_t_row, q.scale_t_k = scales_t.data_ptr(), 1, C
    if rstd is not None:
        q.rstd, q.gain, q.gain_type = rstd.data_ptr(), _ptr(gain), 0 if gain is None else TYPES[gain.dtype]
    if colsum is not None:
        part = torch.empty(rb, C, dtype=torch.float32, device=dev)
        q.colsum = part.data_ptr()
    _call(L.jb_quantize, dev, ctypes.byref(q))
    _lib.count_launches(1)
    sums = None
    if part is not None:
        sums = torch.empty(C, dtype=colsum, device=dev)
        _call(L.jb_column_sum, dev, part.data_ptr(), rb, C, sums.data_ptr(), TYPES[colsum])
        _lib.count_launches(1)
    return codes, scales if rows else None, codes_t, scales_t if cols else None, sums


def _operand(codes: torch.Tensor, scales: torch.Tensor, square: bool) -> tuple:
    """The C struct of an operand, and the tensors that have to outlive the launch."""
    rows, K = codes.shape
    if (codes.stride(1) != 1 and K > 1) or (rows > 1 and codes.stride(0) % 16) or codes.data_ptr() % 16 or (rows > 1 and codes.stride(0) < K):
        fresh = _new_codes(rows, K, codes.device)
        fresh.view(torch.uint8).copy_(codes.view(torch.uint8))
        codes = fresh
    o = _lib.JbScaledOperand()
    o.codes, o.pitch = codes.data_ptr(), codes.stride(0) if rows > 1 else _pitch(K)
    o.scales, o.scale_row, o.scale_k, o.rows, o.square = scales.data_ptr(), scales.stride(0), scales.stride(1), rows, int(square)
    return o, codes


@_lib.traced("jb.maybe_fused_scaled_matmul")
@_lib.audited("scaled_matmul")
def maybe_fused_scaled_matmul(a_codes: torch.Tensor, a_scales: torch.Tensor, a_square: bool, b_codes: torch.Tensor,
                              b_scales: torch.Tensor, b_square: bool, bias: torch.Tensor | None,
                              out_dtype: torch.dtype) -> torch.Tensor | None:
    """``A B^T + bias`` for ``A [M, K]`` and ``B [N, K]`` in e4m3 codes with e8m0 block scales."""
    if not a_codes.is_cuda or out_dtype not in TYPES or not _covers(bias):
        return _lib.decline("needs CUDA operands and fp32, bf16 or fp16 bias and output")
    (M, K), N, dev = a_codes.shape, b_codes.shape[0], a_codes.device
    if M == 0 or N == 0 or K == 0:
        return _lib.decline("empty operand")
    out = torch.empty(M, N, dtype=out_dtype, device=dev)
    a, keep_a = _operand(a_codes, a_scales, a_square)
    b, keep_b = _operand(b_codes, b_scales, b_square)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    _call(_lib.lib().jb_scaled_gemm, dev, ctypes.byref(a), ctypes.byref(b), K, out.data_ptr(), N, TYPES[out_dtype], _ptr(bias),
          0 if bias is None else TYPES[bias.dtype], _lib.sm_count(dev.index), symm.arena(dev).status.data_ptr())
    _lib.count_launches(1)
    return out


@_lib.traced("jb.maybe_fused_rms_norm")
@_lib.audited("rms_norm")
def maybe_fused_rms_norm(x: torch.Tensor, gain: torch.Tensor | None, eps: float, residual: torch.Tensor | None,
                         out_dtype: torch.dtype | None, quantize: bool, keep_rstd: bool) -> tuple | None:
    """``(y, codes, scales, sum, rstd)`` of ``x [R, C]`` (+ ``residual``): ``y`` in ``out_dtype`` unless that is ``None``,
    8-bit codes with a scale per row and 128 columns if ``quantize``."""
    if not _covers(x, gain, residual) or x.numel() == 0:
        return _lib.decline("needs non-empty fp32, bf16 or fp16 tensors")
    R, C, dev = x.shape[0], x.shape[1], x.device
    L = _lib.lib()
    if C > L.jb_rms_max_cols() or out_dtype not in (None, torch.float32, x.dtype):
        return _lib.decline("rows longer than the kernel keeps in registers, or another output type")
    x = _rows_contiguous(x)
    q = _lib.JbRms()
    q.x, q.ldx, q.rows, q.cols, q.type, q.eps = x.data_ptr(), x.stride(0), R, C, TYPES[x.dtype], eps
    if gain is not None:
        gain = gain.contiguous()
        q.gain, q.gain_type = gain.data_ptr(), TYPES[gain.dtype]
    total = y = codes = scales = rstd = None
    if residual is not None:
        residual = _rows_contiguous(residual)
        total = torch.empty(R, C, dtype=x.dtype, device=dev)
        q.residual, q.ldr, q.sum = residual.data_ptr(), residual.stride(0), total.data_ptr()
    if keep_rstd:
        rstd = torch.empty(R, dtype=torch.float32, device=dev)
        q.rstd = rstd.data_ptr()
    if out_dtype is not None:
        y = torch.empty(R, C, dtype=out_dtype, device=dev)
        q.y, q.y_type = y.data_ptr(), TYPES[out_dtype]
    if quantize:
        codes, scales = _new_codes(R, C, dev), _new_scales(R, (C + 127) // 128, dev)
        q.codes, q.pitch = codes.data_ptr(), codes.stride(0) if R > 1 else _pitch(C)
        q.scales, q.scale_row, q.scale_k = scales.data_ptr(), 1, R
    _call(L.jb_rms_norm_fwd, dev, ctypes.byref(q))
    _lib.count_launches(1)
    return y, codes, scales, total, rstd


def rms_norm_backward(t: torch.Tensor, rstd: torch.Tensor, gain: torch.Tensor | None, g: torch.Tensor,
                      gsum: torch.Tensor | None, want_gain: bool) -> tuple:
    """``(gradient of the normalised sum t, gradient of the gain)`` for ``y = t * rstd * gain``; ``g`` is the gradient of
    ``y`` in the type of ``t`` or in fp32, ``gsum`` a gradient that reaches ``t`` on its own."""
    R, C, dev = t.shape[0], t.shape[1], t.device
    L = _lib.lib()
    sm = _lib.sm_count(dev.index)
    g = g.contiguous()
    q = _lib.JbRmsBwd()
    q.t, q.ldt, q.rows, q.cols, q.type = t.data_ptr(), t.stride(0), R, C, TYPES[t.dtype]
    q.g, q.g_f32, q.rstd = g.data_ptr(), int(g.dtype == torch.float32), rstd.data_ptr()
    if gsum is not None:
        gsum = gsum.to(t.dtype).contiguous()
        q.gsum = gsum.data_ptr()
    if gain is not None:
        gain = gain.contiguous()
        q.gain, q.gain_type = gain.data_ptr(), TYPES[gain.dtype]
    dx = torch.empty(R, C, dtype=t.dtype, device=dev)
    q.dx = dx.data_ptr()
    dgain = part = None
    if want_gain and gain is not None:
        parts = L.jb_rms_bwd_parts(R, C, sm)
        part = torch.empty(parts, C, dtype=torch.float32, device=dev)
        q.part = part.data_ptr()
    _call(L.jb_rms_norm_bwd, dev, ctypes.byref(q), sm)
    _lib.count_launches(1)
    if part is not None and gain is not None:
        dgain = torch.empty(C, dtype=gain.dtype, device=dev)
        _call(L.jb_column_sum, dev, part.data_ptr(), part.shape[0], C, dgain.data_ptr(), TYPES[gain.dtype])
        _lib.count_launches(1)
    return dx, dgain
