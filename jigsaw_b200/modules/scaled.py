"""The 8-bit token path: root-mean-square norm, block quantisation and matrix products in 8-bit floating point.

=========================  ======================================================================================
``DistributedRMSNorm``     root-mean-square norm layer, feature axis cut over a column group, optional residual
``distributed_rms_norm``   its function form
``BlockScaled``            a matrix as e4m3 codes with one power-of-two scale per block of 128 (or 128 x 128)
``quantize_blockwise``     makes one
``scaled_matmul``          product of two, fp32 accumulation
``scaled_linear``          differentiable linear layer whose three products run in 8 bits
``rms_norm_quantize``      norm (with the residual's addition) whose output is a ``BlockScaled``; inference
``rms_norm_linear``        norm and 8-bit linear layer in one, differentiable
=========================  ======================================================================================

``DistributedLinear`` takes the path with ``LinearConfig(..., precision="fp8")``, ``ViT`` with
``ViTConfig(norm="rms", linear_precision="fp8")``.  A weight that serves inference is prepared once::

    w8 = scaled.quantize_blockwise(layer.weight, (128, 128))
    with torch.no_grad():
        y, h = scaled.rms_norm_linear(x, norm.weight, w8, layer.bias, residual=h)

The functions are importable from ``modules.functional`` as well.  The reference has no counterpart of this path.
"""

from .._core.public import set_module
from .linear._scaled import BlockScaled, quantize_blockwise, scaled_linear, scaled_matmul
from .normalization._rms_functional import distributed_rms_norm, rms_norm_linear, rms_norm_quantize
from .normalization._rms_norm import DistributedRMSNorm

__all__ = [
    "BlockScaled",
    "DistributedRMSNorm",
    "distributed_rms_norm",
    "quantize_blockwise",
    "rms_norm_linear",
    "rms_norm_quantize",
    "scaled_linear",
    "scaled_matmul",
]

set_module(globals(), __all__)
