"""Residual addition, RMS norm and an 8-bit output with scales (B200).

``residual_rms_quant`` is the prologue of a block without adaLN tables and without
the ConvRot rotation: its INT8 codes and row scales are what ``ops.gemm.int8_linear``
takes.  One pass through ``h3_rms_quant_run`` of libh3sk_b200.so:

    h = round(x + residual)                     in x's type; h is x without a residual
    y = h * weight / sqrt(mean(h^2) + eps)      FP32
    scale = max(max|y| / top, 1e-30)            top = 127 (INT8) or 448 (E4M3)
    codes = round(y / scale)                    to nearest, ties to even

Rows whose h, or whose y in FP32, are not all finite get a NaN scale; the other rows are
unaffected.  Rows whose squares pass FP32 are computed smaller by a power of two.
Inference only, like every op of this package: nothing is recorded for autograd.
"""
from __future__ import annotations

import torch

from .. import _lib

CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}


def residual_rms_quant(x, weight, *, residual=None, eps=1e-6, dtype=torch.int8, residual_out=None, out=None,
                       out_scale=None):
    """Codes [M, K] and FP32 scales [M, 1] of the RMS norm of h = x + residual, and h.

    x, residual: BF16 or FP16 [M, K], unit column stride, rows K or more apart, K from 1
    to 16384, M from 0.  weight: [K] of x's type or FP32.  residual_out takes h and may be
    ``residual`` or ``x`` themselves (in place); a new tensor is made by default.
    dtype: torch.int8 or torch.float8_e4m3fn.  Returns (codes, scale, h)."""
    code = CODES.get(dtype)
    if code is None:
        raise ValueError('dtype must be torch.int8 or torch.float8_e4m3fn')
    return _lib.binding().rms_quant(x, weight, residual, eps, code, residual_out, out, out_scale)
