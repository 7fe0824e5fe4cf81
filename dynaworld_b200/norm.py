"""Root-mean-square norm of the decoder's token stream, with the residual's addition and an 8-bit
output, and row-wise 8-bit quantisation.

    h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight

The layers in front of the decoder heads (GaussianParameterHeads, src/train/gs_models/blocks.py)
are torch modules in the reference; these are the B200 kernels for them, next to ``linear``.
"""
from __future__ import annotations

import torch

from . import _token


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x + residual.

    x and residual [..., D], weight [D], all float32, bfloat16 or float16 of one type.  Returns y,
    or with a residual the pair (y, h): h is the new residual stream.  The sum, the statistics and
    the product are formed in float (a row whose squares add up past float's range, 3e38, gives zeros); y
    and h are rounded once.  Differentiable in x, weight and
    residual (once, in reverse mode; the backward forms h again from x and residual); the weight gradient is the same
    on every run."""
    return _token.ext().rms_norm(x, weight, residual, eps, _token.traced())


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``rms_norm`` with y in 8 bits for ``linear_fp8``: (codes [..., D] float8_e4m3fn, scale [...]
    float32), and h as the third value with a residual.  Per row top = max(max |y|, 1e-30),
    scale = top / 448 and code = e4m3(y * (448 / top)), from y in float.  A row with a NaN or an
    infinity stands for NaN.  Not differentiable."""
    return _token.ext().rms_norm_fp8(x, weight, residual, eps, _token.traced())


def quantize_rows_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., D] in 8 bits with one scale per row: (codes float8_e4m3fn, scale [...] float32), as
    ``rms_norm_fp8`` quantises its y.  For ``linear_fp8``: weights once, the activations between two
    8-bit products every step.  Not differentiable."""
    return _token.ext().quantize_rows_fp8(x, _token.traced())
