"""Matrix product with bias, activation and residual: the layers of the decoder's heads and
feed-forward blocks.

    y = act(x weight^T + bias) + residual

``linear`` takes float32, bfloat16 or float16 operands and is differentiable; ``linear_fp8`` takes
e4m3 codes with per-row scales (``rms_norm_fp8``, ``quantize_rows_fp8``) and serves only.  The
reference's heads (GaussianParameterHeads, src/train/gs_models/blocks.py:84-186) are torch layers;
these are the B200 kernels for them.
"""
from __future__ import annotations

import torch

from . import _token


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = act(x weight^T + bias) + residual, x [..., k], weight [n, k], bias [n], residual and y
    [..., n]; all float32, bfloat16 or float16 of one type.  ``activation``: "none", "relu",
    "gelu", "gelu_tanh" (its tanh form) or "silu".

    Sums, bias, activation and residual are formed in float and rounded once; on the tensor cores the
    additions of 16-bit (and e4m3) products truncate, about 2^-25 of the sum for every 16 (32) of k.
    Differentiable once in x, weight, bias and residual (reverse mode; tangents of forward mode are
    refused).  With an activation the forward keeps x weight^T + bias for the backward (float beside
    float32 operands, else float16), and the backward rounds dy act'(z) to the operands' type before its
    two products.  The same inputs give the same bits.  Rows may lie apart (any row stride); other
    layouts are copied.  float32 products of more than 8 rows (64 with at most 8 MB of weights), and the
    backward's, take their operands as sums of three bfloat16 parts, as exact as float32 sums (two
    infinities multiplied give NaN there).  An infinite sum gives what the activation's formula gives
    (-infinity: NaN with GELU and SiLU, 0 with ReLU)."""
    return _token.ext().linear(x, weight, bias, residual, activation, _token.traced())


def linear_fp8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               bias: torch.Tensor | None = None, *, activation: str = "none", residual: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear`` on e4m3 codes: x [..., k] with x_scale [...], weight [n, k] with weight_scale [n]
    (float32; a value is its code times its row's scale).  bias, residual and y are of ``dtype``.
    Not differentiable."""
    return _token.ext().linear_fp8(x, x_scale, weight, weight_scale, bias, residual, activation, dtype, _token.traced())
