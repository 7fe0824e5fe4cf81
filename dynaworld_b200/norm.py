"""Root-mean-square norm of the decoder's token stream, with the residual's addition and an 8-bit
output, and row-wise 8-bit quantisation.

    h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight

The layers in front of the decoder heads (GaussianParameterHeads, src/train/gs_models/blocks.py)
are torch modules in the reference; these are the B200 kernels for them, next to ``linear``.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._rows import E4M3, address, call, check_device, check_input, check_like, rows_of, workspace


def _norm(x, code: int, eps: float, residual, weight) -> bytes:
    """gsb_norm"""
    return _lib.pack_norm(x.shape[0], x.shape[1], code, eps, 0, x.data_ptr(), x.stride(0), address(residual),
                          0 if residual is None else residual.stride(0), address(weight))


def _forward(x, weight, residual, eps, code, need_rstd):
    """x [rows, dim] -> y, summed (None without a residual), rstd (None unless needed)."""
    y = x.new_empty(x.shape)
    summed = None if residual is None else x.new_empty(x.shape)
    rstd = x.new_empty(x.shape[0], dtype=torch.float32) if need_rstd else None
    call("rms_norm", "gsb_rms_norm_fwd", x.device, _norm(x, code, eps, residual, weight), y.data_ptr(), address(summed),
         address(rstd))
    return y, summed, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, code):
        y, summed, rstd = _forward(x, weight, residual, eps, code, True)
        ctx.eps, ctx.code = eps, code
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, weight, rstd)
        return y, summed

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsummed):
        x, residual, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:  # only the stream was used
            return (dsummed if need_x else None, None if not need_w else torch.zeros_like(weight),
                    dsummed if need_r else None, None, None)
        dim = x.shape[1]
        dy = rows_of(dy, dim)
        dsummed = None if dsummed is None else rows_of(dsummed, dim)
        dx = x.new_empty(x.shape)
        dw = x.new_empty(dim) if need_w else None
        norm = _norm(x, ctx.code, ctx.eps, residual, weight)
        nbytes = _lib.lib().gsb_rms_norm_bwd_workspace(norm)
        ws = workspace(x, nbytes)
        call("rms_norm_bwd", "gsb_rms_norm_bwd", x.device, norm, rstd.data_ptr(), dy.data_ptr(), dy.stride(0),
             address(dsummed), 0 if dsummed is None else dsummed.stride(0), dx.data_ptr(), address(dw), address(ws),
             nbytes)
        return dx if need_x else None, dw, dx if need_r else None, None, None


def _check(what, x, weight, residual, eps):
    code = check_input(what, x)
    if weight is not None:
        check_like(what, "weight", weight, (x.shape[-1],), x.dtype, x.device)
    if residual is not None:
        check_like(what, "residual", residual, x.shape, x.dtype, x.device)
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    check_device(what, x)
    return code


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x + residual.

    x and residual [..., D], weight [D], all float32, bfloat16 or float16 of one type.  Returns y,
    or with a residual the pair (y, h): h is the new residual stream.  The sum, the statistics and
    the product are formed in float; y and h are rounded once.  Differentiable in x, weight and
    residual (once; the backward forms h again from x and residual); the weight gradient is the same on every run."""
    code = _check("rms_norm", x, weight, residual, eps)
    dim = x.shape[-1]
    x2 = rows_of(x, dim)
    r2 = None if residual is None else rows_of(residual, dim)
    w = weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        y, h = _RmsNorm.apply(x2, w, r2, float(eps), code)
    else:
        y, h, _ = _forward(x2, w, r2, float(eps), code, False)
    if x.ndim != 2:
        y, h = y.view(x.shape), None if h is None else h.view(x.shape)
    return y if residual is None else (y, h)


def _refuse_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} is not differentiable; call it under torch.no_grad() or detach its inputs.")


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``rms_norm`` with y in 8 bits for ``linear_fp8``: (codes [..., D] float8_e4m3fn, scale [...]
    float32), and h as the third value with a residual.  Per row top = max(max |y|, 1e-30),
    scale = top / 448 and code = e4m3(y * (448 / top)), from y in float.  A row with a NaN or an
    infinity stands for NaN.  Not differentiable."""
    code = _check("rms_norm_fp8", x, weight, residual, eps)
    _refuse_grad("rms_norm_fp8", x, weight, residual)
    dim = x.shape[-1]
    x2 = rows_of(x, dim)
    r2 = None if residual is None else rows_of(residual, dim)
    w = weight.contiguous()
    q = x.new_empty(x.shape, dtype=E4M3)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    h = None if residual is None else x.new_empty(x.shape)
    call("rms_norm_fp8", "gsb_rms_norm_fp8", x.device, _norm(x2, code, float(eps), r2, w), q.data_ptr(), scale.data_ptr(),
         address(h))
    return (q, scale) if residual is None else (q, scale, h)


def quantize_rows_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., D] in 8 bits with one scale per row: (codes float8_e4m3fn, scale [...] float32), as
    ``rms_norm_fp8`` quantises its y.  For ``linear_fp8``: weights once, the activations between two
    8-bit products every step.  Not differentiable."""
    code = _check("quantize_rows_fp8", x, None, None, 0.0)
    _refuse_grad("quantize_rows_fp8", x)
    dim = x.shape[-1]
    x2 = rows_of(x, dim)
    q = x.new_empty(x.shape, dtype=E4M3)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    call("quantize_rows_fp8", "gsb_quantize_rows_fp8", x.device, _norm(x2, code, 0.0, None, None), q.data_ptr(),
         scale.data_ptr())
    return q, scale
