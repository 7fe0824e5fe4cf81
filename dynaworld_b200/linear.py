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
from torch.autograd.function import once_differentiable

from . import _lib
from ._rows import E4M3, TYPE_CODES, address, call, check_device, check_input, check_like, rows_of, workspace
from .norm import _refuse_grad


def _activation(name: str) -> int:
    code = _lib.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"Unknown activation: {name!r} (one of {', '.join(_lib.ACTIVATIONS)})")
    return code


def _spec(x, weight, bias, residual, act, code, out_code, x_scale=None, weight_scale=None) -> bytes:
    """gsb_linear"""
    n, k = weight.shape
    return _lib.pack_linear(x.shape[0], n, k, code, out_code, act, 0, x.data_ptr(), x.stride(0), weight.data_ptr(),
                            weight.stride(0), address(bias), address(residual),
                            0 if residual is None else residual.stride(0), address(x_scale), address(weight_scale))


def _run_forward(spec: bytes, y: torch.Tensor, preact: torch.Tensor | None) -> None:
    nbytes = _lib.lib().gsb_linear_fwd_workspace(spec)
    ws = workspace(y, nbytes)
    call("linear", "gsb_linear_fwd", y.device, spec, y.data_ptr(), address(preact), address(ws), nbytes)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, code):
        y = x.new_empty((x.shape[0], weight.shape[0]))
        preact = None
        if act and any(ctx.needs_input_grad[:3]):
            preact = y.new_empty(y.shape, dtype=torch.float32 if code == _lib.F32 else torch.float16)
        _run_forward(_spec(x, weight, bias, residual, act, code, code), y, preact)
        ctx.act, ctx.code = act, code
        ctx.save_for_backward(x, weight, preact)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, preact = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        if not (need_x or need_w or need_b):
            return None, None, None, dy if need_r else None, None, None
        n, k = weight.shape
        g = rows_of(dy, n)
        dx = x.new_empty((x.shape[0], k)) if need_x else None
        dw = x.new_empty((n, k)) if need_w else None
        db = x.new_empty(n) if need_b else None
        spec = _spec(x, weight, None, None, ctx.act, ctx.code, ctx.code)
        gp, gs = g.data_ptr(), g.stride(0)
        nbytes = _lib.lib().gsb_linear_bwd_workspace(spec, gp, gs)
        ws = workspace(x, nbytes)
        call("linear_bwd", "gsb_linear_bwd", x.device, spec, address(preact), gp, gs, address(dx), address(dw),
             address(db), address(ws), nbytes)
        return dx, dw, db, dy if need_r else None, None, None


def _check_shapes(what, x, weight, bias, residual, dtype):
    if weight.ndim != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"{what}: weight must be [n, {x.shape[-1]}], got {tuple(weight.shape)}")
    n = weight.shape[0]
    if weight.dtype != x.dtype:
        raise TypeError(f"{what}: weight must be {x.dtype}, got {weight.dtype}")
    if weight.device != x.device:
        raise RuntimeError(f"{what}: weight is on {weight.device}, the input on {x.device}")
    if bias is not None:
        check_like(what, "bias", bias, (n,), dtype, x.device)
    if residual is not None:
        check_like(what, "residual", residual, (*x.shape[:-1], n), dtype, x.device)
    return n


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = act(x weight^T + bias) + residual, x [..., k], weight [n, k], bias [n], residual and y
    [..., n]; all float32, bfloat16 or float16 of one type.  ``activation``: "none", "relu",
    "gelu", "gelu_tanh" (its tanh form) or "silu".

    Sums, bias, activation and residual are formed in float and rounded once.  Differentiable once
    in x, weight, bias and residual.  With an activation the forward keeps x weight^T + bias for the
    backward (float beside float32 operands, else float16), and the backward rounds
    dy act'(z) to the operands' type before its two products.  The same inputs give the same bits."""
    code = check_input("linear", x)
    act = _activation(activation)
    n = _check_shapes("linear", x, weight, bias, residual, x.dtype)
    check_device("linear", x)
    x2, w2 = rows_of(x, x.shape[-1]), rows_of(weight, weight.shape[1])
    r2 = None if residual is None else rows_of(residual, n)
    b = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (b is not None and b.requires_grad)
                                    or (r2 is not None and r2.requires_grad)):
        y = _Linear.apply(x2, w2, b, r2, act, code)
        return y if x.ndim == 2 else y.view(*x.shape[:-1], n)
    y = x.new_empty((*x.shape[:-1], n))
    _run_forward(_spec(x2, w2, b, r2, act, code, code), y, None)
    return y


def linear_fp8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               bias: torch.Tensor | None = None, *, activation: str = "none", residual: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear`` on e4m3 codes: x [..., k] with x_scale [...], weight [n, k] with weight_scale [n]
    (float32; a value is its code times its row's scale).  bias, residual and y are of ``dtype``.
    Not differentiable."""
    if x.dtype != E4M3:
        raise TypeError(f"linear_fp8 takes {E4M3} codes, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"linear_fp8 needs rows of at least one element, got shape {tuple(x.shape)}")
    out_code = TYPE_CODES.get(dtype)
    if out_code is None:
        raise TypeError(f"linear_fp8 gives float32, bfloat16 or float16, not {dtype}")
    act = _activation(activation)
    n = _check_shapes("linear_fp8", x, weight, bias, residual, dtype)
    check_like("linear_fp8", "x_scale", x_scale, x.shape[:-1], torch.float32, x.device)
    check_like("linear_fp8", "weight_scale", weight_scale, (n,), torch.float32, x.device)
    check_device("linear_fp8", x)
    _refuse_grad("linear_fp8", x_scale, weight_scale, bias, residual)
    x2, w2 = rows_of(x, x.shape[-1]), rows_of(weight, weight.shape[1])
    r2 = None if residual is None else rows_of(residual, n)
    b = None if bias is None else bias.contiguous()
    y = x.new_empty((*x.shape[:-1], n), dtype=dtype)
    _run_forward(_spec(x2, w2, b, r2, act, _lib.E4M3, out_code, x_scale.contiguous(), weight_scale.contiguous()), y, None)
    return y
