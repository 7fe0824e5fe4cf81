"""Argument handling shared by the token-side operators (linear, norm)."""
from __future__ import annotations

import contextlib

import torch

from . import _lib, render

TYPE_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
E4M3 = torch.float8_e4m3fn
_NOTHING = contextlib.nullcontext()


def on_device(device: torch.device):
    """Makes ``device`` current for the launches inside (nothing to do when it already is)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NOTHING
    return torch.cuda.device(device)


def call(stage: str, name: str, device: torch.device, *args) -> None:
    """C entry point ``name`` with ``args`` and the device's current stream, on that device; its status
    raises.  Without tracing and on the current device nothing is set up around it: the operators of a
    single token take as long on the host as on the GPU."""
    fn = getattr(_lib.lib(), name)
    index = device.index
    if render.STAGE_EVENTS is None and not render.NVTX and index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with on_device(device), render._stage(stage):
            status = fn(*args, render._stream(device))
    if status:
        _lib.check(name, status)


def address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] as [rows, width] with adjacent row elements: a view where the strides allow it
    (any positive row stride), else a copy."""
    if t.ndim != 2:
        t = t.reshape(-1, width)
    down, along = t.stride()
    if (along != 1 and width > 1) or (down < 1 and t.shape[0] > 1):
        t = t.contiguous()
    return t


def workspace(like: torch.Tensor, nbytes: int) -> torch.Tensor | None:
    """Scratch on the device of ``like``, or None when none is needed."""
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def check_input(what: str, x: torch.Tensor) -> int:
    """The element-type code of x, or the error that refuses it."""
    code = TYPE_CODES.get(x.dtype)
    if code is None:
        raise TypeError(f"{what} takes float32, bfloat16 or float16 tensors, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} needs rows of at least one element, got shape {tuple(x.shape)}")
    return code


def check_device(what: str, x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"the b200 {what} runs on CUDA devices only (got a tensor on {x.device})")


def check_like(what: str, name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> None:
    if t.shape != shape:
        raise ValueError(f"{what}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, the input on {device}")
