"""The torch binding of the token-side operators (csrc/token_torch.cpp), loaded at their first use."""
from __future__ import annotations

import ctypes

from . import _lib, render

_ext = None


def load():
    """Imports _token_torch and gives it libgsb200's entry points."""
    global _ext
    if _ext is None:
        lib = _lib.lib()
        try:
            from . import _token_torch
        except ImportError as exc:
            raise RuntimeError(f"the token-side operators are not built ({exc}): "
                               "build them with `python -m dynaworld_b200.build`") from exc
        names = [n for n in _lib.SIGNATURES if n.startswith(("gsb_rms_norm", "gsb_quantize", "gsb_linear"))]
        _token_torch.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
        _ext = _token_torch
    return _ext


def ext():
    return _ext if _ext is not None else load()


def traced() -> bool:
    """Whether stages are bracketed (render.STAGE_EVENTS, diagnostics.nvtx).  A call's backward goes by
    what its forward saw."""
    return render.NVTX or render.STAGE_EVENTS is not None
