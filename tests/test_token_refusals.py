"""What the token-side operators refuse, before any kernel: on the host, without a GPU."""
import ctypes

import pytest
import torch

from dynaworld_b200 import _lib, build
from dynaworld_b200.linear import linear, linear_fp8
from dynaworld_b200.norm import quantize_rows_fp8, rms_norm, rms_norm_fp8

E4M3 = torch.float8_e4m3fn
F = torch.zeros


@pytest.mark.parametrize("error, match, call", [
    (TypeError, "float32, bfloat16 or float16", lambda: linear(F(2, 4, dtype=torch.float64), F(3, 4))),
    (TypeError, "float32, bfloat16 or float16", lambda: linear(F(2, 4, dtype=torch.int32), F(3, 4))),
    (ValueError, "at least one element", lambda: linear(F(2, 0), F(3, 0))),
    (ValueError, "at least one element", lambda: linear(torch.tensor(1.0), F(3, 1))),
    (ValueError, "weight must be", lambda: linear(F(2, 4), F(3, 5))),
    (ValueError, "weight must be", lambda: linear(F(2, 4), F(4))),
    (ValueError, "weight must be", lambda: linear(F(2, 4), F(0, 4))),
    (TypeError, "weight must be", lambda: linear(F(2, 4), F(3, 4, dtype=torch.bfloat16))),
    (ValueError, "bias must have shape", lambda: linear(F(2, 4), F(3, 4), F(4))),
    (TypeError, "bias must be", lambda: linear(F(2, 4), F(3, 4), F(3, dtype=torch.float16))),
    (ValueError, "residual must have shape", lambda: linear(F(2, 4), F(3, 4), residual=F(3))),
    (ValueError, "Unknown activation", lambda: linear(F(2, 4), F(3, 4), activation="swish")),
    (RuntimeError, "CUDA devices only", lambda: linear(F(2, 4), F(3, 4))),
    (TypeError, "takes torch.float8_e4m3fn", lambda: linear_fp8(F(2, 4), F(2), F(3, 4), F(3))),
    (TypeError, "weight must be", lambda: linear_fp8(F(2, 4, dtype=E4M3), F(2), F(3, 4), F(3))),
    (ValueError, "x_scale must have shape",
     lambda: linear_fp8(F(2, 4, dtype=E4M3), F(3), F(3, 4, dtype=E4M3), F(3))),
    (TypeError, "weight_scale must be",
     lambda: linear_fp8(F(2, 4, dtype=E4M3), F(2), F(3, 4, dtype=E4M3), F(3, dtype=torch.float16))),
    (TypeError, "gives float32, bfloat16 or float16",
     lambda: linear_fp8(F(2, 4, dtype=E4M3), F(2), F(3, 4, dtype=E4M3), F(3), dtype=torch.float64)),
    (TypeError, "bias must be torch.bfloat16",
     lambda: linear_fp8(F(2, 4, dtype=E4M3), F(2), F(3, 4, dtype=E4M3), F(3), F(3))),
    (RuntimeError, "CUDA devices only", lambda: linear_fp8(F(2, 4, dtype=E4M3), F(2), F(3, 4, dtype=E4M3), F(3))),
    (TypeError, "float32, bfloat16 or float16", lambda: rms_norm(F(2, 4, dtype=E4M3), F(4))),
    (ValueError, "weight must have shape", lambda: rms_norm(F(2, 4), F(5))),
    (TypeError, "weight must be", lambda: rms_norm(F(2, 4), F(4, dtype=torch.bfloat16))),
    (ValueError, "residual must have shape", lambda: rms_norm(F(2, 4), F(4), residual=F(4))),
    (ValueError, "eps must not be negative", lambda: rms_norm(F(2, 4), F(4), eps=-1.0)),
    (ValueError, "eps must not be negative", lambda: rms_norm(F(2, 4), F(4), eps=float("nan"))),
    (RuntimeError, "CUDA devices only", lambda: rms_norm(F(2, 4), F(4))),
    (RuntimeError, "CUDA devices only", lambda: rms_norm_fp8(F(2, 4), F(4))),
    (ValueError, "at least one element", lambda: quantize_rows_fp8(F(2, 0))),
    (RuntimeError, "CUDA devices only", lambda: quantize_rows_fp8(F(2, 4))),
    (ValueError, "values are too long", lambda: quantize_rows_fp8(F(1).expand(1, (1 << 24) + 1))),
    (ValueError, "larger than 2\\^24", lambda: linear(F(2, 1), F(1, 1).expand((1 << 24) + 1, 1))),
])
def test_refused(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_dual_tensors_are_refused():
    """A tangent in any argument raises (its derivative would be lost), with and without reverse mode beside
    it; without one, or with forward mode off, the call goes on to the check of the device."""
    import torch.autograd.forward_ad as fwd

    q = F(2, 4, dtype=E4M3)
    with fwd.dual_level():
        d24, d34, d3, d23, d4, d2 = (fwd.make_dual(F(*s), torch.ones(*s)) for s in ((2, 4), (3, 4), (3,), (2, 3), (4,), (2,)))
        for call in (lambda: linear(d24, F(3, 4)), lambda: linear(F(2, 4), d34), lambda: linear(F(2, 4), F(3, 4), d3),
                     lambda: linear(F(2, 4), F(3, 4), residual=d23),
                     lambda: linear(d24, F(3, 4).requires_grad_(True)),
                     lambda: linear_fp8(q, d2, F(3, 4, dtype=E4M3), F(3)),
                     lambda: linear_fp8(q, F(2), F(3, 4, dtype=E4M3), d3),
                     lambda: linear_fp8(q, F(2), F(3, 4, dtype=E4M3), F(3), d3, dtype=torch.float32),
                     lambda: linear_fp8(q, F(2), F(3, 4, dtype=E4M3), F(3), residual=d23, dtype=torch.float32),
                     lambda: rms_norm(d24, F(4)), lambda: rms_norm(F(2, 4), d4),
                     lambda: rms_norm(F(2, 4), F(4), residual=d24), lambda: rms_norm_fp8(d24, F(4)),
                     lambda: rms_norm_fp8(F(2, 4), d4), lambda: quantize_rows_fp8(d24)):
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call()
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            linear(fwd.unpack_dual(d24).primal, F(3, 4))
        with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA devices only"):
            linear(d24, F(3, 4))
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        linear(F(2, 4), F(3, 4))


def test_codes_that_want_gradients_are_refused():
    """float8 tensors may require gradients like any floating type; the 8-bit product has none to give."""
    x, w = F(2, 4, dtype=E4M3), F(3, 4, dtype=E4M3)
    for call in (lambda: linear_fp8(x.clone().requires_grad_(True), F(2), w, F(3)),
                 lambda: linear_fp8(x, F(2), w.clone().requires_grad_(True), F(3))):
        with pytest.raises(NotImplementedError, match="not differentiable"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA devices only"):
            call()


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_struct_sizes_match_header():
    assert ctypes.sizeof(_lib.Norm) == 8 + 4 * 4 + 5 * 8
    assert ctypes.sizeof(_lib.Linear) == 8 + 6 * 4 + 9 * 8


def test_entry_points_refuse_before_a_launch(lib):
    """Bad sizes, types and missing pointers give a status on the host; no rows are no work."""
    n = _lib.Norm(rows=4, dim=8, dtype=_lib.F32, eps=1e-6, x=256, x_stride=8, weight=256)
    b = ctypes.byref(n)
    assert lib.gsb_rms_norm_fwd(None, 256, None, None, None) == 7
    assert lib.gsb_rms_norm_fwd(b, None, None, None, None) == 7
    assert lib.gsb_rms_norm_fp8(b, 256, None, None, None) == 7
    assert lib.gsb_quantize_rows_fp8(b, None, 256, None) == 7
    assert lib.gsb_rms_norm_bwd(b, 256, 256, 8, None, 0, 256, None, 256, 16, None) == 2
    assert lib.gsb_rms_norm_bwd(b, None, 256, 8, None, 0, 256, None, 256, 1 << 20, None) == 7
    for field, bad, status in (("dim", 0, 1), ("dim", (1 << 24) + 1, 1), ("rows", -1, 1), ("rows", 1 << 31, 1), ("dtype", _lib.E4M3, 7),
                               ("eps", -1.0, 7), ("weight", None, 7), ("x", None, 7)):
        keep = getattr(n, field)
        setattr(n, field, bad)
        assert lib.gsb_rms_norm_fwd(b, 256, None, None, None) == status, field
        setattr(n, field, keep)
    n.rows = 0
    assert lib.gsb_rms_norm_fwd(b, 256, None, None, None) == 0

    p = _lib.Linear(m=4, n=8, k=8, dtype=_lib.BF16, out_dtype=_lib.BF16, x=256, x_stride=8, weight=256,
                    weight_stride=8)
    b = ctypes.byref(p)
    big = 1 << 30
    assert lib.gsb_linear_fwd(None, 256, None, 256, big, None) == 7
    assert lib.gsb_linear_fwd(b, None, None, 256, big, None) == 7
    for field, bad, status in (("n", 0, 1), ("k", 0, 1), ("m", -1, 1), ("m", 1 << 31, 1), ("n", (1 << 24) + 1, 1),
                               ("dtype", 4, 7), ("dtype", _lib.F16, 7), ("dtype", _lib.E4M3, 7),
                               ("out_dtype", _lib.E4M3, 7), ("activation", 5, 7), ("activation", -1, 7),
                               ("weight", None, 7), ("x", None, 7)):
        keep = getattr(p, field)
        setattr(p, field, bad)
        assert lib.gsb_linear_fwd(b, 256, None, 256, big, None) == status, field
        setattr(p, field, keep)
    assert lib.gsb_linear_bwd(b, None, None, 8, 256, 256, 256, 256, big, None) == 7
    assert lib.gsb_linear_bwd(b, None, 256, 8, 256, 256, 256, 256, 16, None) == 2
    p.activation = 2
    assert lib.gsb_linear_bwd(b, None, 256, 8, 256, 256, 256, 256, big, None) == 7  # no pre-activation
    p.dtype = _lib.E4M3
    assert lib.gsb_linear_bwd(b, 256, 256, 8, 256, 256, 256, 256, big, None) == 7  # serving only
    p.m, p.dtype, p.x = 0, _lib.BF16, None
    assert lib.gsb_linear_fwd(b, 256, None, 256, big, None) == 0


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.BF16, _lib.F16, _lib.E4M3])
def test_workspaces_off_their_boundary_are_refused(lib, dtype):
    """Rows in the workspace are read and written 16 bytes at a time: an address that allows no such access
    gives a status before any kernel."""
    out = _lib.BF16 if dtype == _lib.E4M3 else dtype
    p = _lib.Linear(m=300, n=40, k=67, dtype=dtype, out_dtype=out, x=256, x_stride=67, weight=256, weight_stride=67,
                    x_scale=256, weight_scale=256)
    b = ctypes.byref(p)
    assert lib.gsb_linear_fwd_workspace(b) > 0
    for ws in (264, 260, 257):
        assert lib.gsb_linear_fwd(b, 256, None, ws, 1 << 30, None) == 7
        if dtype != _lib.E4M3:
            assert lib.gsb_linear_bwd(b, None, 256, 40, 256, 256, 256, ws, 1 << 30, None) == 7
