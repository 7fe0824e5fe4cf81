"""linear and linear_fp8 on the GPU against their formulas in 64 bits.

Bounds.  half(t) is half a relative step of the type t.  A product's sum over K float terms, added in
any order with additions that truncate (an error of at most 2^-23 of the partial sum each), is within
K 2^-23 sum |x w|.  float32 operands of the tensor-core path are split into three bf16 parts; the
parts that it does not multiply are below 2^-25 |x w| each, which the same bound's first term covers.
The activations' slopes are at most 1.13 and their second derivatives at most 1.13, |z act''| at most
1.1; the functions themselves are evaluated within 2^-20 |z| (+ 2^-24).  The kept z has half(float16)
relative error beside 16-bit operands; dz is rounded to the operands' type.  Within its error of 0 the
slope of relu is either side's."""
import math

import pytest
import torch

from dynaworld_b200 import _lib
from dynaworld_b200.linear import linear, linear_fp8
from dynaworld_b200.norm import quantize_rows_fp8
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = list(_lib.ACTIVATIONS)
E4M3 = torch.float8_e4m3fn


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def act64(z, kind):
    if kind == "relu":
        return z.clamp_min(0), (z > 0).double()
    if kind == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def make(m, k, n, t, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(m, k, generator=g)).to(t)
    w = (torch.randn(n, k, generator=g) / math.sqrt(k)).to(t)
    b = (0.5 * torch.randn(n, generator=g)).to(t)
    r = torch.randn(m, n, generator=g).to(t)
    dy = torch.randn(m, n, generator=g).to(t)
    return [v.to(DEV) for v in (x, w, b, r, dy)]


def within(got, ref, bound, what=""):
    assert got.shape == ref.shape
    over = (got.double() - ref).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {over.max().item():.3e} past the bound"


def check(x, w, b, r, dy, act, grads=True):
    t = x.dtype
    n, k = w.shape
    X, W = x.detach().double().reshape(-1, k), w.detach().double()
    leaves = [None if v is None else v.detach().clone().requires_grad_(grads) for v in (x, w, b, r)]
    y = linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    z = X @ W.T
    mag = X.abs() @ W.abs().T
    if b is not None:
        z = z + b.double()
        mag = mag + b.double().abs()
    dz_fwd = (k + 2) * U * mag
    a, slope = act64(z, act)
    ref = a if r is None else a + r.double().reshape(-1, n)
    eval_err = z.abs() * 2.0 ** -20 + 2.0 ** -24
    bound = ref.abs() * half(t) * (1 + 1e-3) + 1.13 * dz_fwd + eval_err + tiny(t)
    if r is not None:
        bound = bound + r.double().reshape(-1, n).abs() * U
    within(y.reshape(-1, n), ref, bound, "y")
    if not grads:
        return y
    used = [v for v in leaves if v is not None]
    got = dict(zip([i for i, v in enumerate(leaves) if v is not None], torch.autograd.grad(y, used, dy)))
    G = dy.double().reshape(-1, n)
    m = G.shape[0]
    dz = G * slope
    err = dz.abs() * half(t) + tiny(t)
    if act != "none":
        kept = 0.0 if t == torch.float32 else 1.1 * half(torch.float16) + 2.0 ** -24
        err = err + G.abs() * (1.13 * dz_fwd + kept + 2.0 ** -20)
        if act == "relu":
            near = z.abs() <= dz_fwd + z.abs() * half(torch.float16) + 2.0 ** -24
            err = torch.where(near, G.abs() * (1 + half(t)), dz.abs() * half(t) + tiny(t))
    else:
        err = torch.zeros_like(dz)
    whole = dz.abs() + err
    dx = dz @ W
    within(got[0].reshape(-1, k), dx, dx.abs() * half(t) + err @ W.abs() + (n + 2) * U * (whole @ W.abs()) + tiny(t),
           "dx")
    dw = dz.T @ X
    within(got[1], dw, dw.abs() * half(t) + err.T @ X.abs() + (m + 2) * U * (whole.T @ X.abs()) + tiny(t), "dw")
    if b is not None:
        db = dz.sum(0)
        within(got[2], db, db.abs() * half(t) + err.sum(0) + (m + 2) * U * whole.sum(0) + tiny(t), "db")
    if r is not None:
        assert torch.equal(got[3].reshape(-1, n), dy.reshape(-1, n))
    return y


# one token, few tokens, tile edges and one past them, odd widths, long sums, widths below a vector
SHAPES = [(1, 1, 1), (1, 64, 128), (1, 1000, 77), (2, 515, 24), (8, 256, 513), (9, 64, 40), (16, 2048, 96),
          (63, 100, 300), (64, 64, 64), (127, 129, 255), (128, 128, 256), (129, 136, 264), (300, 771, 1285),
          (513, 72, 56), (1025, 512, 130), (2500, 40, 3), (5, 4096, 16), (257, 1037, 9), (700, 520, 1032),
          # backward products in pieces along a long K: both, aligned; one of them much smaller
          (4100, 264, 520), (20000, 64, 72),
          # a few aligned rows: one and two blocks of 16, columns past a block of 32, a ragged last step of K
          (13, 96, 4741), (2, 208, 4800), (24, 128, 520), (31, 2064, 33), (17, 48, 4744)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_and_gradients(m, k, n, t):
    x, w, b, r, dy = make(m, k, n, t, seed=m + n)
    act = ACTS[(m + k + n) % len(ACTS)]
    check(x, w, b if (m + n) % 3 else None, r if m % 2 else None, dy, act)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 200])
def test_activations(m, act, t):
    """Pre-activations over the whole range of the functions, small and saturated."""
    x, w, b, r, dy = make(m, 96, 160, t, seed=5, scale=4.0)
    check(x, w, b, None, dy, act)
    check(x, w, None, r, dy, act)


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_leading_dimensions(t):
    """Rows of wider tensors whose starts are aligned to 16 bytes or not, leading dimensions, a
    transposed input and weight, an expanded gradient."""
    x, w, b, r, dy = make(130, 64, 72, t)
    for first, width in ((0, 80), (16, 96), (1, 67)):
        wide_x = torch.full((130, width), float("nan"), dtype=t, device=DEV)
        wide_x[:, first:first + 64] = x
        wide_w = torch.full((72, width), float("nan"), dtype=t, device=DEV)
        wide_w[:, first:first + 64] = w
        wide_r = torch.full((130, width + 72), float("nan"), dtype=t, device=DEV)
        wide_r[:, first:first + 72] = r
        got = linear(wide_x[:, first:first + 64], wide_w[:, first:first + 64], b, activation="silu",
                     residual=wide_r[:, first:first + 72])
        X, W = x.double(), w.double()
        z = X @ W.T + b.double()
        ref = act64(z, "silu")[0] + r.double()
        mag = X.abs() @ W.abs().T + b.double().abs()
        within(got, ref, ref.abs() * half(t) * 1.001 + 70 * U * mag + z.abs() * 2.0 ** -20 + 2.0 ** -22)
        leaf = wide_x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(linear(leaf[:, first:first + 64], w), leaf, dy)
        ref = dy.double() @ W
        within(g[:, first:first + 64], ref, ref.abs() * half(t) + 74 * U * (dy.double().abs() @ W.abs()) + tiny(t))
        assert bool((g[:, :first] == 0).all()) and bool((g[:, first + 64:] == 0).all())
    y = linear(x, w, b)
    assert torch.equal(linear(x.view(2, 65, 64), w, b).view(130, 72), y)
    assert torch.equal(linear(x.t().contiguous().t(), w.t().contiguous().t(), b), y)
    one = linear(x[7], w, b)
    assert one.shape == (72,)
    leaf, leaf2 = (x.clone().requires_grad_(True) for _ in range(2))
    linear(leaf, w, b, activation="gelu").sum().backward()
    linear(leaf2, w, b, activation="gelu").backward(torch.ones_like(y))
    assert torch.equal(leaf.grad, leaf2.grad)
    # rows that are one row repeated
    rep = x[:1].expand(130, 64)
    assert torch.equal(linear(rep, w, b)[5], linear(rep, w, b)[77])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [1, 20, 300])
def test_rows_that_overlap(m, t):
    """Windows over one line of values: rows whose distance is less than their length."""
    line = torch.randn(8 * m + 64, generator=torch.Generator().manual_seed(m)).to(DEV, t)
    x, w = line.as_strided((m, 64), (8, 1)), line.as_strided((min(m, 40), 64), (8, 1))
    dy = torch.ones(m, w.shape[0], dtype=t, device=DEV)
    got, ref = [x.detach().requires_grad_(True), w.detach()], [x.contiguous().requires_grad_(True), w.contiguous()]
    a, b = (linear(*v, activation="silu") for v in (got, ref))
    assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(a, got[0], dy)[0], torch.autograd.grad(b, ref[0], dy)[0])


def test_views_that_stand_for_negatives():
    """The imaginary part of a conjugate is a view of the parts' memory with a sign: operands, bias,
    residual, gradient and the norm's tensors."""
    from dynaworld_b200.norm import rms_norm

    x, w, b, r, dy = (torch._neg_view(v) for v in make(20, 16, 24, torch.float32))
    assert x.is_neg()
    X, W, B, R, G = (v.clone().resolve_neg() for v in (x, w, b, r, dy))
    leaf, LEAF = (v.requires_grad_(True) for v in (x.detach(), X.detach()))
    got, ref = (linear(*v[:3], activation="silu", residual=v[3]) for v in ((leaf, w, b, r), (LEAF, W, B, R)))
    assert torch.equal(got, ref)
    assert torch.equal(torch.autograd.grad(got, leaf, dy)[0], torch.autograd.grad(ref, LEAF, G)[0])
    assert torch.equal(rms_norm(x, w[0], residual=x)[0], rms_norm(X, W[0], residual=X)[0])
    one = torch.randn(6, 1, dtype=torch.complex64, device=DEV).conj().imag
    assert one.is_neg() and torch.equal(linear(one, torch.ones(1, 1, device=DEV)), one.clone().resolve_neg())
    assert all(torch.equal(a.float(), c.float()) for a, c in zip(quantize_rows_fp8(x), quantize_rows_fp8(X)))


@pytest.mark.parametrize("t", TYPES)
def test_nothing_to_do(t):
    w = torch.ones(24, 16, dtype=t, device=DEV, requires_grad=True)
    b = torch.ones(24, dtype=t, device=DEV, requires_grad=True)
    x = torch.empty(0, 16, dtype=t, device=DEV, requires_grad=True)
    y = linear(x, w, b, activation="gelu")
    assert y.shape == (0, 24)
    y.sum().backward()
    assert x.grad.shape == (0, 16) and bool((w.grad == 0).all()) and bool((b.grad == 0).all())


@pytest.mark.parametrize("t", TYPES)
def test_only_some_gradients(t):
    x, w, b, r, dy = make(200, 72, 88, t)
    full = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
    ref = torch.autograd.grad(linear(full[0], full[1], full[2], activation="silu", residual=full[3]), full, dy)
    for i in range(4):
        part = [v.clone().requires_grad_(j == i) for j, v in enumerate((x, w, b, r))]
        (g,) = torch.autograd.grad(linear(part[0], part[1], part[2], activation="silu", residual=part[3]), part[i], dy)
        assert torch.equal(g, ref[i])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [4, 300])
def test_nonfinite_rows_stay_in_their_row(m, t):
    x, w, b, r, dy = make(m, 128, 96, t)
    y = linear(x, w, b, activation="silu")
    x2 = x.clone()
    x2[2, 5] = float("nan")
    x2[3, 6] = float("inf")
    y2 = linear(x2, w, b, activation="silu")
    assert bool(y2[2].isnan().all()) and not bool(torch.isfinite(y2[3]).all())
    keep = [i for i in range(m) if i not in (2, 3)]
    assert torch.equal(y2[keep], y[keep])


def same_kind(got, ref):
    """Equal, or both NaN."""
    return bool(((got == ref) | (got.isnan() & ref.isnan())).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k", [(1, 64), (4, 64), (4, 65), (130, 64), (130, 65), (64, 4096)])
def test_infinite_preactivations(m, k, act, t):
    """z of +infinity and -infinity (float and bf16: finite operands whose products overflow) give what the
    formula gives, on every path."""
    x, w = torch.zeros(m, k, dtype=t, device=DEV), torch.zeros(512, k, dtype=t, device=DEV)
    x[:, 0], x[:, 1] = (math.inf if t == torch.float16 else 3e38), 1
    w[:, 0], w[:, 1] = 1, 0.5
    w[::2, 0], w[1::2, 0] = 4, -4
    ref = act64(torch.tensor([math.inf, -math.inf], dtype=torch.float64), act)[0].to(DEV, t)
    y = linear(x, w, activation=act)
    assert float(ref[0]) == math.inf
    assert same_kind(y, ref.repeat(256).expand(m, 512)), y[0, :2]
    if t == torch.float32:
        return
    q, s = torch.ones(m, k, device=DEV).to(E4M3), torch.full((m,), 2e38, device=DEV)
    q2 = w.float().clamp(-1, 1).to(E4M3)
    y = linear_fp8(q, s, q2, torch.full((512,), 2e38, device=DEV), activation=act, dtype=t)
    assert same_kind(y, ref.repeat(256).expand(m, 512)), y[0, :2]


def bf16_parts(v):
    """v (float32) as three bf16 values, in 64 bits."""
    out = []
    for _ in range(3):
        out.append(v.bfloat16())
        v = v - out[-1].float()
    return [p.double() for p in out]


@pytest.mark.parametrize("m,k,n", [(1, 4096, 64), (9, 64, 40), (65, 64, 64), (127, 129, 255), (129, 136, 264),
                                   (300, 771, 1285), (1025, 512, 130), (257, 1037, 9), (700, 520, 1032),
                                   (4100, 264, 520), (20000, 64, 72), (100, 4100, 512), (300, 4096, 1024)])
def test_float32_products_are_as_exact_as_float32_sums(m, k, n):
    """In norm: four steps of float (2^-24) for the split operands, the tensor core's chain over 64 of K and
    the last rounding, and one more per addition of such a chain's sum, whose roundings add up as their root.
    Products without the parts' small cross terms are past that bound, so it holds the split to all six."""
    x, w, _, _, dy = make(m, k, n, torch.float32, seed=m + n)
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    y = linear(*leaves)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    for got, a, b in ((y, x, w.T), (dx, dy, w), (dw, dy.T, x)):
        ref = a.double() @ b.double()
        bound = 2.0 ** -24 * (4 + math.sqrt(a.shape[1] / 64))
        assert float((got.detach().double() - ref).norm() / ref.norm()) <= bound
        if min(got.shape) > 1 and a.shape[1] > 16:
            (a1, a2, a3), (b1, b2, b3) = bf16_parts(a), bf16_parts(b)
            for lost in (a1 @ b3 + a3 @ b1, a2 @ b2, a1 @ b3):
                assert float(lost.norm() / ref.norm()) > bound


def test_gelu_in_float32():
    """GELU and its slope over |z| <= 12 to float's accuracy, the tail's relative one included.  Phi(-|z|)
    and the density carry: the fit (2^-23), 8 steps of the polynomial whose terms' magnitudes are at most
    1.8 times its value (8 x 1.8 x 2^-24), the reciprocal (2^-23 times t's weight, at most 2.5), the
    exponential (2^-22) and three products: 2^-19 in all, and the exponent's roundings, z^2 2^-23.  The sums
    around them round once each (2^-23)."""
    z = torch.linspace(-12, 12, 40001, device=DEV, dtype=torch.float64).float()[:, None].requires_grad_(True)
    y = linear(z, torch.ones(1, 1, device=DEV), activation="gelu")  # z itself is exact: one product with 1
    (slope,) = torch.autograd.grad(y.sum(), z)
    Z = z.detach().double()
    ref, ref_slope = act64(Z, "gelu")
    tail = 0.5 * torch.special.erfc(Z.abs() / math.sqrt(2))
    gauss = torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)
    rel = 2.0 ** -19 + Z * Z * U
    within(y, ref, Z.abs() * tail * rel + ref.abs() * U + 1e-37, "y")
    within(slope, ref_slope, (tail + Z.abs() * gauss) * rel + ref_slope.abs() * U + 1e-37, "slope")


@pytest.mark.parametrize("m,k,n", [(3, 64, 40), (130, 64, 72), (130, 67, 41), (300, 512, 264), (100, 4096, 512)])
def test_infinities_in_float32(m, k, n):
    """Infinite operands give what sums of float products give, however many rows there are: an infinity of
    the factors' sign, NaN where it meets a zero or the other infinity; everything else is untouched."""
    x, w, _, _, dy = make(m, k, n, torch.float32, seed=m)
    w[::2] = w[::2].bfloat16().float()  # values whose second and third part are 0
    w[5, 3] = 0
    x[1, 3], x[2, 7], x[2, 9], dy[0, 6] = math.inf, -math.inf, math.inf, -math.inf
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    y = linear(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    X, W, G = x.detach().double(), w.detach().double(), dy.double()

    def product(a, b):
        """a b^T with the terms of infinities counted one by one."""
        fa, fb = a.nan_to_num(0, 0, 0), b.nan_to_num(0, 0, 0)
        out = fa @ fb.T
        for c in torch.nonzero(a.isinf().any(0) | b.isinf().any(0)).flatten().tolist():
            out = out + a[:, c, None] * b[None, :, c] - fa[:, c, None] * fb[None, :, c]
        return out, (fa.abs() @ fb.abs().T) * ((a.shape[1] + 2) * U)

    for what, v, (ref, bound) in zip(("y", "dx", "dw"), got, (product(X, W), product(G, W.T), product(G.T, X.T))):
        kind = ~torch.isfinite(ref)
        assert same_kind(v.double()[kind], ref[kind]), what
        within(v[~kind], ref[~kind], ref[~kind].abs() * half(torch.float32) + bound[~kind], what)
        assert 0 < int(kind.sum()) < kind.numel()


def test_large_values_in_float32():
    """Values near the type's largest, whose bf16 rounding would overflow."""
    x = torch.full((130, 64), 0.0, device=DEV)
    x[:, 0] = torch.finfo(torch.float32).max
    w = torch.zeros(70, 64, device=DEV)
    w[:, 0] = 0.5
    y = linear(x, w)
    ref = x.double() @ w.double().T
    within(y, ref, ref * 66 * U)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_saturated_preactivations(t):
    """z beyond fp16's range: the kept z saturates and the slope there is 1 or 0."""
    x = torch.full((140, 64), 200.0, dtype=t, device=DEV)
    x[70:] = -200.0
    w = torch.full((32, 64), 60.0 if t == torch.float16 else 100.0, dtype=t, device=DEV)
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        leaf = (x / 64).requires_grad_(True) if t == torch.float16 else x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(linear(leaf, w, activation=act).float().sum(), leaf)
        assert bool((g[70:] == 0).all())
        assert bool((g[:70].float() == 32 * float(w[0, 0])).all())


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (3, 64, 40), (5, 65, 41), (300, 64, 264), (129, 65, 131),
                                   (200, 2048, 64)])
def test_relu_of_small_preactivations(m, k, n, t):
    """Every |z| is far below fp16's least value: ReLU's slope is still 1 wherever z > 0, on every path (one
    row, few rows, tiles, rows off 16 bytes, pieces).  Only within the sum's own error of 0 is it open."""
    x, w, _, _, dy = make(m, k, n, torch.float32, seed=m + k)
    s = 2.0 ** -15 if t == torch.float16 else 2.0 ** -30
    x, w, dy = (s * x).to(t), (s * math.sqrt(k) * w).to(t), dy.to(t)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, torch.zeros(n, dtype=t, device=DEV))]
    dx, dw, db = torch.autograd.grad(linear(*leaves, activation="relu"), leaves, dy)
    X, W, G = x.double(), w.double(), dy.double()
    z = X @ W.T
    dz = torch.where(z > 0, G, 0.0)
    err = torch.where(z.abs() <= (k + 2) * U * (X.abs() @ W.abs().T), G.abs(), 0.0)
    whole = dz.abs() + err
    ref = dz @ W
    within(dx, ref, ref.abs() * half(t) + err @ W.abs() + (n + 2) * U * (whole @ W.abs()) + tiny(t), "dx")
    ref = dz.T @ X
    within(dw, ref, ref.abs() * half(t) + err.T @ X.abs() + (m + 2) * U * (whole.T @ X.abs()) + tiny(t), "dw")
    ref = dz.sum(0)
    within(db, ref, ref.abs() * half(t) + err.sum(0) + (m + 2) * U * whole.sum(0) + tiny(t), "db")


def test_same_bits_every_run():
    for t in TYPES:
        x, w, b, r, dy = make(3000, 136, 72, t)

        def once():
            leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
            y = linear(leaves[0], leaves[1], leaves[2], activation="gelu")
            return [y, *torch.autograd.grad(y, leaves, dy)]
        for a, c in zip(once(), once()):
            assert torch.equal(a, c)


def test_gradient_against_differences():
    """Central differences in 64 bits of the formula against the kernels' 32-bit gradients."""
    x, w, b, r, dy = make(3, 24, 10, torch.float32, seed=9)
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        got = torch.autograd.grad(linear(leaves[0], leaves[1], leaves[2], activation=act), leaves, dy)

        def f(parts):
            return (act64(parts[0] @ parts[1].T + parts[2], act)[0] * dy.double()).sum()

        base = [v.double() for v in (x, w, b)]
        step = 1e-4
        for i, idx in ((0, (1, 5)), (0, (2, 23)), (1, (9, 0)), (1, (4, 13)), (2, (7,))):
            plus, minus = [v.clone() for v in base], [v.clone() for v in base]
            plus[i][idx] += step
            minus[i][idx] -= step
            assert abs(float((f(plus) - f(minus)) / (2 * step)) - float(got[i][idx])) < 2e-5


# products that are cut into pieces along K: small outputs of long sums, aligned and not
LONG = [(300, 4096, 1024), (64, 4096, 512), (100, 4100, 515), (40, 8192, 264)]


def pieces_of(dtype, m, k, n):
    """Bytes of the forward's float sums of pieces: its workspace, where the operands are read in place."""
    import ctypes

    p = _lib.Linear(m=m, n=n, k=k, dtype=dtype, out_dtype=dtype if dtype != _lib.E4M3 else _lib.BF16, x=256,
                    x_stride=k, weight=256, weight_stride=k, x_scale=256, weight_scale=256)
    return _lib.lib().gsb_linear_fwd_workspace(ctypes.byref(p)) // (4 * m * n)


def test_long_sums_are_cut():
    """What the tests below are about: every aligned shape of LONG runs in pieces, in every type that is
    read in place."""
    for m, k, n in LONG:
        for dtype in (_lib.BF16, _lib.F16, _lib.E4M3):
            if k % (16 if dtype == _lib.E4M3 else 8) == 0:
                assert pieces_of(dtype, m, k, n) >= 2, (m, k, n, dtype)
    assert pieces_of(_lib.BF16, 8192, 1024, 4096) == 0


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", LONG)
def test_long_sums_and_gradients(m, k, n, act, t):
    x, w, b, r, dy = make(m, k, n, t, seed=m)
    check(x, w, b, r, dy, act)
    check(x, w, None, None, dy, act)


# ---- 8-bit operands ----


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_fp8(m, k, n, t):
    x, w, b, r, _ = make(m, k, n, torch.float32, seed=m + k)
    b, r = b.to(t), r.to(t)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    act = ACTS[(m + n) % len(ACTS)]
    y = linear_fp8(xq, xs, wq, ws, b, activation=act, residual=r, dtype=t)
    X, W = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    z = X @ W.T + b.double()
    mag = X.abs() @ W.abs().T + b.double().abs()
    ref = act64(z, act)[0] + r.double()
    within(y, ref, ref.abs() * half(t) * 1.001 + 1.13 * (k + 4) * U * mag + z.abs() * 2.0 ** -20 + 2.0 ** -24 +
           r.double().abs() * U + tiny(t))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", LONG)
def test_fp8_long_sums(m, k, n, act, t):
    x, w, b, r, _ = make(m, k, n, torch.float32, seed=m + k)
    b, r = b.to(t), r.to(t)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    X, W = xq.double() * xs.double()[:, None], wq.double() * ws.double()[:, None]
    z, mag = X @ W.T, X.abs() @ W.abs().T
    for bias, res in ((b, r), (None, None)):
        y = linear_fp8(xq, xs, wq, ws, bias, activation=act, residual=res, dtype=t)
        zb, mb, rd = z, mag, torch.zeros_like(z)
        if bias is not None:
            zb, mb, rd = z + b.double(), mag + b.double().abs(), r.double()
        ref = act64(zb, act)[0] + rd
        within(y, ref, ref.abs() * half(t) * 1.001 + 1.13 * (k + 4) * U * mb + zb.abs() * 2.0 ** -20 + 2.0 ** -24 +
               rd.abs() * U + tiny(t))


def test_fp8_strides_and_dimensions():
    x, w, b, r, _ = make(130, 128, 96, torch.float32)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    ref = linear_fp8(xq, xs, wq, ws)
    assert ref.dtype == torch.bfloat16
    assert torch.equal(linear_fp8(xq.view(2, 65, 128), xs.view(2, 65), wq, ws).view(130, 96), ref)
    for first, width in ((16, 160), (3, 135)):
        wide = torch.zeros(130, width, dtype=torch.uint8, device=DEV)
        wide[:, first:first + 128] = xq.view(torch.uint8)
        got = linear_fp8(wide.view(E4M3)[:, first:first + 128], xs, wq, ws)
        assert torch.equal(got, ref)
    one = linear_fp8(xq[3], xs[3], wq, ws)
    assert one.shape == (96,)
    assert linear_fp8(xq[:0], xs[:0], wq, ws).shape == (0, 96)


def test_refusals_on_the_gpu():
    x, w, b, r, dy = make(4, 16, 8, torch.float32)
    xq, xs = quantize_rows_fp8(x)
    wq, ws = quantize_rows_fp8(w)
    with pytest.raises(NotImplementedError, match="not differentiable"):
        linear_fp8(xq, xs, wq, ws, b.requires_grad_(True), dtype=torch.float32)
    with pytest.raises(RuntimeError, match="weight is on cpu"):
        linear(x, w.cpu())
    with pytest.raises(RuntimeError, match="bias is on cpu"):
        linear(x, w, b.detach().cpu())
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(linear(leaf, w, activation="gelu").sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- streams and graphs ----


def test_calls_at_once_from_threads():
    """Four threads on streams of their own, forward and backward at the same time: every result is that of
    the call alone."""
    import threading

    cases = [make(m, 264, 520, t, seed=m) for m, t in ((700, torch.bfloat16), (20, torch.float16),
                                                       (600, torch.float32), (1, torch.bfloat16))]

    def step(case):
        x, w, b, r, dy = case
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        y = linear(leaves[0], leaves[1], leaves[2], activation="gelu_tanh", residual=r)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    refs = [step(c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step(cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, refs[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("t", TYPES)
def test_other_stream(t):
    x, w, b, r, dy = make(260, 200, 136, t)
    ref = linear(x, w, b, activation="gelu", residual=r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = linear(x, w, b, activation="gelu", residual=r)
    side.synchronize()
    assert torch.equal(y, ref)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [1, 300])
def test_two_captured_graphs_replayed_together(m, t):
    """Two graphs of the forward and backward with workspaces of their own, replayed on two streams."""
    sets = [make(m, 264, 144, t, seed=s) for s in (1, 2)]
    graphs, outs, refs, kept = [], [], [], []
    for x, w, b, r, dy in sets:
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        kept.append(leaves)  # a graph reads its inputs where they were

        def step(leaves=leaves, dy=dy):
            y = linear(leaves[0], leaves[1], leaves[2], activation="silu")
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

        refs.append([v.clone() for v in step()])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, refs):
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """Outputs, kept pre-activations and dz of more than 2^31 values: the last rows equal those of a call
    on them alone (the same sums in the same order), forward and backward."""
    m, k, n, tail = 530_000, 64, 4104, 1000
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(m, k, generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    w = (torch.randn(n, k, generator=g, device=DEV) / 8).bfloat16()
    b = torch.randn(n, generator=g, device=DEV, dtype=torch.bfloat16)
    y = linear(x, w, b, activation="gelu")
    dy = torch.empty_like(y).fill_(0.25)
    dy[-tail:] = torch.randn(tail, n, generator=g, device=DEV, dtype=torch.bfloat16)
    (dx,) = torch.autograd.grad(y, x, dy)
    part = x.detach()[-tail:].clone().requires_grad_(True)
    y2 = linear(part, w, b, activation="gelu")
    (dx2,) = torch.autograd.grad(y2, part, dy[-tail:])
    assert torch.equal(y[-tail:], y2)
    X, W = part.detach().double(), w.double()
    ref = act64(X @ W.T + b.double(), "gelu")[0]
    bound = ref.abs() * half(torch.bfloat16) * 1.001 + 1.13 * (k + 2) * U * (X.abs() @ W.abs().T + b.double().abs())
    within(y2, ref, bound + ref.abs() * 2.0 ** -20 + 2.0 ** -22)
    # dx's plan may cut K differently for the two sizes: the sums' own bound, on equal dz
    mag = dy[-tail:].double().abs() * 1.13 @ W.abs()
    within(dx[-tail:], dx2.double(), dx2.double().abs() * 2 * half(torch.bfloat16) + 2 * (n + 2) * U * mag)


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
def test_first_call_of_a_process_is_captured(t):
    """Nothing that a first call sets up is refused by a capturing stream (a process of its own)."""
    import subprocess
    import sys

    from conftest import ROOT

    code = f"""
import torch
from dynaworld_b200.linear import linear, linear_fp8
from dynaworld_b200.norm import quantize_rows_fp8, rms_norm
t = torch.{t}
g = torch.Generator(device="cuda").manual_seed(0)
x = torch.randn(5000, 512, generator=g, device="cuda").to(t).requires_grad_(True)
w = (torch.randn(320, 512, generator=g, device="cuda") / 22).to(t).requires_grad_(True)
n = torch.ones(512, device="cuda", dtype=t)

def step():
    y = rms_norm(x, n)
    z = linear(y, w, activation="gelu")
    a, b = quantize_rows_fp8(y.detach()), quantize_rows_fp8(w.detach())
    return [z.detach(), *torch.autograd.grad(z.float().sum(), [x, w]), linear_fp8(*a, *b, dtype=t),
            linear(x[:3].detach(), w.detach())]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, step()))
print("equal")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert run.returncode == 0 and "equal" in run.stdout, run.stderr[-2000:]


def test_backward_captured_beside_a_live_eager_graph():
    """Capturing .backward() while an eager graph of the same leaf lives: torch refuses it with an
    exception (the leaf's accumulation belongs to the eager stream), the process and the eager graph
    live on; without the eager graph it is captured."""
    x, w, b, r, dy = make(40, 64, 48, torch.float32)
    leaf = w.clone().requires_grad_(True)
    eager = linear(x, leaf).sum()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(graph):
            linear(2 * x, leaf).sum().backward()
    torch.cuda.synchronize()
    leaf.grad = None
    eager.backward()
    ref = leaf.grad.clone()
    within(ref, torch.ones_like(dy).double().T @ x.double(), 42 * U * x.double().abs().sum(0).expand(48, 64))


def test_no_wait_gave_up():
    x, w, b, r, dy = make(300, 264, 144, torch.bfloat16)
    linear(x, w, b)
    assert _lib.lib().gsb_token_status() == _lib.GSB_OK


def test_status_waits_for_every_stream():
    """The status of work that is still queued on a non-blocking stream is not given before that work ends."""
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # about 0.2 s
        done.record()
    assert not done.query()
    assert _lib.lib().gsb_token_status() == _lib.GSB_OK
    assert done.query()


def test_a_wait_that_gives_up_is_reported_once():
    """A wait on a barrier that nothing completes gives up after 1 ms: the status reports it once, on the
    device it happened, and the context goes on."""
    from dynaworld_b200 import diagnostics

    diagnostics.check_token_status()
    with torch.cuda.stream(torch.cuda.Stream()):
        _lib.check("gsb_debug_token_timeout",
                   _lib.lib().gsb_debug_token_timeout(1000, torch.cuda.current_stream().cuda_stream))
    with pytest.raises(_lib.GsbError, match="TIMEOUT"):
        diagnostics.check_token_status(DEV)
    diagnostics.check_token_status()
    x, w, b, r, dy = make(300, 264, 144, torch.bfloat16)
    check(x, w, b, r, dy, "gelu")
    diagnostics.check_token_status(torch.device(DEV))
