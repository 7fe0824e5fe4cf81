"""rms_norm, rms_norm_fp8 and quantize_rows_fp8 on the GPU against their formulas in 64 bits.

Bounds.  u = 2^-24 is half a float step; half(t) half a relative step of the type t.  A sum over D
values with at most 64 of them added one after the other per thread and the rest in trees is within
80 u of the sum of magnitudes; with the handful of roundings after it every factor below is within
128 u.  The backward forms h from x and the residual, unrounded."""
import pytest
import torch

from dynaworld_b200.norm import quantize_rows_fp8, rms_norm, rms_norm_fp8
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn
EPS = 1e-5


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half a step of the type's subnormals."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(rows, dim, t, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g).to(t)
    r = (2 * torch.randn(rows, dim, generator=g)).to(t) if residual else None
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(t)
    dy = torch.randn(rows, dim, generator=g).to(t)
    dh = torch.randn(rows, dim, generator=g).to(t)
    return [None if v is None else v.to(DEV) for v in (x, r, w, dy, dh)]


def within(got, ref, bound):
    assert got.shape == ref.shape
    over = ((got.double() - ref).abs() - bound)
    assert bool((over <= 0).all()), f"{over.max().item():.3e} past the bound"


def check_all(x, r, w, dy, dh, t):
    leaves = [v.clone().requires_grad_(True) for v in (x, w)] + ([] if r is None else [r.clone().requires_grad_(True)])
    if r is None:
        y = rms_norm(leaves[0], leaves[1], eps=EPS)
        grads = torch.autograd.grad(y, leaves, dy)
    else:
        y, h_out = rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
        grads = torch.autograd.grad([y, h_out], leaves, [dy, dh])
    X, W, G = x.double(), w.double(), dy.double()
    H = X if r is None else X + r.double()
    D = x.shape[-1]
    rstd = 1 / (H.square().mean(-1, keepdim=True) + EPS).sqrt()
    ref = H * rstd * W
    within(y, ref, ref.abs() * (half(t) + 128 * U) + tiny(t))
    if r is not None:
        within(h_out, H, H.abs() * (half(t) + U) + tiny(t))
    dot = (G * W * H).sum(-1, keepdim=True) / D
    mag = (G * W * H).abs().sum(-1, keepdim=True) / D
    dx = rstd * (G * W - H * rstd.square() * dot)
    terms = rstd * ((G * W).abs() + H.abs() * rstd.square() * mag)
    if r is not None:
        dx = dx + dh.double()
        terms = terms + dh.double().abs()
    within(grads[0], dx, dx.abs() * half(t) + 128 * U * terms + tiny(t))
    if r is not None:
        assert torch.equal(grads[2], grads[0])
    dw = (G * H * rstd).reshape(-1, D).sum(0)
    mag = (G * H * rstd).abs().reshape(-1, D).sum(0)
    rows = x.numel() // D
    within(grads[1], dw, dw.abs() * half(t) + mag * ((rows + 128) * U) + tiny(t))


# one value, one access, a warp's row, odd widths (scalar accesses), a block's row, rows wider than
# a block's registers (16-bit: 256 x 8 x 8 values; scalar: 256 x 8)
SHAPES = [(1, 1), (3, 8), (5, 31), (1, 1024), (33, 257), (1000, 512), (7, 515), (9, 2048), (4, 4100), (2, 16384),
          (3, 16400), (5, 2051), (2300, 64)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_norm_and_gradients(rows, dim, t, residual):
    check_all(*make(rows, dim, t, seed=dim, residual=residual), t)


# many aligned rows: a warp per row (two, four and, forward, eight accesses), a block per row; row
# counts that leave the last round ragged; rows apart in a wider tensor
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", [(4739, 256), (9500, 520), (4800, 1024), (5001, 2048), (1000, 2080), (700, 4096),
                                      (611, 8192), (601, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_many_rows(rows, dim, t, residual):
    x, r, w, dy, dh = make(rows, dim, t, seed=rows, residual=residual)
    wide = torch.full((rows, dim + 64), float("nan"), dtype=t, device=DEV)
    wide[:, 32:32 + dim] = x
    part = wide[:, 32:32 + dim]
    check_all(x, r, w, dy, dh, t)
    got, ref = rms_norm(part, w, eps=EPS), rms_norm(x, w, eps=EPS)
    assert torch.equal(got, ref)
    q, s = quantize_rows_fp8(part)
    rq, rs = ref_codes(x.float())
    assert torch.equal(s, rs) and torch.equal(q.view(torch.uint8), rq.view(torch.uint8))


@pytest.mark.parametrize("t", TYPES)
def test_leading_dimensions_and_strides(t):
    """[2, 3, D] inputs, rows of a wider tensor (aligned and not), a transposed input."""
    x, r, w, dy, dh = make(6, 64, t)
    a, ha = rms_norm(x, w, residual=r, eps=EPS)
    b, hb = rms_norm(x.view(2, 3, 64), w, residual=r.view(2, 3, 64), eps=EPS)
    assert b.shape == (2, 3, 64) and torch.equal(a, b.view(6, 64)) and torch.equal(ha, hb.view(6, 64))
    for first, width in ((0, 96), (8, 96), (3, 77)):
        wide = torch.full((6, width), float("nan"), dtype=t, device=DEV)
        wide[:, first:first + 64] = x
        leaf = wide.requires_grad_(True)
        check = rms_norm(leaf[:, first:first + 64], w, eps=EPS)
        ref = rms_norm(x, w, eps=EPS)
        within(check, ref.double(), ref.double().abs() * 2 * (half(t) + 128 * U))
        (g,) = torch.autograd.grad(check, leaf, dy)
        assert bool((g[:, :first] == 0).all()) and bool((g[:, first + 64:] == 0).all())
    xt = x.t().contiguous().t()
    assert torch.equal(rms_norm(xt, w, eps=EPS), rms_norm(x, w, eps=EPS))
    # an expanded gradient (a sum's)
    leaf = x.clone().requires_grad_(True)
    rms_norm(leaf, w, eps=EPS).sum().backward()
    leaf2 = x.clone().requires_grad_(True)
    rms_norm(leaf2, w, eps=EPS).backward(torch.ones_like(x))
    assert torch.equal(leaf.grad, leaf2.grad)


def test_only_one_output_used():
    x, r, w, dy, dh = make(5, 64, torch.float32)
    leaves = [v.clone().requires_grad_(True) for v in (x, r, w)]
    y, h = rms_norm(leaves[0], leaves[2], residual=leaves[1])
    gx, gr, gw = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    assert torch.equal(gx, dh) and torch.equal(gr, dh) and bool((gw == 0).all())
    gx, gr, gw = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    full = torch.autograd.grad([y, h], leaves, [dy, torch.zeros_like(dh)])
    assert torch.equal(gx, full[0]) and torch.equal(gw, full[2])


@pytest.mark.parametrize("t", TYPES)
def test_no_rows(t):
    w = torch.ones(16, dtype=t, device=DEV, requires_grad=True)
    x = torch.empty(0, 16, dtype=t, device=DEV, requires_grad=True)
    y, h = rms_norm(x, w, residual=torch.empty(0, 16, dtype=t, device=DEV))
    assert y.shape == h.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16) and bool((w.grad == 0).all())
    q, s = quantize_rows_fp8(x.detach())
    assert q.shape == (0, 16) and s.shape == (0,)


def test_zero_rows_and_nonfinite_rows_stay_apart():
    """A row of zeros gives zeros; a row with a NaN or infinity does not touch its neighbours."""
    x, r, w, dy, dh = make(6, 300, torch.float32)
    x[1] = 0
    x[2, 7] = float("nan")
    x[4, 9] = float("inf")
    y = rms_norm(x, w, eps=0.0 + 1e-6)
    assert bool((y[1] == 0).all()) and bool(y[2].isnan().all()) and bool(y[4, 9].isnan())
    clean = [0, 3, 5]
    ref = rms_norm(x[clean].contiguous(), w, eps=1e-6)
    assert torch.equal(y[clean], ref)


def ref_codes(y):
    """On the host, tensor by tensor: a GPU division by a Python number multiplies by its reciprocal."""
    y = y.cpu()
    top, most = y.abs().amax(-1).clamp_min(1e-30), torch.full((y.shape[0],), 448.0)
    return (y * torch.div(most, top)[..., None]).to(E4M3).to(DEV), torch.div(top, most).to(DEV)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_quantised_rows_are_exact(rows, dim, t):
    """One multiplication and one rounding in float: the codes and scales are those of the formula."""
    x = make(rows, dim, t, seed=rows)[0]
    q, s = quantize_rows_fp8(x)
    rq, rs = ref_codes(x.float())
    assert torch.equal(s, rs)
    assert torch.equal(q.view(torch.uint8), rq.view(torch.uint8))


@pytest.mark.parametrize("t", TYPES)
def test_quantised_special_rows(t):
    x = make(8, 129, t)[0]
    x[0] = 0
    x[1] = torch.finfo(t).smallest_normal
    x[2] = 0
    x[2, 5] = torch.finfo(t).max
    x[3, 128] = float("nan")
    x[4, 0] = float("-inf")
    x[5] = -x[6]
    q, s = quantize_rows_fp8(x)
    v = q.float() * s[:, None]
    assert bool((v[0] == 0).all()) and float(s[0]) > 0
    assert bool(torch.isfinite(v[[0, 1, 2, 5, 6, 7]]).all())
    assert bool(v[3].isnan().all()) and bool(v[4].isnan().all())
    assert torch.equal(q[5].float(), -q[6].float()) and torch.equal(s[5], s[6])
    # within half a step of e4m3 (2^-4 relative, subnormal step 2^-9 of the scale)
    for k in (2, 5, 7):
        err = (v[k].double() - x[k].double()).abs()
        assert bool((err <= x[k].double().abs() * 2.0 ** -4 + 2.0 ** -10 * s[k].double() * (1 + 1e-6)).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [256, 520, 1024, 2048])
def test_special_rows_among_many(dim, t):
    """Rows that come through the ring of copies: a NaN, an infinity or a row of zeros stays in its row,
    forward, in 8 bits and backward."""
    x, r, w, dy, _ = make(9500, dim, t, seed=dim)
    x[5], r[5] = 0, 0
    clean = x.clone()
    x[7, 3], x[4000, 9], x[9499, 0] = float("nan"), float("inf"), float("-inf")
    bad = torch.tensor([7, 4000, 9499], device=DEV)
    rest = torch.ones(9500, dtype=torch.bool, device=DEV).index_fill(0, bad, False)
    for a, b in zip(rms_norm(x, w, residual=r), rms_norm(clean, w, residual=r)):
        assert torch.equal(a[rest], b[rest]) and bool((a[5] == 0).all())
    for got, ref in ((rms_norm_fp8(x, w, residual=r), rms_norm_fp8(clean, w, residual=r)),
                     (quantize_rows_fp8(x), quantize_rows_fp8(clean))):
        assert torch.equal(got[0].view(torch.uint8)[rest], ref[0].view(torch.uint8)[rest])
        assert torch.equal(got[1][rest], ref[1][rest])
        value = got[0].float() * got[1][:, None]
        assert bool(value[bad].isnan().all()) and bool((value[5] == 0).all())
    leaf = clean.requires_grad_(True)
    dirty = dy.clone()
    dirty[bad] = float("nan")
    for a, b in zip(torch.autograd.grad(rms_norm(leaf, w, residual=r)[0], leaf, dy),
                    torch.autograd.grad(rms_norm(leaf, w, residual=r)[0], leaf, dirty)):
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", SHAPES + [(4800, 1024), (5001, 2048), (700, 4096), (601, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_in_8_bits(rows, dim, t, residual):
    x, r, w, _, _ = make(rows, dim, t, seed=dim + 1, residual=residual)
    got = rms_norm_fp8(x, w, residual=r, eps=EPS)
    H = x.double() if r is None else x.double() + r.double()
    y = H / (H.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    top = y.abs().amax(-1).clamp_min(1e-30)
    within(got[1], top / 448, top / 448 * 130 * U)
    value = got[0].float().double() * got[1].double()[:, None]
    # half a step of the code, taken at the value itself, and the float error of y and the scale
    step = y.abs() * 2.0 ** -4 + 2.0 ** -10 * (top / 448)[:, None]
    within(value, y, step * (1 + 1e-4) + y.abs() * 300 * U)
    if r is not None:
        within(got[2], H, H.abs() * (half(t) + U) + tiny(t))


def test_same_bits_every_run():
    x, r, w, dy, dh = make(3001, 264, torch.bfloat16)
    def once():
        leaves = [v.clone().requires_grad_(True) for v in (x, r, w)]
        y, h = rms_norm(leaves[0], leaves[2], residual=leaves[1])
        return [y, h, *torch.autograd.grad([y, h], leaves, [dy, dh])]
    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_gradient_against_differences():
    """Central differences in 64 bits of the formula, against the kernel's 32-bit gradients: the
    difference quotient's own error is h^2 / 6 times third derivatives (below 1e-7 here)."""
    x, r, w, dy, _ = make(2, 40, torch.float32, seed=3)
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    gx, gw = torch.autograd.grad(rms_norm(leaves[0], leaves[1], eps=EPS), leaves, dy)

    def f(X, W):
        return (X / (X.square().mean(-1, keepdim=True) + EPS).sqrt() * W * dy.double()).sum()

    step = 1e-4
    X, W = x.double(), w.double()
    for idx in ((0, 0), (1, 17), (1, 39)):
        e = torch.zeros_like(X)
        e[idx] = step
        assert abs(float((f(X + e, W) - f(X - e, W)) / (2 * step)) - float(gx[idx])) < 1e-5
    e = torch.zeros_like(W)
    e[11] = step
    assert abs(float((f(X, W + e) - f(X, W - e)) / (2 * step)) - float(gw[11])) < 1e-5


def test_other_stream_and_captured_graph():
    x, r, w, _, _ = make(65, 520, torch.bfloat16)
    ref, ref_h = rms_norm(x, w, residual=r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y, h = rms_norm(x, w, residual=r)
    side.synchronize()
    assert torch.equal(y, ref) and torch.equal(h, ref_h)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s, h2 = rms_norm_fp8(x, w, residual=r)
    x.mul_(0.5)
    graph.replay()
    q1, s1, h1 = rms_norm_fp8(x, w, residual=r)
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1) and torch.equal(h1, h2)


def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last rows equal those of a call on them alone."""
    rows, dim, tail = 1_060_000, 2048, 500
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(rows, dim, generator=g, device=DEV, dtype=torch.bfloat16)
    w = torch.randn(dim, generator=g, device=DEV, dtype=torch.bfloat16)
    leaf = x.requires_grad_(True)
    y, h = rms_norm(leaf, w, residual=x.detach())
    dy = torch.full_like(y, 0.5)
    (dx,) = torch.autograd.grad([y, h], leaf, [dy, dy])
    part = x.detach()[-tail:].clone().requires_grad_(True)
    y2, h2 = rms_norm(part, w, residual=part.detach())
    (dx2,) = torch.autograd.grad([y2, h2], part, [dy[-tail:], dy[-tail:]])
    bound = 2 * half(torch.bfloat16) + 300 * U  # one rounding either side; the sums' orders may differ
    for a, b in ((y, y2), (h, h2), (dx, dx2)):
        within(a[-tail:].detach(), b.detach().double(), b.detach().double().abs() * bound + 1e-5)
    del dx, dy, y, h
    q, s = quantize_rows_fp8(x.detach())
    q2, s2 = quantize_rows_fp8(part.detach())
    assert torch.equal(q[-tail:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-tail:], s2)


def test_refusals_on_the_gpu():
    x = torch.zeros(2, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV)
    with pytest.raises(NotImplementedError, match="not differentiable"):
        rms_norm_fp8(x, w)
    with pytest.raises(NotImplementedError, match="not differentiable"):
        quantize_rows_fp8(x)
    with pytest.raises(RuntimeError, match="is on cpu"):
        rms_norm(x, w.cpu())
    (g,) = torch.autograd.grad(rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
