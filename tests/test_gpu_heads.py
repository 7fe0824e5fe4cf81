"""render_b200_tokens: norm, feed-forward block, head MLPs and render together, forward and backward,
in float and in 8 bits, against torch layers in 64 bits in front of the same render call."""
import math

import pytest
import torch
import torch.nn.functional as F

from conftest import grad_close
from dynaworld_b200.heads import HEAD_CHANNELS, FeedForward, Layer, TokenHeads, head_outputs, render_b200_tokens
from dynaworld_b200.losses import reconstruction_loss_per_image
from dynaworld_b200.renderer import HeadActivation, render_b200_head
from gpu_helpers import DEV

pytestmark = pytest.mark.gpu

EPS = 1e-6


def make(dtype, dim=72, hidden=136, per_token=4, seed=0):
    g = torch.Generator().manual_seed(seed)

    def layer(n, k, gain=1.0):
        return Layer((gain * torch.randn(n, k, generator=g) / math.sqrt(k)).to(DEV, dtype).requires_grad_(True),
                     (0.1 * torch.randn(n, generator=g)).to(DEV, dtype).requires_grad_(True))

    def norm():
        return (1 + 0.1 * torch.randn(dim, generator=g)).to(DEV, dtype).requires_grad_(True)

    heads = {n: (layer(hidden, dim), layer(per_token * c, hidden, 0.7)) for n, c in HEAD_CHANNELS.items()}
    blocks = (FeedForward(norm(), layer(hidden, dim), layer(dim, hidden)),)
    return TokenHeads(**heads, head=HeadActivation(1.0, 1.0, 3.0, 0.08), activation="gelu", norm_weight=norm(),
                      blocks=blocks, eps=EPS)


def inputs(dtype, sets=2, tokens=45, dim=72, seed=1):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(sets, tokens, dim, generator=g).to(DEV, dtype).requires_grad_(True)
    r = torch.randn(sets, tokens, dim, generator=g).to(DEV, dtype).requires_grad_(True)
    return t, r


def weights(heads):
    out = [heads.norm_weight]
    for b in heads.blocks:
        out += [b.norm_weight, b.up.weight, b.up.bias, b.down.weight, b.down.bias]
    for n in HEAD_CHANNELS:
        for layer in getattr(heads, n):
            out += [layer.weight, layer.bias]
    return out


def reference(tokens, residual, heads):
    """The layers in 64 bits."""

    def norm(h, w):
        return h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()

    def lin(x, layer):
        return x @ layer.weight.double().T + layer.bias.double()

    h = tokens.double() + residual.double()
    for b in heads.blocks:
        h = h + lin(F.gelu(lin(norm(h, b.norm_weight), b.up)), b.down)
    y = norm(h, heads.norm_weight)
    return tuple(lin(F.gelu(lin(y, getattr(heads, n)[0])), getattr(heads, n)[1]).reshape(h.shape[0], -1, c)
                 for n, c in HEAD_CHANNELS.items())


def cameras(sets, views):
    B = sets * views
    c2w = torch.eye(4).expand(B, 4, 4).clone()
    c2w[:, 0, 3] = 0.05 * torch.arange(B)
    intr = torch.tensor([40.0, 40.0, 24.0, 20.0]).expand(B, 4)
    return dict(intrinsics=intr.to(DEV), camera_to_world=c2w.to(DEV), height=40, width=48, views_per_set=views)


# Chains of four products: the relative error of the norm over a row is a few steps of the type per
# layer (half a step each for norm, hidden, block output, stream), against outputs of magnitude 1.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-6), (torch.bfloat16, 8 * 2.0 ** -8),
                                       (torch.float16, 8 * 2.0 ** -11)])
def test_head_outputs(dtype, tol):
    heads, (t, r) = make(dtype), inputs(dtype)
    got = head_outputs(t, heads, residual=r)
    ref = reference(t, r, heads)
    for a, b, c in zip(got, ref, HEAD_CHANNELS.values()):
        assert a.shape == (2, 45 * 4, c) and a.dtype == dtype
        assert float(((a.double() - b).norm() / b.norm()).detach()) < tol
    # half the rows may take another kernel, whose sums have another order: the same bound, not the same bits
    one = head_outputs(t[0], heads, residual=r[0])
    for a, b in zip(one, ref):
        assert a.shape == b[:1].shape
        assert float(((a.double() - b[:1]).norm() / b[:1].norm()).detach()) < tol


def test_image_and_gradients():
    """Image and every gradient in float32 against 64-bit torch layers in front of the same render."""
    heads, (t, r) = make(torch.float32), inputs(torch.float32)
    cam = cameras(2, 2)
    target = torch.rand(4, 3, 40, 48, generator=torch.Generator().manual_seed(2)).to(DEV)
    leaves = [t, r, *weights(heads)]
    image, _, _ = render_b200_tokens(t, heads, residual=r, **cam)
    got = torch.autograd.grad(reconstruction_loss_per_image(image, target).sum(), leaves)
    raw = [v.float() for v in reference(t, r, heads)]
    ref_image, _, _ = render_b200_head(*raw, head=heads.head, **cam)
    ref = torch.autograd.grad(reconstruction_loss_per_image(ref_image, target).sum(), leaves)
    assert (image - ref_image).abs().max().item() <= 1e-4
    for a, b in zip(got, ref):
        ok, err, scale = grad_close(a, b)
        assert ok, f"{tuple(a.shape)}: {err:.3e} vs {scale:.3e}"


def test_training_step_in_bf16():
    heads, (t, r) = make(torch.bfloat16), inputs(torch.bfloat16)
    image, alpha, _ = render_b200_tokens(t, heads, residual=r, **cameras(2, 1))
    target = torch.rand(2, 3, 40, 48, generator=torch.Generator().manual_seed(3)).to(DEV)
    reconstruction_loss_per_image(image, target).sum().backward()
    for v in (t, r, *weights(heads)):
        assert v.grad.dtype == torch.bfloat16 and bool(torch.isfinite(v.grad).all())
        assert bool((v.grad != 0).any())


# 8 bits: e4m3 keeps 2^-4 relative per value (2.6e-2 in norm); every product's sum averages them, the
# weights' and activations' errors of four layers add up to at most about 4 x sqrt(2) x 2.6e-2.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_heads_in_8_bits(dtype):
    heads, (t, r) = make(dtype), inputs(dtype)
    with torch.no_grad():
        served = heads.quantized()
        assert served.is_fp8 and served.quantized() is served
        got = head_outputs(t, served, residual=r)
        ref = reference(t, r, heads)
        for a, b in zip(got, ref):
            assert a.dtype == torch.float32
            assert float((a.double() - b).norm() / b.norm()) < 4 * math.sqrt(2) * 2.6e-2
        image, alpha, _ = render_b200_tokens(t, served, residual=r, **cameras(2, 1))
        full, _, _ = render_b200_tokens(t, heads, residual=r, **cameras(2, 1))
    assert bool(torch.isfinite(image).all()) and float((image - full).abs().mean()) < 0.05
    with pytest.raises(NotImplementedError, match="not differentiable"):
        head_outputs(t, served, residual=r)


def test_one_token_and_captured():
    """A single token through the 8-bit heads, captured once and replayed on other tokens."""
    heads = make(torch.bfloat16).quantized()
    t, r = (v.detach()[:1, :1].clone() for v in inputs(torch.bfloat16))
    t2, r2 = (v.detach()[1:2, :1].clone() for v in inputs(torch.bfloat16))
    with torch.no_grad():
        ref = [v.clone() for v in head_outputs(t2, heads, residual=r2)]
        head_outputs(t, heads, residual=r)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = head_outputs(t, heads, residual=r)
        t.copy_(t2)
        r.copy_(r2)
        graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_no_norm_and_no_blocks():
    heads = make(torch.float32)
    plain = TokenHeads(heads.xyz, heads.scale, heads.rot, heads.opacity, heads.rgb, head=heads.head)
    t, r = inputs(torch.float32)
    got = head_outputs(t, plain, residual=r)
    h = t.double() + r.double()
    for (n, c), a in zip(HEAD_CHANNELS.items(), got):
        l0, l1 = getattr(heads, n)
        ref = F.gelu(h @ l0.weight.double().T + l0.bias.double()) @ l1.weight.double().T + l1.bias.double()
        assert float(((a.double() - ref.reshape(2, -1, c)).norm() / ref.norm()).detach()) < 2e-6


def test_stages_are_traced():
    """Stage events name the operators like the render's stages; without tracing nothing is recorded."""
    from dynaworld_b200 import render

    heads, (t, r) = make(torch.float32), inputs(torch.float32)
    assert render.STAGE_EVENTS is None
    render.STAGE_EVENTS = []
    try:
        sum(v.sum() for v in head_outputs(t, heads, residual=r)).backward()
        torch.cuda.synchronize()
        names = [e[0] for e in render.STAGE_EVENTS]
        assert all(e[1].elapsed_time(e[2]) >= 0 for e in render.STAGE_EVENTS)
    finally:
        render.STAGE_EVENTS = None
    assert names.count("rms_norm") == names.count("rms_norm_bwd") == 2
    assert names.count("linear") == names.count("linear_bwd") == 12


@pytest.mark.parametrize("sets,tokens", [(0, 5), (2, 0), (0, 0)])
def test_no_tokens(sets, tokens):
    """Empty batches keep their shapes, forward and backward and in 8 bits."""
    heads = make(torch.float32)
    t = torch.zeros(sets, tokens, 72, device=DEV, requires_grad=True)
    outs = head_outputs(t, heads, residual=torch.zeros_like(t))
    for o, c in zip(outs, HEAD_CHANNELS.values()):
        assert o.shape == (sets, tokens * 4, c)
    sum(o.sum() for o in outs).backward()
    assert t.grad.shape == t.shape and bool((heads.xyz[0].weight.grad == 0).all())
    with torch.no_grad():
        for o, c in zip(head_outputs(t, heads.quantized()), HEAD_CHANNELS.values()):
            assert o.shape == (sets, tokens * 4, c)
