"""From decoder tokens to the rendered image: the decoder's heads on the library's kernels.

The reference's splat decoders end in GaussianParameterHeads (src/train/gs_models/blocks.py:84-186):
five MLPs over the tokens [S, T, D] whose outputs, reshaped to [S, T * gaussians_per_token, C], are
the raw Gaussian parameters that ``render_b200_head`` activates inside its projection.  Here the
layers in front of it run on ``rms_norm`` and ``linear`` too, and for serving on their 8-bit forms:

    h      = tokens (+ residual)                                  the residual stream
    h      = h + down(act(up(rms_norm(h))))                       every feed-forward block
    raw_p  = mlp_p(rms_norm(h)), p = xyz, scale, rot, opacity, rgb  (the norm is optional)

``render_b200_tokens`` renders them; gradients reach the tokens and every weight.
"""
from __future__ import annotations

import copy
import math
from dataclasses import dataclass, replace

import torch
import torch.nn.functional as F

from . import _lib
from .linear import linear, linear_fp8
from .norm import quantize_rows_fp8, rms_norm, rms_norm_fp8
from .renderer import HeadActivation, render_b200_head

HEAD_CHANNELS = {"xyz": 3, "scale": 3, "rot": 4, "opacity": 1, "rgb": 3}


@dataclass(frozen=True)
class Layer:
    """weight [n, k] and bias [n]; an 8-bit layer holds e4m3 codes with ``weight_scale`` [n]."""

    weight: torch.Tensor
    bias: torch.Tensor | None = None
    weight_scale: torch.Tensor | None = None

    def quantized(self, bias_dtype: torch.dtype) -> "Layer":
        codes, scale = quantize_rows_fp8(self.weight.detach())
        bias = None if self.bias is None else self.bias.detach().to(bias_dtype)
        return Layer(codes, bias, scale)


@dataclass(frozen=True)
class FeedForward:
    """Pre-norm feed-forward block: h + down(act(up(rms_norm(h))))."""

    norm_weight: torch.Tensor
    up: Layer
    down: Layer


@dataclass(frozen=True)
class TokenHeads:
    """The five head MLPs (tuples of layers, the activation between them) and what stands in front of
    them.  ``activation`` is linear's; ``norm_weight`` None feeds the tokens to the heads as they are."""

    xyz: tuple[Layer, ...]
    scale: tuple[Layer, ...]
    rot: tuple[Layer, ...]
    opacity: tuple[Layer, ...]
    rgb: tuple[Layer, ...]
    head: HeadActivation = HeadActivation()
    activation: str = "gelu"
    norm_weight: torch.Tensor | None = None
    blocks: tuple[FeedForward, ...] = ()
    eps: float = 1e-6

    def __post_init__(self):
        if self.activation not in _lib.ACTIVATIONS:
            raise ValueError(f"Unknown activation: {self.activation!r} (one of {', '.join(_lib.ACTIVATIONS)})")
        per_token = set()
        for name, channels in HEAD_CHANNELS.items():
            layers = getattr(self, name)
            if not layers:
                raise ValueError(f"the {name} head has no layers")
            n = layers[-1].weight.shape[0]
            if n % channels:
                raise ValueError(f"the {name} head gives {n} values per token, not a multiple of {channels}")
            per_token.add(n // channels)
        if len(per_token) != 1:
            raise ValueError(f"the heads give different numbers of Gaussians per token: {sorted(per_token)}")
        quantized = {layer.weight_scale is not None for layer in self._layers()}
        if len(quantized) != 1:
            raise ValueError("either every layer is 8-bit or none is")
        if self.is_fp8 and self.norm_weight is None:
            raise ValueError("8-bit heads need the norm in front of them (norm_weight)")

    def _layers(self):
        for name in HEAD_CHANNELS:
            yield from getattr(self, name)
        for b in self.blocks:
            yield from (b.up, b.down)

    @property
    def is_fp8(self) -> bool:
        return self.xyz[0].weight_scale is not None

    @property
    def gaussians_per_token(self) -> int:
        return self.xyz[-1].weight.shape[0] // HEAD_CHANNELS["xyz"]

    @classmethod
    def from_heads(cls, heads, *, norm_weight=None, blocks=(), eps: float = 1e-6) -> "TokenHeads":
        """Reads a GaussianParameterHeads-like module: its five ``*_head`` MLPs (torch.nn.Linear layers
        with one kind of activation between them) and its activation constants.  The parameters are
        shared, not copied.  An MLP class with a forward of its own is run once (a copy) on four rows and refused
        where that differs from its layers one after the other."""
        activations = set()
        parts = {name: _layers_of(getattr(heads, f"{name}_head"), name, activations) for name in HEAD_CHANNELS}
        if len(activations) > 1:
            raise ValueError(f"the head MLPs use different activations: {sorted(activations)}")
        if blocks and not activations:
            raise ValueError("the feed-forward blocks take the head MLPs' activation, and these heads have none: build "
                             "TokenHeads with the activation named")
        return cls(**parts, head=HeadActivation.from_heads(heads), activation=next(iter(activations), "none"),
                   norm_weight=norm_weight, blocks=tuple(blocks), eps=eps)

    def quantized(self) -> "TokenHeads":
        """The same heads with 8-bit weights, for serving.  Biases of the last layers become float32, as
        the raw outputs then are."""
        if self.is_fp8:
            return self
        parts = {}
        for name in HEAD_CHANNELS:
            layers = getattr(self, name)
            parts[name] = tuple(layer.quantized(torch.float32 if i == len(layers) - 1 else layer.weight.dtype)
                                for i, layer in enumerate(layers))
        blocks = tuple(FeedForward(b.norm_weight.detach(), b.up.quantized(b.up.weight.dtype),
                                   b.down.quantized(b.down.weight.dtype)) for b in self.blocks)
        norm = None if self.norm_weight is None else self.norm_weight.detach()
        return replace(self, **parts, blocks=blocks, norm_weight=norm)


def _walk(module):
    """The module and what it holds, in order: one that stands in several places each time."""
    yield module
    for child in module._modules.values():
        if child is not None:
            yield from _walk(child)


def _plain(m, kind) -> bool:
    """Whether m computes what torch's class does (no forward of its own)."""
    return isinstance(m, kind) and type(m).forward is kind.forward


def _layers_of(mlp, name: str, activations: set) -> tuple[Layer, ...]:
    nn = torch.nn
    layers, between, acts, own_forward = [], None, [], False
    for m in _walk(mlp):
        if m._forward_hooks or m._forward_pre_hooks:
            raise ValueError(f"the {name} head holds a {type(m).__name__} with forward hooks, which would not run here")
        if _plain(m, nn.Linear) and not m._modules:
            if layers and between is None:
                raise ValueError(f"the {name} head has two linear layers with no activation between them")
            if between is not None and not layers:
                raise ValueError(f"the {name} head starts with an activation")
            layers.append(Layer(m.weight, m.bias))
            if between is not None:
                acts.append(between)
            between = None
        elif _plain(m, nn.GELU) or _plain(m, nn.SiLU) or _plain(m, nn.ReLU):
            if between is not None:
                raise ValueError(f"the {name} head has two activations in a row")
            if isinstance(m, nn.GELU):
                between = "gelu" if m.approximate == "none" else "gelu_tanh"
            else:
                between = "silu" if isinstance(m, nn.SiLU) else "relu"
        elif isinstance(m, nn.Dropout):
            if m.training and m.p > 0:
                raise ValueError(f"the {name} head holds an active dropout, which has no kernel here")
        elif m._modules and not isinstance(m, nn.Linear):
            if next(m.parameters(recurse=False), None) is not None or next(m.buffers(recurse=False), None) is not None:
                raise ValueError(f"the {name} head holds a {type(m).__name__} with parameters of its own")
            own_forward |= not _plain(m, nn.Sequential)
        elif not isinstance(m, nn.Identity):
            raise ValueError(f"the {name} head holds a {type(m).__name__}, which has no kernel here")
    if not layers or between is not None:
        raise ValueError(f"the {name} head must end in a linear layer")
    if own_forward and not _is_chain(mlp, acts):
        raise ValueError(f"the {name} head ({type(mlp).__name__}) computes something else than its layers one after "
                         "the other")
    activations.update(acts)
    return tuple(layers)


@torch.no_grad()
def _is_chain(mlp, acts) -> bool:
    """Whether a module with a forward of its own gives on a few rows what its layers give one after the
    other (a skip, a scale or another order does not show in what it holds).  On a copy with values of its
    own in 64 bits: no rounding and no layer that starts at zero hides a difference."""
    fn = {"gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh"), "silu": F.silu, "relu": F.relu}

    def wave(shape, device, phase):
        n = torch.arange(1.0, math.prod(shape) + 1, dtype=torch.float64, device=device)
        return torch.sin(n * n + phase).view(shape)

    mlp = copy.deepcopy(mlp).double()
    for i, p in enumerate(mlp.parameters()):
        p.copy_(wave(p.shape, p.device, i))
    layers = [m for m in _walk(mlp) if isinstance(m, torch.nn.Linear)]
    w = layers[0].weight
    x = 2 * wave((1, 4, w.shape[1]), w.device, 0.5)
    got, ref = mlp(x), x
    for act, layer in zip([None, *acts], layers):
        ref = F.linear(ref if act is None else fn[act](ref), layer.weight, layer.bias)
    return got.shape == ref.shape and float((got - ref).norm()) <= 1e-9 * float(ref.norm())


def _mlp(x, layers, activation):
    for i, layer in enumerate(layers):
        x = linear(x, layer.weight, layer.bias, activation=activation if i + 1 < len(layers) else "none")
    return x


def _mlp_fp8(codes, scale, layers, activation, dtype):
    for i, layer in enumerate(layers):
        last = i + 1 == len(layers)
        y = linear_fp8(codes, scale, layer.weight, layer.weight_scale, layer.bias,
                       activation="none" if last else activation, dtype=torch.float32 if last else dtype)
        if last:
            return y
        codes, scale = quantize_rows_fp8(y)


def head_outputs(tokens: torch.Tensor, heads: TokenHeads, *, residual: torch.Tensor | None = None):
    """The five raw head outputs [S, T * gaussians_per_token, C] of tokens [S, T, D] (or [T, D], one
    set), in the order xyz, scale, rot, opacity, rgb.  ``residual``: the stream that the tokens are
    still to be added to (the last block's output is usually not).  8-bit heads give float32 and run
    without gradients."""
    if tokens.ndim == 2:
        tokens = tokens.unsqueeze(0)
        residual = None if residual is None else residual.unsqueeze(0)
    if tokens.ndim != 3:
        raise ValueError(f"tokens must be [S, T, D] or [T, D], got {tuple(tokens.shape)}")
    h, add = tokens, residual
    for block in heads.blocks:
        if heads.is_fp8:
            got = rms_norm_fp8(h, block.norm_weight, residual=add, eps=heads.eps)
            h, add = (got[2] if add is not None else h), None
            u = linear_fp8(got[0], got[1], block.up.weight, block.up.weight_scale, block.up.bias,
                           activation=heads.activation, dtype=h.dtype)
            codes, scale = quantize_rows_fp8(u)
            h = linear_fp8(codes, scale, block.down.weight, block.down.weight_scale, block.down.bias, residual=h,
                           dtype=h.dtype)
        else:
            got = rms_norm(h, block.norm_weight, residual=add, eps=heads.eps)
            y, h = got if add is not None else (got, h)
            add = None
            u = linear(y, block.up.weight, block.up.bias, activation=heads.activation)
            h = linear(u, block.down.weight, block.down.bias, residual=h)
    if heads.is_fp8:
        codes, scale = rms_norm_fp8(h, heads.norm_weight, residual=add, eps=heads.eps)[:2]
        outs = [_mlp_fp8(codes, scale, getattr(heads, n), heads.activation, h.dtype) for n in HEAD_CHANNELS]
    else:
        if heads.norm_weight is not None:
            h = rms_norm(h, heads.norm_weight, residual=add, eps=heads.eps)
            h = h if add is None else h[0]
        elif add is not None:
            h = h + add
        outs = [_mlp(h, getattr(heads, n), heads.activation) for n in HEAD_CHANNELS]
    sets, count = tokens.shape[0], tokens.shape[1] * heads.gaussians_per_token
    return tuple(o.reshape(sets, count, c) for o, c in zip(outs, HEAD_CHANNELS.values()))


def render_b200_tokens(tokens: torch.Tensor, heads: TokenHeads, *, residual: torch.Tensor | None = None, **render):
    """Renders tokens [S, T, D] through their heads: ``head_outputs`` followed by ``render_b200_head``,
    whose keyword arguments (intrinsics, camera_to_world, height, width, views_per_set, ...) follow.
    Returns image, alpha and depth as it does; differentiable in the tokens, the residual and every
    weight (not with 8-bit heads, which serve only)."""
    raw = head_outputs(tokens, heads, residual=residual)
    return render_b200_head(*raw, head=heads.head, **render)
