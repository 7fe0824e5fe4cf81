"""TokenHeads: reading a GaussianParameterHeads-like module and its refusals (no GPU)."""
import pytest
import torch
from torch import nn

from dynaworld_b200.heads import FeedForward, Layer, TokenHeads, head_outputs
from dynaworld_b200.renderer import HeadActivation


class Heads(nn.Module):
    """The attributes of the reference's module (blocks.py:84-186)."""

    def __init__(self, dim=8, hidden=16, per_token=4, act=nn.GELU, **override):
        super().__init__()
        self.xy_extent, self.z_min, self.z_extent, self.scale_init = 1.0, 1.0, 2.0, 0.08
        for name, c in (("xyz", 3), ("scale", 3), ("rot", 4), ("opacity", 1), ("rgb", 3)):
            setattr(self, f"{name}_head",
                    override.get(name) or nn.Sequential(nn.Linear(dim, hidden), act(), nn.Linear(hidden, per_token * c)))


@pytest.mark.parametrize("act,name", [(nn.GELU, "gelu"), (lambda: nn.GELU("tanh"), "gelu_tanh"), (nn.SiLU, "silu"),
                                      (nn.ReLU, "relu")])
def test_reads_the_module(act, name):
    m = Heads(act=act)
    h = TokenHeads.from_heads(m)
    assert h.activation == name and h.gaussians_per_token == 4 and not h.is_fp8
    assert h.head == HeadActivation(1.0, 1.0, 3.0, 0.08)
    assert h.rot[1].weight is m.rot_head[2].weight and h.rot[1].bias is m.rot_head[2].bias


def test_reads_shared_modules_at_every_place():
    """One activation object between all layers, and one layer used twice."""
    act, mid = nn.GELU(), nn.Linear(8, 8)
    m = Heads(rgb=nn.Sequential(nn.Linear(8, 8), act, nn.Linear(8, 8), act, nn.Linear(8, 12)),
              xyz=nn.Sequential(nn.Sequential(mid, nn.GELU()), mid, act, nn.Linear(8, 12)))
    h = TokenHeads.from_heads(m)
    assert all(layer.weight is m.rgb_head[i].weight for layer, i in zip(h.rgb, (0, 2, 4))) and len(h.rgb) == 3
    assert len(h.xyz) == 3 and h.xyz[0].weight is h.xyz[1].weight is mid.weight


@pytest.mark.parametrize("match, make", [
    ("no activation between", lambda: Heads(rgb=nn.Sequential(nn.Linear(8, 8), nn.Linear(8, 12)))),
    ("starts with an activation", lambda: Heads(rgb=nn.Sequential(nn.GELU(), nn.Linear(8, 12)))),
    ("two activations", lambda: Heads(rgb=nn.Sequential(nn.Linear(8, 8), nn.GELU(), nn.GELU(), nn.Linear(8, 12)))),
    ("must end in a linear", lambda: Heads(rgb=nn.Sequential(nn.Linear(8, 12), nn.GELU()))),
    ("holds a LayerNorm", lambda: Heads(rgb=nn.Sequential(nn.LayerNorm(8), nn.Linear(8, 12)))),
    ("active dropout", lambda: Heads(rgb=nn.Sequential(nn.Linear(8, 8), nn.GELU(), nn.Dropout(0.1), nn.Linear(8, 12)))),
    ("different activations", lambda: Heads(rgb=nn.Sequential(nn.Linear(8, 8), nn.SiLU(), nn.Linear(8, 12)))),
    ("not a multiple of 3", lambda: Heads(rgb=nn.Linear(8, 13))),
    ("different numbers of Gaussians", lambda: Heads(rgb=nn.Linear(8, 15))),
])
def test_refused_modules(match, make):
    with pytest.raises(ValueError, match=match):
        TokenHeads.from_heads(make())


class Wrapped(nn.Module):
    """An MLP class of its own around the layers; `how` is what its forward makes of them."""

    def __init__(self, how, *layers):
        super().__init__()
        self.net, self.how = nn.Sequential(*layers), how

    def forward(self, x):
        return self.how(self.net, x)


class Scaled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class Gated(Wrapped):
    def __init__(self, *args):
        super().__init__(*args)
        self.gate = nn.Parameter(torch.zeros(12))


def layers(first=8):
    return nn.Linear(first, 8), nn.GELU(), nn.Linear(8, 12)


def hooked():
    m = nn.Sequential(*layers())
    m[0].register_forward_hook(lambda mod, args, out: 2 * out)
    return m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_reads_a_class_that_runs_its_layers(dtype):
    m = Heads(rgb=Wrapped(lambda net, x: net(x), *layers()), xyz=Wrapped(lambda net, x: net(x) + 0, nn.Linear(8, 12))).to(dtype)
    h = TokenHeads.from_heads(m)
    assert h.rgb[1].weight is m.rgb_head.net[2].weight and len(h.xyz) == 1


@pytest.mark.parametrize("match, make", [
    ("something else", lambda: Wrapped(lambda net, x: 0.5 * net(x), *layers())),
    ("something else", lambda: Wrapped(lambda net, x: net(x) + x[..., :1], *layers())),
    ("something else", lambda: Wrapped(lambda net, x: net(torch.tanh(x)), *layers())),
    ("something else", lambda: Wrapped(lambda net, x: net(x)[..., :6], *layers())),
    ("something else", lambda: nn.Sequential(Wrapped(lambda net, x: net(x) + x, nn.Linear(8, 8)), nn.GELU(), nn.Linear(8, 12))),
    ("parameters of its own", lambda: Gated(lambda net, x: net(x), *layers())),
    ("holds a Scaled", lambda: nn.Sequential(nn.Linear(8, 8), nn.GELU(), Scaled(8, 12))),
    ("forward hooks", hooked),
    ("which has no kernel", lambda: nn.utils.parametrizations.weight_norm(nn.Linear(8, 12))),
])
def test_refuses_what_is_no_chain(match, make):
    with pytest.raises(ValueError, match=match):
        TokenHeads.from_heads(Heads(rgb=make()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [0.5, 1.01])
def test_refuses_a_scale_that_rounding_or_zeros_would_hide(dtype, scale):
    m = Heads(rgb=Wrapped(lambda net, x: scale * net(x), *layers())).to(dtype)
    with pytest.raises(ValueError, match="something else"):
        TokenHeads.from_heads(m)
    nn.init.zeros_(m.rgb_head.net[2].weight)  # a head that starts at zero
    nn.init.zeros_(m.rgb_head.net[2].bias)
    with pytest.raises(ValueError, match="something else"):
        TokenHeads.from_heads(m)


def test_blocks_need_an_activation_to_take():
    """Heads of one layer have no activation between layers: the blocks would run without any."""
    single = {n: nn.Linear(8, c) for n, c in (("xyz", 3), ("scale", 3), ("rot", 4), ("opacity", 1), ("rgb", 3))}
    block = FeedForward(torch.ones(8), Layer(torch.zeros(16, 8)), Layer(torch.zeros(8, 16)))
    with pytest.raises(ValueError, match="activation named"):
        TokenHeads.from_heads(Heads(**single), blocks=(block,))
    h = TokenHeads.from_heads(Heads(**single))
    named = TokenHeads(h.xyz, h.scale, h.rot, h.opacity, h.rgb, head=h.head, activation="silu", blocks=(block,))
    assert named.activation == "silu" and h.activation == "none"


def test_refused_arguments():
    layers = {n: (Layer(torch.zeros(c, 8)),) for n, c in (("xyz", 3), ("scale", 3), ("rot", 4), ("opacity", 1),
                                                         ("rgb", 3))}
    with pytest.raises(ValueError, match="Unknown activation"):
        TokenHeads(**layers, activation="swish")
    with pytest.raises(ValueError, match="no layers"):
        TokenHeads(**{**layers, "rot": ()})
    mixed = {**layers, "rgb": (Layer(torch.zeros(3, 8), None, torch.zeros(3)),)}
    with pytest.raises(ValueError, match="every layer is 8-bit or none"):
        TokenHeads(**mixed)
    coded = {n: (Layer(v[0].weight, None, torch.zeros(v[0].weight.shape[0])),) for n, v in layers.items()}
    with pytest.raises(ValueError, match="need the norm"):
        TokenHeads(**coded)
    heads = TokenHeads(**layers, blocks=(FeedForward(torch.ones(8), Layer(torch.zeros(8, 8)),
                                                     Layer(torch.zeros(8, 8))),))
    with pytest.raises(ValueError, match=r"tokens must be \[S, T, D\]"):
        head_outputs(torch.zeros(8), heads)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        head_outputs(torch.zeros(2, 8), heads)
