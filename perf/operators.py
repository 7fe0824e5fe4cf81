"""The token-side operators of the Gaussian decoder: the cases they are measured on.

The decoder turns tokens into the raw head outputs that ``render_b200_head`` draws: a
root-mean-square norm of the residual stream, matrix products with bias, activation and residual,
and for serving the same with 8-bit operands.  With ``own`` false ``run`` computes them in plain
torch operations in 32 bits; with ``own`` true through the package's public functions.

    linear             y = act(x w^T + b) + r                        (forward, or with its gradients)
    linear_fp8         y = act((q_x q_w^T) s_x s_w + b) + r          (e4m3 operands, per-row scales)
    rms_norm           h = x + r, y = h / sqrt(mean(h^2) + eps) * w  (forward with its gradients)
    rms_norm_fp8       the same norm, written as e4m3 with one scale per row
    quantize_rows_fp8  s = max(|x|, 1e-30) / 448, q = e4m3(x * (448 / max(|x|, 1e-30)))
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E4M3 = torch.float8_e4m3fn
MOST_FLOPS = 3 * 2 * 16384 * 1024 * 4096
MOST_VALUES = 65536 * 2048


def listed():
    return [
        # one token through the first layer of a feed-forward block, as a decode loop calls it
        {"name": "linear_one_token_bf16", "op": "linear", "m": 1, "k": 1024, "n": 4096, "type": "bf16",
         "act": "gelu", "bias": True, "residual": False, "train": False},
        # first layers of the five Gaussian heads (5 x 512) over 4,096 tokens of 8 Gaussians: the
        # 32,768 Gaussians of the dynamic128 workload, in the renderer's own 32-bit type
        {"name": "linear_heads_train_f32", "op": "linear", "m": 4096, "k": 512, "n": 2560, "type": "f32",
         "act": "gelu", "bias": True, "residual": False, "train": True},
        # a ragged batch through odd widths with a residual: nothing is a multiple of a tile
        {"name": "linear_ragged_train_f16", "op": "linear", "m": 1023, "k": 771, "n": 1285, "type": "f16",
         "act": "silu", "bias": True, "residual": True, "train": True},
        # widening layer of a feed-forward block, a training step over a long clip's tokens
        {"name": "linear_ffn_train_bf16", "op": "linear", "m": 16384, "k": 1024, "n": 4096, "type": "bf16",
         "act": "gelu", "bias": True, "residual": False, "train": True},
        # 8-bit serving: a handful of tokens, bound by the weights' bytes
        {"name": "linear_fp8_few_tokens", "op": "linear_fp8", "m": 16, "k": 2048, "n": 8192, "type": "bf16",
         "act": "silu", "bias": True, "residual": False},
        # 8-bit serving: a whole clip's tokens, bound by the tensor cores
        {"name": "linear_fp8_clip", "op": "linear_fp8", "m": 8192, "k": 2048, "n": 8192, "type": "bf16",
         "act": "none", "bias": True, "residual": True},
        # a training step's norm over a long clip's tokens with the block's residual addition
        {"name": "rms_norm_train_bf16", "op": "rms_norm", "m": 16384, "d": 1024, "type": "bf16", "residual": True},
        # odd rows and width, 32 bits, no residual
        {"name": "rms_norm_odd_train_f32", "op": "rms_norm", "m": 4099, "d": 515, "type": "f32", "residual": False},
        # one token's norm in a decode loop
        {"name": "rms_norm_fp8_one_token", "op": "rms_norm_fp8", "m": 1, "d": 1024, "type": "bf16",
         "residual": True},
        # a batch of clips through the norm in front of an 8-bit product
        {"name": "rms_norm_fp8_batch", "op": "rms_norm_fp8", "m": 65536, "d": 2048, "type": "bf16",
         "residual": True},
        # laying out a feed-forward weight for 8-bit serving
        {"name": "quantize_weight_f32", "op": "quantize_rows_fp8", "m": 8192, "d": 2048, "type": "f32"},
        # the activations between two 8-bit layers, odd sizes
        {"name": "quantize_odd_f16", "op": "quantize_rows_fp8", "m": 1021, "d": 771, "type": "f16"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """Half of the widths are multiples of 16, the others whatever comes."""
    v = _between(rng, low, high)
    return max(16, v // 16 * 16) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "linear_fp8", "rms_norm", "rms_norm_fp8", "quantize_rows_fp8"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "linear":
        case = {"op": op, "m": _between(rng, 1, 16384), "k": _width(rng, 24, 4096), "n": _width(rng, 24, 4096),
                "type": kind, "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.4, "train": rng.random() < 0.6}
        while (3 if case["train"] else 1) * 2 * case["m"] * case["k"] * case["n"] > MOST_FLOPS:
            case["m"] = case["m"] * 2 // 3
        return case
    if op == "linear_fp8":
        return {"op": op, "m": _between(rng, 1, 8192), "k": _width(rng, 64, 2048), "n": _width(rng, 64, 8192),
                "type": kind, "act": rng.choice(["none", "gelu", "silu"]), "bias": rng.random() < 0.8,
                "residual": rng.random() < 0.4}
    case = {"op": op, "m": _between(rng, 1, 65536), "d": _width(rng, 64, 8192), "type": kind}
    if op != "quantize_rows_fp8":
        case["residual"] = rng.random() < 0.6
    while case["m"] * case["d"] > MOST_VALUES // 2:
        case["m"] = case["m"] * 2 // 3
    return case


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)

    m = case["m"]
    s = dict(case)
    if case["op"] in ("linear", "linear_fp8"):
        k, n = case["k"], case["n"]
        if case["op"] == "linear":
            s["x"] = normal(m, k)
            s["w"] = normal(n, k, scale=k ** -0.5)
        else:
            for name, v in (("x", normal(m, k, dtype=torch.float32)),
                            ("w", normal(n, k, scale=k ** -0.5, dtype=torch.float32))):
                most = v.abs().amax(1).clamp_min(1e-30)
                s[name], s[name + "_scale"] = (v * (448.0 / most)[:, None]).to(E4M3), most / 448.0
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["r"] = normal(m, n) if case["residual"] else None
        if case.get("train"):
            s["dy"] = normal(m, n, scale=0.1)
            s["leaves"] = [v.requires_grad_(True) for v in (s["x"], s["w"], s["b"], s["r"]) if v is not None]
        return s
    d = case["d"]
    s["x"] = normal(m, d)
    if case["op"] == "quantize_rows_fp8":
        return s
    s["r"] = normal(m, d, scale=2.0) if case["residual"] else None
    s["w"] = normal(d, scale=0.1, shift=1.0)
    if case["op"] == "rms_norm":
        s["dy"] = normal(m, d, scale=0.1)
        s["dh"] = normal(m, d, scale=0.1) if case["residual"] else None
        s["leaves"] = [v.requires_grad_(True) for v in (s["x"], s["w"], s["r"]) if v is not None]
    return s


# ---- the plain forms: elementary torch operations in 32 bits, rounded once ------------------------

C_TANH = math.sqrt(2.0 / math.pi)


def _act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(C_TANH * (z + 0.044715 * z * z * z)))
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        t = torch.tanh(C_TANH * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * C_TANH * (1.0 + 3 * 0.044715 * z * z)
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_linear(s):
    t = TYPES[s["type"]]
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        z = x @ w.t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, s["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        out = {"y": y.to(t)}
        if s["train"]:
            dz = s["dy"].float() * _act_grad(z, s["act"])
            out["dx"], out["dw"] = (dz @ w).to(t), (dz.t() @ x).to(t)
            if s["b"] is not None:
                out["db"] = dz.sum(0).to(t)
            if s["r"] is not None:
                out["dr"] = s["dy"]
        return out


def _plain_linear_fp8(s):
    z = (s["x"].float() @ s["w"].float().t()) * s["x_scale"][:, None] * s["w_scale"][None, :]
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(TYPES[s["type"]])}


def _plain_norm(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    rstd = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    return h, rstd


def _plain_rms_norm(s):
    t = TYPES[s["type"]]
    with torch.no_grad():
        h, rstd = _plain_norm(s)
        w, dy = s["w"].float(), s["dy"].float()
        out = {"y": (h * rstd * w).to(t)}
        g = dy * w
        dx = rstd * (g - h * (rstd * rstd) * (g * h).mean(1, keepdim=True))
        if s["r"] is not None:
            out["h"] = h.to(t)
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(t)
        out["dw"] = (dy * h * rstd).sum(0).to(t)
        return out


def _quantize(v):
    most = v.abs().amax(1).clamp_min(1e-30)
    return {"q": (v * (448.0 / most)[:, None]).to(E4M3), "scale": most / 448.0}


def _plain_rms_norm_fp8(s):
    h, rstd = _plain_norm(s)
    out = _quantize(h * rstd * s["w"].float())
    if s["r"] is not None:
        out["h"] = h.to(TYPES[s["type"]])
    return out


# ---- the package's functions, as a user calls them -----------------------------------------------


def _own_linear(s):
    from dynaworld_b200.linear import linear

    y = linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["r"])
    if not s["train"]:
        return {"y": y}
    grads = iter(torch.autograd.grad(y, s["leaves"], s["dy"]))
    out = {"y": y.detach(), "dx": next(grads), "dw": next(grads)}
    if s["b"] is not None:
        out["db"] = next(grads)
    if s["r"] is not None:
        out["dr"] = next(grads)
    return out


def _own_linear_fp8(s):
    from dynaworld_b200.linear import linear_fp8

    return {"y": linear_fp8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["b"], activation=s["act"],
                            residual=s["r"], dtype=TYPES[s["type"]])}


def _own_rms_norm(s):
    from dynaworld_b200.norm import rms_norm

    if s["r"] is None:
        y = rms_norm(s["x"], s["w"], eps=EPS)
        dx, dw = torch.autograd.grad(y, s["leaves"], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, h = rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
    dx, dw, _ = torch.autograd.grad([y, h], s["leaves"], [s["dy"], s["dh"]])
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dw": dw}


def _own_rms_norm_fp8(s):
    from dynaworld_b200.norm import rms_norm_fp8

    got = rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=EPS)
    return dict(zip(("q", "scale", "h"), got))


def _own_quantize(s):
    from dynaworld_b200.norm import quantize_rows_fp8

    return dict(zip(("q", "scale"), quantize_rows_fp8(s["x"])))


def run(s):
    op = s["op"]
    if op == "linear":
        return _own_linear(s) if own else _plain_linear(s)
    if op == "linear_fp8":
        return _own_linear_fp8(s) if own else _plain_linear_fp8(s)
    if op == "rms_norm":
        return _own_rms_norm(s) if own else _plain_rms_norm(s)
    if op == "rms_norm_fp8":
        return _own_rms_norm_fp8(s) if own else _plain_rms_norm_fp8(s)
    return _own_quantize(s) if own else _quantize(s["x"].float())


def work(case):
    m, e = case["m"], SIZE[case["type"]]
    if case["op"] in ("linear", "linear_fp8"):
        k, n = case["k"], case["n"]
        products = 2 * m * k * n
        if case["op"] == "linear_fp8":
            read = m * k + n * k + 4 * (m + n)
        else:
            read = (m * k + n * k) * e
        both = read + (n * case["bias"] + m * n * (1 + case["residual"])) * e
        if not case.get("train"):
            return {"bytes": both, "flops": products}
        # the backward reads dy and writes the gradients of x, w and b (the residual's is dy)
        return {"bytes": both + (m * n + m * k + n * k + n * case["bias"]) * e, "flops": 3 * products}
    d = case["d"]
    if case["op"] == "quantize_rows_fp8":
        return {"bytes": m * d * (e + 1) + 4 * m, "flops": 3 * m * d}
    streams = 2 if case["residual"] else 1
    if case["op"] == "rms_norm_fp8":
        # x (and r) in; codes, scales (and h) out
        return {"bytes": m * d * (e * (2 * streams - 1) + 1) + 4 * m + d * e, "flops": 8 * m * d}
    # x, dy (and r, dh) in; y, dx (and h) out; w in, dw out
    return {"bytes": m * d * e * (7 if case["residual"] else 4) + 2 * d * e, "flops": 16 * m * d}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def _phi(z):
    """The normal distribution function."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _exact_act(z, kind):
    """(act(z), act'(z)) in 64 bits."""
    if kind == "relu":
        step = torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        return z * step, step
    if kind == "gelu":
        cdf = _phi(z)
        return z * cdf, cdf + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z.pow(3))
        gate = torch.sigmoid(2 * u)
        return z * gate, gate + z * gate * (1 - gate) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z.square())
    if kind == "silu":
        gate = torch.sigmoid(z)
        return z * gate, gate + z * gate * (1 - gate)
    return z, torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    op = case["op"]
    if op in ("linear", "linear_fp8"):
        x, w = wide["x"], wide["w"]
        if op == "linear_fp8":
            x, w = x * wide["x_scale"].unsqueeze(1), w * wide["w_scale"].unsqueeze(1)
        z = torch.mm(x, w.T)
        if "b" in wide:
            z += wide["b"]
        y, slope = _exact_act(z, case["act"])
        del z
        out = {"y": y + wide["r"] if "r" in wide else y}
        if case.get("train"):
            dz = wide["dy"] * slope
            out["dx"], out["dw"] = torch.mm(dz, w), torch.mm(dz.T, x)
            if "b" in wide:
                out["db"] = dz.sum(dim=0)
            if "r" in wide:
                out["dr"] = wide["dy"]
        return out
    h = wide["x"] + wide["r"] if "r" in wide else wide["x"]
    if op == "quantize_rows_fp8":
        top = torch.clamp(h.abs().max(dim=1).values, min=1e-30)
        return {"q": h * (448 / top).unsqueeze(1), "scale": top / 448}
    norm = torch.rsqrt(h.square().sum(dim=1) / h.shape[1] + EPS).unsqueeze(1)
    unit = h * norm
    y = unit * wide["w"]
    if op == "rms_norm_fp8":
        top = torch.clamp(y.abs().max(dim=1).values, min=1e-30)
        out = {"q": y * (448 / top).unsqueeze(1), "scale": top / 448}
        if "r" in wide:
            out["h"] = h
        return out
    out = {"y": y}
    slope = wide["dy"] * wide["w"]
    dx = norm * (slope - unit * (slope * unit).sum(dim=1, keepdim=True) / h.shape[1])
    if "r" in wide:
        out["h"] = h
        dx += wide["dh"]
    out["dx"] = dx
    out["dw"] = (wide["dy"] * unit).sum(dim=0)
    return out
