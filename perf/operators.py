"""The cases on which the dense linear layer (bias, activation and gated residual in its epilogue) and layer norm are
measured, each forward and as a training step, with their plain forms in 32 bits and their definitions in 64.

``linear``: y = r + g[row // rows_per_group] * act(x W^T + b); ``layer_norm``: y = (x - mean) * rstd * w + b with one
row of w and b for all rows or for each group of rows_per_group rows. A training step returns the output and the
gradient of every input."""

import importlib
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6


def _linear(name, m, k, n, act="none", bias=True, groups=0, type="bf16", train=False):
    """groups: rows of the gate, each for m / groups rows of the output; 0: neither gate nor residual."""
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias, "groups": groups,
            "type": type, "train": train}


def _norm(name, m, d, groups=1, type="bf16", wtype="bf16", train=False):
    """groups: rows of weight and bias, each for m / groups rows; 0: no weight and bias."""
    return {"name": name, "op": "norm", "m": m, "d": d, "groups": groups, "type": type, "wtype": wtype, "train": train}


def listed():
    return [
        # the adaLN output layer of a 2048-wide block for two samples: 3 * 2048 outputs from the 256-wide bottleneck
        _linear("linear adaln 2 rows", 2, 256, 6144, bias=False),
        # one token through an MLP's input layer: the weight is all there is to read
        _linear("linear one token", 1, 2048, 8192, act="gelu"),
        # a handful of tokens through the widest layer (5120 -> 20480)
        _linear("linear 24 tokens", 24, 5120, 20480, act="silu", type="f16"),
        # keys of the cross-attention from a ragged text context
        _linear("linear text context", 333, 1024, 5120, bias=False),
        # the patch embedding: 17 channels of 2 x 2 patches, whose 68 inputs are no multiple of 8
        _linear("linear patch embedding", 5001, 68, 2048),
        # the widest MLP's output layer with the block's gated residual, two samples of 4096 tokens
        _linear("linear mlp out residual", 8192, 20480, 5120, bias=False, groups=2),
        # a training step of the 2048-wide block's MLP input layer
        _linear("linear train mlp in", 8192, 2048, 8192, act="gelu", train=True),
        # a training step on odd sizes with every operand
        _linear("linear train odd", 777, 1001, 1013, act="gelu_tanh", groups=7, type="f16", train=True),
        # the norm in front of the adaLN of a few rows
        _norm("norm 2 rows", 2, 5120),
        # the adaLN norm of the 5120-wide block over two samples of 8192 tokens, a weight row a sample
        _norm("norm grouped", 16384, 5120, groups=2),
        # a training step of an affine norm over long rows of tokens, master weights in 32 bits
        _norm("norm train", 16384, 2048, wtype="f32", train=True),
        # a training step in 32 bits on an odd width
        _norm("norm train odd", 4099, 1001, type="f32", wtype="f32", train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    train = rng.random() < 0.4
    if rng.random() < 0.6:
        while True:
            m, k, n = _log(rng, 1, 16384), _log(rng, 16, 20480), _log(rng, 8, 20480)
            if rng.random() < 0.5:  # widths of a model are mostly round, lengths are not
                k, n = max(16, k // 64 * 64), max(8, n // 64 * 64)
            groups = rng.choice([0, 0, 1, 2, 5])
            m = max(1, m // max(1, groups)) * max(1, groups)
            c = _linear("", m, k, n, rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]),
                        rng.random() < 0.5, groups, rng.choice(["bf16", "bf16", "f16"]), train)
            if (6 if train else 2) * m * k * n <= 1.7e12:
                break
    else:
        while True:
            m, d = _log(rng, 1, 65536), _log(rng, 8, 20480)
            if rng.random() < 0.5:
                d = max(8, d // 64 * 64)
            groups = rng.choice([0, 1, 1, 2, 7])
            m = max(1, m // max(1, groups)) * max(1, groups)
            t = rng.choice(["bf16", "bf16", "f16", "f32"])
            c = _norm("", m, d, groups, t, rng.choice([t, "f32"]), train)
            if m * d <= 16384 * 5120:
                break
    del c["name"]
    return c


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, device="cuda", generator=g) * scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[case["type"]]
    m = case["m"]
    s = {"case": case}
    if case["op"] == "linear":
        k, n, groups = case["k"], case["n"], case["groups"]
        # activations after a norm: unit variance, a few loud channels
        loud = torch.exp(0.5 * _normal(g, (k,)))
        s["x"] = (_normal(g, (m, k)) * loud).to(t)
        s["weight"] = _normal(g, (n, k), 1.0 / math.sqrt(k)).to(t)
        s["bias"] = _normal(g, (n,), 0.1).to(t) if case["bias"] else None
        s["residual"] = _normal(g, (m, n), 2.0).to(t) if groups else None
        s["gate"] = (0.3 + _normal(g, (groups, n), 0.3)).to(t) if groups else None
        s["dy"] = _normal(g, (m, n), 0.1).to(t) if case["train"] else None
        names = ("x", "weight", "bias", "residual", "gate")
    else:
        d, groups, wt = case["d"], case["groups"], _TYPES[case["wtype"]]
        # the residual stream: a mean away from zero and channels far louder than the rest
        loud = torch.exp(_normal(g, (d,)))
        s["x"] = (_normal(g, (m, d)) * loud + 0.5).to(t)
        shape = (d,) if groups == 1 else (groups, d)
        s["weight"] = (1 + _normal(g, shape, 0.2)).to(wt) if groups else None
        s["bias"] = _normal(g, shape, 0.2).to(wt) if groups else None
        s["dy"] = _normal(g, (m, d), 0.1).to(t) if case["train"] else None
        names = ("x", "weight", "bias")
    s["leaves"] = [nm for nm in names if s[nm] is not None]
    if case["train"]:
        for nm in s["leaves"]:
            s[nm].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _act(z, kind):
    """(act(z), act'(z))"""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c, a = math.sqrt(2 / math.pi), 0.044715
    th = torch.tanh(c * (z + a * z * z * z))
    return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * a * z * z)


def _plain_linear(s):
    case, t = s["case"], s["x"].dtype
    m, n, groups = case["m"], case["n"], case["groups"]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    h, slope = _act(z, case["act"])
    y = h
    if groups:
        gate = s["gate"].detach().float().view(groups, 1, n)
        y = s["residual"].detach().float() + (gate * h.view(groups, m // groups, n)).view(m, n)
    if not case["train"]:
        return y.to(t)
    dy = s["dy"].float()
    dh = (gate * dy.view(groups, m // groups, n)).view(m, n) if groups else dy
    dz = dh * slope
    grads = {"x": dz @ w, "weight": dz.t() @ x}
    if s["bias"] is not None:
        grads["bias"] = dz.sum(0)
    if groups:
        grads["residual"] = dy
        grads["gate"] = (dy * h).view(groups, m // groups, n).sum(1)
    return {"y": y.to(t), "grads": {nm: v.to(t) for nm, v in grads.items()}}


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    m, d, groups = case["m"], case["d"], max(1, case["groups"])
    x = s["x"].detach().float()
    c = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + _EPS)
    xh = (c * rstd).view(groups, m // groups, d)
    affine = s["weight"] is not None
    y = xh
    if affine:
        w = s["weight"].detach().float().view(groups, 1, d)
        y = xh * w + s["bias"].detach().float().view(groups, 1, d)
    y = y.reshape(m, d).to(t)
    if not case["train"]:
        return y
    dy = s["dy"].float().view(groups, m // groups, d)
    u = dy * w if affine else dy
    dx = rstd * (u - u.mean(2, keepdim=True) - xh * (u * xh).mean(2, keepdim=True)).reshape(m, d)
    grads = {"x": dx.to(t)}
    if affine:
        grads["weight"] = (dy * xh).sum(1).view(s["weight"].shape).to(s["weight"].dtype)
        grads["bias"] = dy.sum(1).view(s["bias"].shape).to(s["bias"].dtype)
    return {"y": y, "grads": grads}


# ------------------------------------------------------------------------------------------- the framework's calls
def _module(name):
    return importlib.import_module("comfyui-weightferry_b200.enhancers." + name)


def _own_call(s):
    case = s["case"]
    if case["op"] == "linear":
        return _module("fused_linear").linear(
            s["x"], s["weight"], s["bias"], activation=case["act"], residual=s["residual"], gate=s["gate"])
    return _module("fused_norm").layer_norm(s["x"], s["weight"], s["bias"], eps=_EPS)


def run(state):
    if not own:
        return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_norm(state)
    y = _own_call(state)
    if not state["case"]["train"]:
        return y
    grads = torch.autograd.grad(y, [state[nm] for nm in state["leaves"]], state["dy"])
    return {"y": y.detach(), "grads": dict(zip(state["leaves"], grads))}


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    e, m, train = _SIZE[case["type"]], case["m"], case["train"]
    if case["op"] == "linear":
        k, n, groups = case["k"], case["n"], case["groups"]
        read = m * k + n * k + (n if case["bias"] else 0) + ((m + groups) * n if groups else 0)
        passes = 1
        if train:  # the inputs and dy in; y and a gradient for each input out
            read, passes = 2 * read + m * n, 3
        return {"bytes": e * (read + m * n), "flops": passes * 2 * m * k * n}
    d, params = case["d"], 2 * case["groups"] * case["d"] * _SIZE[case["wtype"]]
    if train:
        return {"bytes": 4 * e * m * d + 2 * params, "flops": 20 * m * d}
    return {"bytes": 2 * e * m * d + params, "flops": 8 * m * d}


# ------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """From the definitions, in 64 bits; the gradients by the product rule on per-row group indexes."""
    s = prepare(case, seed)
    wide = {nm: (s[nm].detach().double() if torch.is_tensor(s[nm]) else None)
            for nm in ("x", "weight", "bias", "residual", "gate", "dy") if nm in s}
    rows = torch.arange(case["m"], device="cuda")
    group = rows // (case["m"] // max(1, case["groups"]))

    def by_group(v):
        out = torch.zeros((max(1, case["groups"]), v.shape[1]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, group, v)

    grads = {}
    x, dy = wide["x"], wide["dy"]
    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", x, wide["weight"])
        if wide["bias"] is not None:
            z += wide["bias"]
        kind = case["act"]
        if kind == "none":
            h, slope = z, None
        elif kind == "relu":
            h, slope = z.clamp(min=0), torch.where(z > 0, 1.0, 0.0).double()
        elif kind == "silu":
            p = torch.sigmoid(z)
            h, slope = z * p, p + z * p * (1 - p)
        elif kind == "gelu":
            phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
            h, slope = z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:
            b = math.sqrt(2 / math.pi)
            p = torch.sigmoid(2 * b * (z + 0.044715 * z ** 3))  # (1 + tanh(u)) / 2
            h, slope = z * p, p + z * p * (1 - p) * 2 * b * (1 + 3 * 0.044715 * z ** 2)
        y = h if not case["groups"] else wide["residual"] + wide["gate"][group] * h
        if case["train"]:
            dz = dy * wide["gate"][group] if case["groups"] else dy
            if slope is not None:
                dz = dz * slope
            grads = {"x": torch.einsum("mn,nk->mk", dz, wide["weight"]),
                     "weight": torch.einsum("mn,mk->nk", dz, x)}
            if wide["bias"] is not None:
                grads["bias"] = dz.sum(0)
            if case["groups"]:
                grads["residual"], grads["gate"] = dy, by_group(dy * h)
    else:
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        xh = (x - mean) / torch.sqrt(var + _EPS)
        y, u = xh, dy
        if case["groups"]:
            w = wide["weight"].view(case["groups"], -1)[group]
            y = xh * w + wide["bias"].view(case["groups"], -1)[group]
            u = dy * w if case["train"] else None
        if case["train"]:
            d = case["d"]
            inner = d * u - u.sum(1, keepdim=True) - xh * (u * xh).sum(1, keepdim=True)
            grads = {"x": inner / (d * torch.sqrt(var + _EPS))}
            if case["groups"]:
                shape = wide["weight"].shape
                grads["weight"], grads["bias"] = by_group(dy * xh).view(shape), by_group(dy).view(shape)
    return {"y": y, "grads": grads} if case["train"] else y
