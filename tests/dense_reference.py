"""float64 definitions of the dense linear layer and of layer norm with their gradients, and bounds on how far a float32
computation with one rounding to the output's type may be from them, element by element.

U is half a step of float32. A sum of n float32 terms is off by at most n U times the sum of their magnitudes; the tensor
core may truncate where it aligns, a whole step, so its sums get 2 U. A rounding to type t is off by half a step,
finfo(t).eps / 2 of the value (or half of t's smallest subnormal)."""

import math

import torch

U = 2.0 ** -24
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
CURVE = {"none": 0.0, "relu": 0.0, "silu": 0.5, "gelu": 0.8, "gelu_tanh": 0.9}  # most of |act''|
STEEP = 1.13                                                                     # most of |act'|


def half_step(v, dtype):
    f = torch.finfo(dtype)
    return v.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def act(z, kind):
    """(act, act') in float64."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if kind == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    b = math.sqrt(2 / math.pi)
    p = torch.sigmoid(2 * b * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * 2 * b * (1 + 3 * 0.044715 * z ** 2)


def linear_reference(x, w, bias, kind, residual, gate, rpg, dy=None):
    """{"y": (value, bound), and with dy the gradient of each operand: (value, bound)} for 2-D x [m, k]; gate [G, n]."""
    t = x.dtype
    x, w, bias, residual, gate, dy = (None if v is None else v.detach().double() for v in (x, w, bias, residual, gate, dy))
    m, k = x.shape
    n = w.shape[0]
    z = x @ w.t()
    ez = 2 * U * k * (x.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias
        ez = ez + U * z.abs() * 2
    h, slope = act(z, kind)
    eh = STEEP * ez + 8e-6 * h.abs() + 2e-7 * z.abs()  # the float32 exp, erf and division, and 1 + erf's cancellation
    rows = torch.arange(m, device=x.device) // max(1, rpg)
    g = gate[rows] if gate is not None else torch.ones_like(h)
    y, ey = g * h, g.abs() * eh + 2 * U * (g * h).abs()
    if residual is not None:
        ey = ey + 2 * U * (residual.abs() + y.abs())
        y = y + residual
    out = {"y": (y, ey + half_step(y, t) * (1 + 1e-3))}
    if dy is None:
        return out
    # z as it is kept: f16 (its overflow is clamped where the slope is constant), else f32 / the type itself
    kept = ez + half_step(z, torch.float16)
    eslope = CURVE[kind] * kept + 8e-6
    if kind == "relu":
        eslope = (z.abs() <= kept).double()
    if kind == "none":
        eslope = torch.zeros_like(z)
    dh = dy * g
    dz = dh * slope
    edz = dh.abs() * eslope + 4 * U * dz.abs()
    edz16 = edz + half_step(dz, t) * (1 + 1e-3)
    dx = dz @ w
    out["x"] = (dx, edz16 @ w.abs() + 2 * U * n * (dz.abs() @ w.abs()) + half_step(dx, t) * (1 + 1e-3))
    dw = dz.t() @ x
    out["weight"] = (dw, edz16.t() @ x.abs() + 2 * U * m * (dz.abs().t() @ x.abs()) + half_step(dw, t) * (1 + 1e-3))
    if bias is not None:
        db = dz.sum(0)
        out["bias"] = (db, edz.sum(0) + U * m * dz.abs().sum(0) + half_step(db, t) * (1 + 1e-3))
    if residual is not None:
        out["residual"] = (dy, torch.zeros_like(dy))
    if gate is not None:
        eh_kept = eh + (half_step(z, t) if kind == "none" else 0)
        dg = torch.zeros_like(gate).index_add_(0, rows, dy * h)
        e = torch.zeros_like(gate).index_add_(0, rows, dy.abs() * eh_kept + U * m * (dy * h).abs())
        out["gate"] = (dg, e + half_step(dg, t) * (1 + 1e-3))
    return out


def norm_reference(x, w, b, eps, rpg, dy=None):
    """{"y", and with dy "x", "weight", "bias"}: (value, bound); x [m, d], w and b [G, d] or None."""
    t, wt = x.dtype, (w if w is not None else b if b is not None else x).dtype
    x, w, b, dy = (None if v is None else v.detach().double() for v in (x, w, b, dy))
    m, d = x.shape
    terms = 80  # roundings that a value goes through in a row's sum: its thread's serial sum, then two trees
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    emean = terms * U * x.abs().mean(1, keepdim=True)
    # relative error of rstd: half the variance's, the mean's error squared (its first order cancels), two steps of rsqrt
    rel = 0.5 * terms * U + 0.5 * emean ** 2 * rstd ** 2 + 4 * U + emean * rstd * 4 * U
    xh = c * rstd
    exh = rstd * (emean + 2 * U * c.abs()) + xh.abs() * (rel + 2 * U)
    rows = torch.arange(m, device=x.device) // max(1, rpg)
    wr = w[rows] if w is not None else torch.ones_like(x)
    y = xh * wr
    ey = wr.abs() * exh + 3 * U * y.abs()
    if b is not None:
        y = y + b[rows]
        ey = ey + 2 * U * (y.abs() + b[rows].abs())
    out = {"y": (y, ey * (1 + 1e-3) + half_step(y, t) * (1 + 1e-3))}
    if dy is None:
        return out
    v = dy * wr
    m0, m1 = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    em0 = terms * U * v.abs().mean(1, keepdim=True)
    em1 = (v.abs() * exh).mean(1, keepdim=True) + terms * U * (v * xh).abs().mean(1, keepdim=True)
    dx = rstd * (v - m0 - xh * m1)
    edx = rstd * (4 * U * (v.abs() + m0.abs() + (xh * m1).abs()) + em0 + xh.abs() * em1 + exh * m1.abs()) + dx.abs() * rel
    out["x"] = (dx, edx * (1 + 1e-3) + half_step(dx, t) * (1 + 1e-3))
    for name, p, term, e in (("weight", w, dy * xh, dy.abs() * exh), ("bias", b, dy, torch.zeros_like(dy))):
        if p is not None:
            s = torch.zeros_like(p).index_add_(0, rows, term)
            es = torch.zeros_like(p).index_add_(0, rows, e + U * (m + 8) * term.abs())
            out[name] = (s, es * (1 + 1e-3) + half_step(s, wt) * (1 + 1e-3))
    return out


def assert_within(got, want, what):
    """got within want's bound of want's value, element by element."""
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), f"{what}: {tuple(got.shape)} for {tuple(value.shape)}"
    off = (got.double() - value).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad, off / bound.clamp(min=1e-300), torch.zeros_like(off)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values too far off; worst at {i}: "
                             f"{got.reshape(-1)[i]} for {value.reshape(-1)[i]}, bound {bound.reshape(-1)[i]}")
