"""Layer norm with its backward pass on the sm_100a kernels of csrc/layer_norm.cu:

    y = (x - mean) / sqrt(var + eps) * weight[row // rows_per_group] + bias[row // rows_per_group]

One row of weight and bias for all rows is the affine layer norm; a row for each group of rows is the adaLN norm of the
Cosmos blocks (weight = 1 + scale, bias = shift, a row for each (batch, frame)). ``layer_norm`` is differentiable in x,
weight and bias, for any width, in bfloat16, float16 and float32; the statistics and all sums are float32, with one
rounding to the output (``fused_block.ln_modulate`` keeps the reference's rounding steps instead and is for inference).
It launches on the current stream and allocates with PyTorch's allocator."""

import torch

from .. import _ext
from .fused_linear import _CODES, _group_rows, _rows

_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(x, weight, bias, eps, rows_per_group):
    """(rows, width, rows per group) of a call; raises for one that is refused."""
    dtype, shape = x.dtype, x.shape
    if dtype not in _TYPES:
        raise TypeError(f"layer_norm: x is {dtype}; bfloat16, float16 or float32 is needed")
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"layer_norm: x {tuple(shape)} has no values to normalise")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps {eps}")
    d = shape[-1]
    m = x.numel() // d
    index = x.get_device()
    p = weight if weight is not None else bias
    if p is not None:
        for nm, t in (("weight", weight), ("bias", bias)):
            if t is None:
                continue
            if (t.dtype != dtype and t.dtype != torch.float32) or t.dtype != p.dtype:
                raise TypeError(f"layer_norm: {nm} is {t.dtype}; {dtype} or float32 is needed, weight and bias alike")
            if t.dim() not in (1, 2) or t.shape[-1] != d or t.shape != p.shape or t.shape[0] == 0:
                raise ValueError(f"layer_norm: {nm} {tuple(t.shape)} for rows of {d}")
            if t.get_device() != index:
                raise ValueError(f"layer_norm: {nm} is on {t.device}, x on {x.device}")
        rows_per_group = _group_rows("layer_norm: weight", p, m, rows_per_group)
    elif rows_per_group is not None:
        raise ValueError("layer_norm: rows_per_group without weight or bias")
    if index < 0:
        raise ValueError(f"layer_norm: x is on {x.device}; a CUDA device is needed")
    return m, d, rows_per_group or max(1, m)


def _forward(x, weight, bias, eps, rpg, m, d, keep):
    """(y, x's rows, their pitch, the statistics [2, m] or None)"""
    y = x.new_empty(x.shape)
    if m == 0:
        return y, None, d, None
    x2, ldx = _rows(x if x.dim() == 2 else x.reshape(m, d))
    p_w = p_b = p_mean = 0
    code = w_code = _CODES[x.dtype]
    stats = None
    if bias is not None:
        bias = bias.contiguous()
        p_b, w_code = bias.data_ptr(), _CODES[bias.dtype]
    if weight is not None:
        weight = weight.contiguous()
        p_w, w_code = weight.data_ptr(), _CODES[weight.dtype]
    if keep:
        stats = torch.empty((2, m), dtype=torch.float32, device=x.device)
        p_mean = stats.data_ptr()
    _ext.launch("wf_layer_norm", _ext.LAYER_NORM_ARGS.pack(
        x2.data_ptr(), p_w, p_b, y.data_ptr(), p_mean, p_mean + 4 * m if keep else 0, ldx, d, m, d, rpg, eps, code, w_code,
        0), x.get_device())
    return y, x2, ldx, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rpg, m, d):
        y, x2, ldx, stats = _forward(x, weight, bias, eps, rpg, m, d, True)
        ctx.save_for_backward(x2, weight, stats)
        p = weight if weight is not None else bias
        ctx.call = (rpg, m, d, ldx, x.shape, x.dtype, x.device, None if p is None else p.shape,
                    x.dtype if p is None else p.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, stats = ctx.saved_tensors
        rpg, m, d, ldx, shape, dtype, device, p_shape, p_dtype = ctx.call
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        new = torch.empty if m else torch.zeros
        dx = new(shape, dtype=dtype, device=device) if need_x else None
        dw = new(p_shape, dtype=p_dtype, device=device) if need_w else None
        db = new(p_shape, dtype=p_dtype, device=device) if need_b else None
        if m:
            dy2, lddy = _rows(dy if dy.dim() == 2 else dy.reshape(m, d))
            size, work = 0, None
            if need_w or need_b:
                size = _ext.lib().wf_layer_norm_backward_workspace(m, d, rpg, _CODES[dtype])
                work = torch.empty(size, dtype=torch.uint8, device=device)
            if weight is not None:
                weight = weight.contiguous()

            def at(t):
                return 0 if t is None else t.data_ptr()
            mean = stats.data_ptr()
            _ext.launch("wf_layer_norm_backward", _ext.LAYER_NORM_GRAD_ARGS.pack(
                dy2.data_ptr(), x2.data_ptr(), at(weight), mean, mean + 4 * m, at(dx), at(dw), at(db), at(work), lddy, ldx,
                d, m, d, rpg, size, _CODES[dtype], _CODES[p_dtype]), device.index)
        return dx, dw, db, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-6, rows_per_group=None):
    """Layer norm over the last dimension of x [..., d] (bfloat16, float16 or float32, on a CUDA device, any strides).

    weight and bias: None, [d], or [groups, d] whose row g holds for rows g * rows_per_group .. of x (rows_per_group: all
    rows divided evenly where it is not given; the last group may be short); of x's type or float32, both alike. Returns a
    new contiguous tensor of x's shape and type. Differentiable once in x, weight and bias."""
    m, d, rpg = _check(x, weight, bias, eps, rows_per_group)
    if torch.is_grad_enabled() and (x.requires_grad or any(t is not None and t.requires_grad for t in (weight, bias))):
        return _LayerNorm.apply(x, weight, bias, eps, rpg, m, d)
    return _forward(x, weight, bias, eps, rpg, m, d, False)[0]
