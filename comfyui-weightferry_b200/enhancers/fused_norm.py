"""Layer norm with its backward pass on the sm_100a kernels of csrc/layer_norm.cu:

    y = (x - mean) / sqrt(var + eps) * weight[row // rows_per_group] + bias[row // rows_per_group]

One row of weight and bias for all rows is the affine layer norm; a row for each group of rows is the adaLN norm of the
Cosmos blocks (weight = 1 + scale, bias = shift, a row for each (batch, frame)). ``layer_norm`` is differentiable in x,
weight and bias, for any width, in bfloat16, float16 and float32; the statistics and all sums are float32, with one
rounding to the output (``fused_block.ln_modulate`` keeps the reference's rounding steps instead and is for inference).
It launches on the current stream and allocates with PyTorch's allocator."""

import torch

from .. import _ext


def _p(t):
    return 0 if t is None else t.data_ptr()


def _rows(t):
    """(tensor, row pitch) of a 2-D tensor with a row's values side by side."""
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else cols)


def _check(x, weight, bias, eps, rows_per_group):
    """(rows, width, groups, rows per group) of a call, or the reason it is refused."""
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"layer_norm: x is {x.dtype}; bfloat16, float16 or float32 is needed")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x {tuple(x.shape)} has no values to normalise")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps {eps}")
    d = x.shape[-1]
    m = x.numel() // d
    p = weight if weight is not None else bias
    if p is None and rows_per_group is not None:
        raise ValueError("layer_norm: rows_per_group without weight or bias")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype not in (x.dtype, torch.float32) or t.dtype != p.dtype:
            raise TypeError(f"layer_norm: {name} is {t.dtype}; {x.dtype} or float32 is needed, weight and bias alike")
        if t.dim() not in (1, 2) or t.shape[-1] != d or t.shape != p.shape or t.numel() == 0:
            raise ValueError(f"layer_norm: {name} {tuple(t.shape)} for rows of {d}")
        if t.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {t.device}, x on {x.device}")
    groups = 1 if p is None or p.dim() == 1 else p.shape[0]
    if rows_per_group is None:
        if m % groups:
            raise ValueError(f"layer_norm: {groups} weight rows do not divide {m} rows; give rows_per_group")
        rows_per_group = max(1, m // groups)
    elif rows_per_group < 1 or (m and groups != -(-m // rows_per_group)):
        raise ValueError(f"layer_norm: {groups} weight rows for {m} rows in groups of {rows_per_group}")
    if not x.is_cuda:
        raise ValueError(f"layer_norm: x is on {x.device}; a CUDA device is needed")
    return m, d, groups, rows_per_group


def _forward(x, weight, bias, eps, rpg, m, d, keep):
    """(y like x, x's rows, mean, rstd); mean and rstd None unless they are to be kept."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x2, ldx = _rows(x.reshape(m, d))
    stats = torch.empty((2, m), dtype=torch.float32, device=x.device) if keep else None
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    p = weight if weight is not None else bias
    rc = _ext.lib().wf_layer_norm(x2.data_ptr(), ldx, _p(weight), _p(bias), _ext.dtype_code(x.dtype if p is None else p.dtype),
                                  y.data_ptr(), d, _p(stats), stats[1].data_ptr() if keep else 0, m, d, rpg, float(eps),
                                  _ext.dtype_code(x.dtype), _ext.stream_of(x.device))
    _ext.check(rc, "wf_layer_norm")
    return y, x2, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rpg, m, d):
        with _ext.on_device(x.device):
            y, x2, stats = _forward(x, weight, bias, eps, rpg, m, d, True)
        ctx.save_for_backward(x2, weight, stats)
        p = weight if weight is not None else bias
        ctx.sizes = (rpg, m, d, x.shape, None if p is None else p.shape, x.dtype if p is None else p.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, stats = ctx.saved_tensors
        rpg, m, d, shape, p_shape, p_dtype = ctx.sizes
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev = x2.device
        if m == 0:
            zeros = dict(dtype=p_dtype, device=dev)
            return (torch.zeros(shape, dtype=x2.dtype, device=dev) if need_x else None,
                    torch.zeros(p_shape, **zeros) if need_w else None, torch.zeros(p_shape, **zeros) if need_b else None,
                    None, None, None, None)
        lib = _ext.lib()
        with _ext.on_device(dev):
            dy2, lddy = _rows(dy.reshape(m, d))
            _, ldx = _rows(x2)
            dx = torch.empty(shape, dtype=x2.dtype, device=dev) if need_x else None
            dw = torch.empty(p_shape, dtype=p_dtype, device=dev) if need_w else None
            db = torch.empty(p_shape, dtype=p_dtype, device=dev) if need_b else None
            size = lib.wf_layer_norm_backward_workspace(m, d, rpg) if need_w or need_b else 0
            work = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
            w = None if weight is None else weight.contiguous()
            rc = lib.wf_layer_norm_backward(dy2.data_ptr(), lddy, x2.data_ptr(), ldx, _p(w), _ext.dtype_code(p_dtype),
                                            stats.data_ptr(), stats[1].data_ptr(), _p(dx), d, _p(dw), _p(db), m, d, rpg,
                                            _ext.dtype_code(x2.dtype), _p(work), size, _ext.stream_of(dev))
            _ext.check(rc, "wf_layer_norm_backward")
        return dx, dw, db, None, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-6, rows_per_group=None):
    """Layer norm over the last dimension of x [..., d] (bfloat16, float16 or float32, on a CUDA device, any strides).

    weight and bias: None, [d], or [groups, d] whose row g holds for rows g * rows_per_group .. of x (rows_per_group: all
    rows divided evenly where it is not given; the last group may be short); of x's type or float32, both alike. Returns a
    new contiguous tensor of x's shape and type. Differentiable once in x, weight and bias."""
    m, d, _groups, rpg = _check(x, weight, bias, eps, rows_per_group)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps, rpg, m, d)
    with _ext.on_device(x.device):
        return _forward(x, weight, bias, eps, rpg, m, d, False)[0]
