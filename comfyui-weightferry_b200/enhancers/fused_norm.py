"""Layer norm with its backward pass on the sm_100a kernels of csrc/layer_norm.cu:

    y = (x - mean) / sqrt(var + eps) * weight[row // rows_per_group] + bias[row // rows_per_group]

One row of weight and bias for all rows is the affine layer norm; a row for each group of rows is the adaLN norm of the
Cosmos blocks (weight = 1 + scale, bias = shift, a row for each (batch, frame)). ``layer_norm`` is differentiable in x,
weight and bias (csrc/torch_ops.cpp), for any width, in bfloat16, float16 and float32; the statistics and all sums are
float32, with one rounding to the output (``fused_block.ln_modulate`` keeps the reference's rounding steps instead and is
for inference). It launches on the current stream and allocates with PyTorch's allocator."""

from .. import _ext


def layer_norm(x, weight=None, bias=None, eps=1e-6, rows_per_group=None):
    """Layer norm over the last dimension of x [..., d] (bfloat16, float16 or float32, on a CUDA device, any strides).

    weight and bias: None, [d], or [groups, d] whose row g holds for rows g * rows_per_group .. of x (rows_per_group: all
    rows divided evenly where it is not given; the last group may be short); of x's type or float32, both alike. Returns a
    new contiguous tensor of x's shape and type. Differentiable once in x, weight and bias, in reverse mode; tangents and traces
    raise NotImplementedError."""
    return (_ext._ops or _ext.ops()).layer_norm(x, weight, bias, eps, rows_per_group)
