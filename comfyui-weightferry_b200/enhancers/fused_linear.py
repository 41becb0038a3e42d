"""The dense linear layer of bf16 / f16 weights (what the GGUF dequantisation produces) with its epilogue, and its
backward pass -- the counterpart of ``fused_int8.gemm_residual`` for layers that are not int8:

    y = residual + gate[row // rows_per_group] * activation(x @ weight^T + bias)

in one launch on tcgen05 tensor cores (csrc/linear.cu), float32 inside and one rounding to the output. ``linear`` is
differentiable in every tensor argument (csrc/torch_ops.cpp); it launches on the current stream and allocates with
PyTorch's allocator, so it can be captured into a CUDA graph (forward, and backward through ``torch.autograd.grad``). The
reference leaves these layers to PyTorch, whose linear, GELU and addcmul kernels round to 16 bits in between."""

import ctypes

from .. import _ext

ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")  # gelu: the erf form


def linear(x, weight, bias=None, activation="none", residual=None, gate=None, rows_per_group=None):
    """residual + gate * activation(x @ weight^T + bias), each of bias, residual and gate optional.

    x [..., k], weight [n, k], bias [n], residual [..., n] (the output's shape), gate [n], or [groups, n] whose row g
    holds for rows g * rows_per_group .. of x (rows_per_group: all rows divided evenly where it is not given; the last
    group may be short). All of one type, bfloat16 or float16, on one CUDA device; any strides (rows whose pitch is a
    multiple of 8 values are read in place, others are copied first). activation: a name of ``ACTIVATIONS``. Returns a
    new contiguous [..., n]. Differentiable once in every tensor, in reverse mode; tangents and traces raise NotImplementedError."""
    return (_ext._ops or _ext.ops()).linear(x, weight, bias, activation, residual, gate, rows_per_group)


def status():
    """0, or the code of a pipeline wait of the linear kernels that ran out of time: what they could not compute is NaN, and
    further calls on the device raise RuntimeError until this has been read. Synchronises and clears it."""
    v = ctypes.c_int()
    _ext.check(_ext.lib().wf_linear_status(ctypes.byref(v)), "wf_linear_status")
    return v.value
