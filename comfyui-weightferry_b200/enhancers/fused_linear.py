"""The dense linear layer of bf16 / f16 weights (what the GGUF dequantisation produces) with its epilogue, and its
backward pass -- the counterpart of ``fused_int8.gemm_residual`` for layers that are not int8:

    y = residual + gate[row // rows_per_group] * activation(x @ weight^T + bias)

in one launch on tcgen05 tensor cores (csrc/linear.cu), float32 inside and one rounding to the output. ``linear`` is
differentiable in every tensor argument; it launches on the current stream and allocates with PyTorch's allocator, so
it can be captured into a CUDA graph (forward, and backward through ``torch.autograd.grad``). The reference leaves these
layers to PyTorch, whose linear, GELU and addcmul kernels round to 16 bits in between."""

import torch

from .. import _ext

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # gelu: the erf form
_CODES = {torch.float16: _ext.WF_F16, torch.bfloat16: _ext.WF_BF16, torch.float32: _ext.WF_F32}
_TYPES = (torch.bfloat16, torch.float16)


def _operand(t):
    """(tensor, row pitch) of a 2-D operand as the tensor cores' loads need it: values of a row side by side, rows a
    multiple of 8 values apart, 16-byte aligned. A tensor that is not so laid out is copied (odd widths, slices)."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if rows == 1:
        s0 = -(-cols // 8) * 8
    if (s1 == 1 or cols == 1) and s0 % 8 == 0 and s0 >= cols and t.data_ptr() % 16 == 0:
        return t, s0
    t, s0 = _rows(t)
    ld = -(-cols // 8) * 8
    out = torch.empty((rows, ld), dtype=t.dtype, device=t.device)
    with _ext.on_device(t.device):
        rc = _ext.lib().wf_copy_rows16(t.data_ptr(), s0, out.data_ptr(), ld, rows, cols, _ext.stream_of(t.device))
    _ext.check(rc, "wf_copy_rows16")
    return out[:, :cols], ld


def _rows(t):
    """(tensor, row pitch) of a 2-D buffer whose rows are read value by value: neighbours side by side, any pitch."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if rows == 1:
        s0 = cols
    if (s1 != 1 and cols > 1) or s0 < cols:
        return t.contiguous(), cols
    return t, s0


def _group_rows(what, p, m, rows_per_group):
    """Rows of x to each row of p ([n], or [groups, n]): as given, or all m rows divided evenly."""
    groups = 1 if p.dim() == 1 else p.shape[0]
    if rows_per_group is None:
        if m % groups:
            raise ValueError(f"{what}: {groups} rows do not divide {m} rows; give rows_per_group")
        return max(1, m // groups)
    if rows_per_group < 1 or (m and groups != -(-m // rows_per_group)):
        raise ValueError(f"{what}: {groups} rows for {m} rows in groups of {rows_per_group}")
    return rows_per_group


def _check(x, weight, bias, activation, residual, gate, rows_per_group):
    """(m, n, k, rows per group) of a call; raises for one that is refused."""
    dtype = x.dtype
    if dtype not in _TYPES:
        raise TypeError(f"linear: x is {dtype}; bfloat16 or float16 is needed")
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    rest = [(nm, t) for nm, t in (("weight", weight), ("bias", bias), ("residual", residual), ("gate", gate)) if t is not None]
    for nm, t in rest:
        if t.dtype != dtype:
            raise TypeError(f"linear: {nm} is {t.dtype}, x is {dtype}")
    shape, w_shape = x.shape, weight.shape
    if len(shape) < 1 or len(w_shape) != 2 or shape[-1] != w_shape[1]:
        raise ValueError(f"linear: x {tuple(shape)} and weight {tuple(w_shape)} do not match")
    n, k = w_shape
    if k < 1:
        raise ValueError("linear: a layer without inputs")
    m = x.numel() // k
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"linear: bias {tuple(bias.shape)} for {n} outputs")
    if residual is not None and residual.shape != (*shape[:-1], n):
        raise ValueError(f"linear: residual {tuple(residual.shape)} for an output {(*shape[:-1], n)}")
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != n or (gate.dim() == 2 and gate.shape[0] == 0):
            raise ValueError(f"linear: gate {tuple(gate.shape)} for {n} outputs")
        rows_per_group = _group_rows("linear: gate", gate, m, rows_per_group)
    elif rows_per_group is not None:
        raise ValueError("linear: rows_per_group without a gate")
    index = x.get_device()
    for nm, t in rest:
        if t.get_device() != index:
            raise ValueError(f"linear: {nm} is on {t.device}, x on {x.device}")
    if index < 0:
        raise ValueError(f"linear: x is on {x.device}; a CUDA device is needed")
    return m, n, k, rows_per_group or max(1, m)


def _forward(x, weight, bias, act, residual, gate, rpg, m, n, k, kept=None):
    """(y, x's operand, weight's operand, the pre-activation as type `kept` or None)"""
    lead = x.shape[:-1]
    y = x.new_empty((*lead, n))
    if m == 0 or n == 0:
        return y, None, None, None
    xo, ldx = _operand(x if len(lead) == 1 else x.reshape(m, k))
    wo, ldw = _operand(weight)
    p_bias = p_gate = p_res = p_z = ldr = ldz = 0
    z = None
    if bias is not None:
        bias = bias.contiguous()
        p_bias = bias.data_ptr()
    if gate is not None:
        gate = gate.contiguous()
        p_gate = gate.data_ptr()
    if residual is not None:
        residual, ldr = _rows(residual if len(lead) == 1 else residual.reshape(m, n))
        p_res = residual.data_ptr()
    if kept is not None:
        ldz = -(-n // 8) * 8
        z = torch.empty((m, ldz), dtype=kept, device=x.device)
        p_z = z.data_ptr()
    _ext.launch("wf_linear", _ext.LINEAR_ARGS.pack(
        xo.data_ptr(), wo.data_ptr(), p_bias, p_gate, p_res, y.data_ptr(), p_z, ldx, ldw, ldr, n, ldz, rpg, m, n, k, act,
        _CODES[x.dtype], _CODES[kept] if kept is not None else 0, 0), x.get_device())
    return y, xo, wo, z


def _kept_dtype(act, need_z, need_gate, dtype):
    """How the forward pass keeps z for the backward pass, or None. The activation's slope is constant where f16 ends,
    so f16 (clamped, 11 bits) keeps it more exactly than bf16 would; the gate's gradient reads activation(z) itself:
    exactly (f32), or as the layer rounds it where there is no activation."""
    if need_gate:
        return torch.float32 if act else dtype
    return torch.float16 if act and need_z else None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, act, rpg, m, n, k):
        need_x, need_w, need_b, _need_r, need_g = ctx.needs_input_grad[:5]
        need_z = need_x or need_w or need_b
        y, xo, wo, z = _forward(x, weight, bias, act, residual, gate, rpg, m, n, k,
                                _kept_dtype(act, need_z, need_g, x.dtype))
        ctx.save_for_backward(xo if need_w else None, wo if need_x else None, gate if need_z else None, z)
        ctx.call = (act, rpg, m, n, k, x.shape, x.dtype, x.device, None if gate is None else gate.shape)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xo, wo, gate, z = ctx.saved_tensors
        act, rpg, m, n, k, x_shape, dtype, device, gate_shape = ctx.call
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        new = torch.empty if m and n else torch.zeros
        dx = new(x_shape, dtype=dtype, device=device) if need_x else None
        dw = new((n, k), dtype=dtype, device=device) if need_w else None
        db = new((n,), dtype=dtype, device=device) if need_b else None
        dg = new(gate_shape, dtype=dtype, device=device) if need_g else None
        if m and n and (need_x or need_w or need_b or need_g):
            dy2, lddy = _rows(dy if dy.dim() == 2 else dy.reshape(m, n))
            size = _ext.lib().wf_linear_backward_workspace(m, n, rpg)
            work = torch.empty(size, dtype=torch.uint8, device=device)
            if gate is not None:
                gate = gate.contiguous()

            def at(t):
                return 0 if t is None else t.data_ptr()

            def pitch(t):  # of an operand of a product, as _operand has it
                return 0 if t is None else t.stride(0) if t.shape[0] > 1 else -(-k // 8) * 8
            _ext.launch("wf_linear_backward", _ext.LINEAR_GRAD_ARGS.pack(
                dy2.data_ptr(), at(xo), at(wo), at(z), at(gate), at(dx), at(dw), at(db), at(dg), work.data_ptr(), lddy,
                pitch(xo), pitch(wo), 0 if z is None else z.stride(0), k, k, rpg, size, m, n, k, act, _CODES[dtype],
                0 if z is None else _CODES[z.dtype], 0), device.index)
        return dx, dw, db, dy if need_r else None, dg, None, None, None, None, None


def linear(x, weight, bias=None, activation="none", residual=None, gate=None, rows_per_group=None):
    """residual + gate * activation(x @ weight^T + bias), each of bias, residual and gate optional.

    x [..., k], weight [n, k], bias [n], residual [..., n] (the output's shape), gate [n], or [groups, n] whose row g
    holds for rows g * rows_per_group .. of x (rows_per_group: all rows divided evenly where it is not given; the last
    group may be short). All of one type, bfloat16 or float16, on one CUDA device; any strides (rows whose pitch is a
    multiple of 8 values are read in place, others are copied first). activation: a name of ``ACTIVATIONS``. Returns a
    new contiguous [..., n]. Differentiable once in every tensor."""
    m, n, k, rpg = _check(x, weight, bias, activation, residual, gate, rows_per_group)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or any(
            t is not None and t.requires_grad for t in (bias, residual, gate))):
        return _Linear.apply(x, weight, bias, residual, gate, act, rpg, m, n, k)
    return _forward(x, weight, bias, act, residual, gate, rpg, m, n, k)[0]


def status():
    """0, or the code of a pipeline wait of the linear kernels that ran out of time (their output is then incomplete);
    synchronises and clears it."""
    import ctypes
    v = ctypes.c_int()
    _ext.check(_ext.lib().wf_linear_status(ctypes.byref(v)), "wf_linear_status")
    return v.value
