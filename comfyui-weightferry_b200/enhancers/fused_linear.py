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


def _p(t):
    return 0 if t is None else t.data_ptr()


def _operand(t):
    """(tensor, row pitch) of a 2-D operand as the tensor cores' loads need it: values of a row side by side, rows a
    multiple of 8 values apart, 16-byte aligned. A tensor that is not so laid out is copied (odd widths, slices)."""
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    ld = t.stride(0) if rows > 1 else -(-cols // 8) * 8
    if t.data_ptr() % 16 == 0 and ld % 8 == 0 and ld >= cols and (cols == 1 or t.stride(1) == 1):
        return t, ld
    if rows > 1 and t.stride(0) < cols:  # expanded rows
        t = t.contiguous()
    ld = -(-cols // 8) * 8
    out = torch.empty((rows, ld), dtype=t.dtype, device=t.device)
    rc = _ext.lib().wf_copy_rows16(t.data_ptr(), t.stride(0) if rows > 1 else cols, out.data_ptr(), ld, rows, cols,
                                   _ext.stream_of(t.device))
    _ext.check(rc, "wf_copy_rows16")
    return out[:, :cols], ld


def _rows(t):
    """(tensor, row pitch) of a 2-D buffer whose rows are read value by value: neighbours side by side, any pitch."""
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, (t.stride(0) if rows > 1 else cols)


def _check(x, weight, bias, activation, residual, gate, rows_per_group):
    """(m, n, k, groups, rows per group) of a call, or the reason it is refused."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"linear: x is {x.dtype}; bfloat16 or float16 is needed")
    operands = [(nm, t) for nm, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual), ("gate", gate))
                if t is not None]
    for name, t in operands:
        if t.dtype != x.dtype:
            raise TypeError(f"linear: {name} is {t.dtype}, x is {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    n, k = weight.shape
    if k < 1:
        raise ValueError("linear: a layer without inputs")
    m = x.numel() // k
    groups = 1
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"linear: bias {tuple(bias.shape)} for {n} outputs")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], n):
        raise ValueError(f"linear: residual {tuple(residual.shape)} for an output {(*x.shape[:-1], n)}")
    if gate is None:
        if rows_per_group is not None:
            raise ValueError("linear: rows_per_group without a gate")
        rows_per_group = max(1, m)
    else:
        if gate.dim() not in (1, 2) or gate.shape[-1] != n or (gate.dim() == 2 and gate.shape[0] == 0):
            raise ValueError(f"linear: gate {tuple(gate.shape)} for {n} outputs")
        groups = 1 if gate.dim() == 1 else gate.shape[0]
        if rows_per_group is None:
            if m % groups:
                raise ValueError(f"linear: {groups} gate rows do not divide {m} rows; give rows_per_group")
            rows_per_group = max(1, m // groups)
        elif rows_per_group < 1 or (m and groups != -(-m // rows_per_group)):
            raise ValueError(f"linear: {groups} gate rows for {m} rows in groups of {rows_per_group}")
    for name, t in operands:
        if not t.is_cuda or t.device != x.device:
            raise ValueError(f"linear: {name} is on {t.device}, x on {x.device}; one CUDA device is needed")
    return m, n, k, groups, rows_per_group


def _forward(x2, w, bias, act, r2, gate, rpg, m, n, k, z=None):
    """(y [m, n], x's operand, weight's operand); z: a [m, n] tensor for the pre-activation, or None."""
    y = torch.empty((m, n), dtype=x2.dtype, device=x2.device)
    if m == 0 or n == 0:
        return y, x2, w
    xo, ldx = _operand(x2)
    wo, ldw = _operand(w)
    if bias is not None:
        bias = bias.contiguous()
    if gate is not None:
        gate = gate.contiguous()
    ldr = 0
    if r2 is not None:
        r2, ldr = _rows(r2)
    rc = _ext.lib().wf_linear(xo.data_ptr(), ldx, wo.data_ptr(), ldw, _p(bias), act, _p(gate), rpg, _p(r2), ldr,
                              y.data_ptr(), n, _p(z), z.stride(0) if z is not None else 0,
                              _ext.dtype_code(z.dtype) if z is not None else 0, m, n, k, _ext.dtype_code(x2.dtype),
                              _ext.stream_of(x2.device))
    _ext.check(rc, "wf_linear")
    return y, xo, wo


def _kept_dtype(act, need_z, need_gate, dtype):
    """How the forward pass keeps z for the backward pass, or None. The activation's slope is constant where f16 ends,
    so f16 (clamped, 11 bits) keeps it more exactly than bf16 would; the gate's gradient reads activation(z) itself:
    exactly (f32), or as the layer rounds it where there is no activation."""
    if need_gate:
        return torch.float32 if act else dtype
    return torch.float16 if act and need_z else None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, gate, act, rpg, m, n, k, groups):
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        kept = _kept_dtype(act, need_x or need_w or need_b, need_g, x.dtype)
        with _ext.on_device(x.device):
            z = None
            if kept is not None:
                z = torch.empty((m, -(-n // 8) * 8), dtype=kept, device=x.device)
            y, xo, wo = _forward(x.reshape(m, k), weight, bias, act, None if residual is None else residual.reshape(m, n),
                                 gate, rpg, m, n, k, z)
        ctx.save_for_backward(xo if need_w else None, wo if need_x else None,
                              gate if need_x or need_w or need_b else None, z)
        ctx.sizes = (act, rpg, m, n, k, groups)
        ctx.shapes = (x.shape, x.dtype, x.device, None if gate is None else gate.shape)
        return y.view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xo, wo, gate, z = ctx.saved_tensors
        act, rpg, m, n, k, groups = ctx.sizes
        x_shape, dtype, device, gate_shape = ctx.shapes
        need_x, need_w, need_b, need_r, need_g = ctx.needs_input_grad[:5]
        dx = dw = db = dg = None
        if m == 0 or n == 0:
            zeros = dict(dtype=dtype, device=device)
            return (torch.zeros(x_shape, **zeros) if need_x else None, torch.zeros((n, k), **zeros) if need_w else None,
                    torch.zeros((n,), **zeros) if need_b else None, dy if need_r else None,
                    torch.zeros(gate_shape, **zeros) if need_g else None, None, None, None, None, None, None)
        lib, code, stream = _ext.lib(), _ext.dtype_code(dtype), _ext.stream_of(device)
        with _ext.on_device(device):
            dy2, lddy = _rows(dy.reshape(m, n))
            dz, lddz = None, 0
            if need_x or need_w:
                if act == 0 and gate is None:
                    if dy2.data_ptr() % 16 == 0 and lddy % 8 == 0:
                        dz, lddz = dy2, lddy
                make = dz is None
                if make:
                    lddz = -(-n // 8) * 8
                    dz = torch.empty((m, lddz), dtype=dtype, device=device)
            else:
                make = False
            if make or need_b or need_g:
                if need_b:
                    db = torch.empty((n,), dtype=dtype, device=device)
                if need_g:
                    dg = torch.empty((groups, n), dtype=dtype, device=device)
                size = lib.wf_linear_backward_act_workspace(m, n, rpg) if need_b or need_g else 0
                work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
                gc = None if gate is None else gate.contiguous()
                rc = lib.wf_linear_backward_act(
                    dy2.data_ptr(), lddy, _p(z), z.stride(0) if z is not None else 0,
                    _ext.dtype_code(z.dtype) if z is not None else 0, act, _p(gc), rpg, _p(dz) if make else 0, lddz,
                    _p(db), _p(dg), m, n, code, _p(work), size, stream)
                _ext.check(rc, "wf_linear_backward_act")
            if need_x:
                dx = torch.empty((m, k), dtype=dtype, device=device)
                rc = lib.wf_linear_backward_input(dz.data_ptr(), lddz, wo.data_ptr(), wo.stride(0) if n > 1 else -(-k // 8) * 8,
                                                  dx.data_ptr(), k, m, n, k, code, stream)
                _ext.check(rc, "wf_linear_backward_input")
                dx = dx.view(x_shape)
            if need_w:
                dw = torch.empty((n, k), dtype=dtype, device=device)
                rc = lib.wf_linear_backward_weight(dz.data_ptr(), lddz, xo.data_ptr(), xo.stride(0) if m > 1 else -(-k // 8) * 8,
                                                   dw.data_ptr(), k, m, n, k, code, stream)
                _ext.check(rc, "wf_linear_backward_weight")
        if dg is not None:
            dg = dg.view(gate_shape)
        return dx, dw, db, dy if need_r else None, dg, None, None, None, None, None, None


def linear(x, weight, bias=None, activation="none", residual=None, gate=None, rows_per_group=None):
    """residual + gate * activation(x @ weight^T + bias), each of bias, residual and gate optional.

    x [..., k], weight [n, k], bias [n], residual [..., n] (the output's shape), gate [n], or [groups, n] whose row g
    holds for rows g * rows_per_group .. of x (rows_per_group: all rows divided evenly where it is not given; the last
    group may be short). All of one type, bfloat16 or float16, on one CUDA device; any strides (rows whose pitch is a
    multiple of 8 values are read in place, others are copied first). activation: a name of ``ACTIVATIONS``. Returns a
    new contiguous [..., n]. Differentiable once in every tensor."""
    m, n, k, groups, rpg = _check(x, weight, bias, activation, residual, gate, rows_per_group)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual, gate)):
        return _Linear.apply(x, weight, bias, residual, gate, act, rpg, m, n, k, groups)
    with _ext.on_device(x.device):
        y, _, _ = _forward(x.reshape(m, k), weight, bias, act, None if residual is None else residual.reshape(m, n), gate,
                           rpg, m, n, k)
    return y.view(*x.shape[:-1], n)


def status():
    """0, or the code of a pipeline wait of the linear kernels that ran out of time (their output is then incomplete);
    synchronises and clears it."""
    import ctypes
    v = ctypes.c_int()
    _ext.check(_ext.lib().wf_linear_status(ctypes.byref(v)), "wf_linear_status")
    return v.value
