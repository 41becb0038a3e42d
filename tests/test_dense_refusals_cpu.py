"""What the dense linear layer and layer norm refuse, without a GPU: wrong shapes, types, devices and groups at the Python
entry points, and bad sizes, pitches, pointers and types at the C entry points (which check before they look at the
device)."""

import ctypes

import pytest

import dense_cabi
from conftest import wf

BF = "bfloat16"


def _t(*shape, dtype=BF):
    import torch
    return torch.zeros(shape, dtype=getattr(torch, dtype))


@pytest.mark.parametrize("kw,error", [
    (dict(x=_t(4, 16, dtype="float32"), weight=_t(8, 16, dtype="float32")), TypeError),
    (dict(x=_t(4, 16), weight=_t(8, 16, dtype="float16")), TypeError),
    (dict(x=_t(4, 16), weight=_t(8, 16), bias=_t(8, dtype="float32")), TypeError),
    (dict(x=_t(4, 16), weight=_t(8, 16), activation="tanh"), ValueError),
    (dict(x=_t(4, 15), weight=_t(8, 16)), ValueError),
    (dict(x=_t(4, 16), weight=_t(16)), ValueError),
    (dict(x=_t(4, 0), weight=_t(8, 0)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), bias=_t(1, 8)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), residual=_t(1, 8)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), gate=_t(4)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), gate=_t(3, 8)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), gate=_t(0, 8)), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), gate=_t(2, 8), rows_per_group=4), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), gate=_t(2, 8), rows_per_group=0), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16), rows_per_group=2), ValueError),
    (dict(x=_t(4, 16), weight=_t(8, 16)), ValueError),  # on the CPU
])
def test_linear_refuses(kw, error):
    with pytest.raises(error):
        wf("enhancers.fused_linear").linear(**kw)


@pytest.mark.parametrize("kw,error", [
    (dict(x=_t(4, 16, dtype="float64")), TypeError),
    (dict(x=_t(4, 16), weight=_t(16, dtype="float16")), TypeError),
    (dict(x=_t(4, 16, dtype="float32"), weight=_t(16)), TypeError),
    (dict(x=_t(4, 16), weight=_t(16), bias=_t(16, dtype="float32")), TypeError),
    (dict(x=_t(4, 0)), ValueError),
    (dict(x=_t(4, 16), eps=-1.0), ValueError),
    (dict(x=_t(4, 16), eps=float("nan")), ValueError),
    (dict(x=_t(4, 16), weight=_t(15)), ValueError),
    (dict(x=_t(4, 16), weight=_t(16), bias=_t(1, 16)), ValueError),
    (dict(x=_t(4, 16), weight=_t(3, 16)), ValueError),
    (dict(x=_t(4, 16), weight=_t(0, 16)), ValueError),
    (dict(x=_t(4, 16), weight=_t(2, 16), rows_per_group=4), ValueError),
    (dict(x=_t(4, 16), rows_per_group=4), ValueError),
    (dict(x=_t(4, 16), weight=_t(16)), ValueError),  # on the CPU
])
def test_layer_norm_refuses(kw, error):
    with pytest.raises(error):
        wf("enhancers.fused_norm").layer_norm(**kw)


ARG, UNSUPPORTED = -1, -2
P = 4096  # an aligned address that no refused call reads


def _call(name, layout, fields, kw):
    assert set(kw) <= set(fields), kw
    return getattr(wf("_ext").lib(), name)(getattr(dense_cabi, layout).pack(*{**fields, **kw}.values()), None)


def _linear(**kw):
    return _call("wf_linear", "LINEAR_ARGS", dict(
        x=P, w=P, bias=0, gate=0, resid=0, y=P, z=0, ldx=64, ldw=64, ldr=0, ldy=32, ldz=0, rpg=1, m=4, n=32, k=64, act=0,
        type=1, zt=0, reserved=0), kw)


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), UNSUPPORTED), (dict(act=5), UNSUPPORTED), (dict(act=-1), UNSUPPORTED), (dict(m=-1), ARG), (dict(k=0), ARG),
    (dict(n=1 << 31), ARG), (dict(x=0), ARG), (dict(x=P + 8), ARG), (dict(ldx=60), ARG), (dict(ldx=68), ARG),
    (dict(ldw=56), ARG), (dict(w=P + 2), ARG), (dict(ldy=31), ARG), (dict(y=P + 1), ARG), (dict(gate=P, rpg=0), ARG),
    (dict(resid=P, ldr=8), ARG), (dict(z=P, ldz=8), ARG), (dict(z=P, ldz=32, zt=3), UNSUPPORTED), (dict(m=0), 0), (dict(n=0), 0),
])
def test_c_linear_refuses(kw, rc):
    assert _linear(**kw) == rc


def test_c_linear_backward_refuses():
    lib = wf("_ext").lib()

    def grad(**kw):
        return _call("wf_linear_backward", "LINEAR_GRAD_ARGS", dict(
            dy=P, x=P, w=P, z=P, gate=0, dx=P, dw=P, db=0, dg=0, ws=P, lddy=32, ldx=64, ldw=64, ldz=32, lddx=64, lddw=64,
            rpg=4, size=1 << 20, m=4, n=32, k=64, act=3, type=1, zt=0, reserved=0), kw)
    assert grad(type=2) == UNSUPPORTED and grad(act=9) == UNSUPPORTED and grad(zt=7) == UNSUPPORTED
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(dy=0), dict(lddy=31), dict(ldz=31), dict(z=0), dict(rpg=0), dict(ws=0),
                dict(size=8), dict(ws=P + 8), dict(dy=P + 1), dict(act=0, z=0, dg=P), dict(w=0), dict(x=0), dict(w=P + 8),
                dict(ldx=63), dict(ldw=68), dict(lddx=63), dict(lddw=63), dict(dx=P + 1), dict(db=P + 1)):
        assert grad(**bad) == ARG, bad
    assert grad(dx=0, dw=0) == 0
    assert lib.wf_linear_backward_workspace(4, 32, 4) >= 4 * 32 * 2 and lib.wf_linear_backward_workspace(0, 32, 4) == 0
    assert lib.wf_linear(None, None) == ARG and lib.wf_linear_backward(None, None) == ARG
    copy = dense_cabi.COPY_ROWS.pack
    assert lib.wf_copy_rows16(copy(P, P, 4, 8, 3, 5), 1, None) == ARG and lib.wf_copy_rows16(copy(P, P, 8, 8, 0, 5), 1, None) == 0
    assert lib.wf_copy_rows16(copy(P, P, 8, 8, 3, 5), 3, None) == ARG and lib.wf_copy_rows16(None, 1, None) == ARG
    assert lib.wf_linear_status(ctypes.POINTER(ctypes.c_int)()) == ARG


def test_c_layer_norm_refuses():
    lib = wf("_ext").lib()

    def norm(**kw):
        return _call("wf_layer_norm", "LAYER_NORM_ARGS", dict(
            x=P, w=P, b=P, y=P, mean=0, rstd=0, ldx=64, ldy=64, rows=4, d=64, rpg=4, eps=1e-6, type=1, wt=1, reserved=0), kw)
    assert norm(type=5) == UNSUPPORTED and norm(wt=0) == UNSUPPORTED and norm(type=2, wt=1) == UNSUPPORTED
    for bad in (dict(rows=-1), dict(d=0), dict(ldx=63), dict(ldy=63), dict(rpg=0), dict(eps=-1.0), dict(eps=float("nan")),
                dict(mean=P), dict(x=0), dict(y=P + 1), dict(w=P + 1), dict(mean=P + 2, rstd=P)):
        assert norm(**bad) == ARG, bad
    assert norm(rows=0) == 0

    def back(**kw):
        return _call("wf_layer_norm_backward", "LAYER_NORM_GRAD_ARGS", dict(
            dy=P, x=P, w=P, mean=P, rstd=P, dx=P, dw=0, db=0, ws=0, lddy=64, ldx=64, lddx=64, rows=4, d=64, rpg=4, size=0,
            type=1, wt=1), kw)
    for bad in (dict(dy=0), dict(mean=0), dict(rows=0), dict(lddx=8), dict(dw=P), dict(dw=P, ws=P, size=16), dict(rpg=0)):
        assert back(**bad) == ARG, bad
    assert back(dx=0) == 0
    assert lib.wf_layer_norm(None, None) == ARG and lib.wf_layer_norm_backward(None, None) == ARG


def test_argument_structures_match_the_header(tmp_path):
    """Each packed layout has the size that a C compiler gives the header's structure."""
    import os
    import subprocess
    from conftest import REPO
    names = {"wf_linear_args": dense_cabi.LINEAR_ARGS, "wf_linear_grad_args": dense_cabi.LINEAR_GRAD_ARGS,
             "wf_copy_rows": dense_cabi.COPY_ROWS, "wf_layer_norm_args": dense_cabi.LAYER_NORM_ARGS,
             "wf_layer_norm_grad_args": dense_cabi.LAYER_NORM_GRAD_ARGS}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "weightferry_b200.h"\nint main(void) {'
                   + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    sizes = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in sizes] == [s.size for s in names.values()]
