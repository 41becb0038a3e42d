"""What the dense linear layer and layer norm refuse, without a GPU: wrong shapes, types, devices and groups at the Python
entry points, and bad sizes, pitches, pointers and types at the C entry points (which check before they look at the
device)."""

import ctypes

import pytest

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


def _linear(**kw):
    a = dict(x=P, ldx=64, w=P, ldw=64, bias=None, act=0, gate=None, rpg=1, resid=None, ldr=0, y=P, ldy=32, z=None, ldz=0,
             zt=0, m=4, n=32, k=64, type=1, st=None)
    a.update(kw)
    return wf("_ext").lib().wf_linear(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(type=2), UNSUPPORTED), (dict(act=5), UNSUPPORTED), (dict(act=-1), UNSUPPORTED), (dict(m=-1), ARG), (dict(k=0), ARG),
    (dict(n=1 << 31), ARG), (dict(x=None), ARG), (dict(x=P + 8), ARG), (dict(ldx=60), ARG), (dict(ldx=68), ARG),
    (dict(ldw=56), ARG), (dict(w=P + 2), ARG), (dict(ldy=31), ARG), (dict(y=P + 1), ARG), (dict(gate=P, rpg=0), ARG),
    (dict(resid=P, ldr=8), ARG), (dict(z=P, ldz=8), ARG), (dict(z=P, ldz=32, zt=3), UNSUPPORTED), (dict(m=0), 0), (dict(n=0), 0),
])
def test_c_linear_refuses(kw, rc):
    assert _linear(**kw) == rc


def test_c_linear_backward_refuses():
    lib = wf("_ext").lib()

    def grad(dy=P, lddy=32, z=P, ldz=32, zt=0, act=3, gate=None, rpg=4, dz=P, lddz=32, db=None, dg=None, m=4, n=32, type=1,
             ws=None, size=0):
        return lib.wf_linear_backward_act(dy, lddy, z, ldz, zt, act, gate, rpg, dz, lddz, db, dg, m, n, type, ws, size, None)
    assert grad(type=2) == UNSUPPORTED and grad(act=9) == UNSUPPORTED
    for bad in (dict(m=0), dict(n=0), dict(dy=None), dict(lddy=31), dict(ldz=31), dict(lddz=31), dict(z=None), dict(rpg=0),
                dict(db=P), dict(dg=P, ws=P, size=4), dict(dy=P + 1), dict(act=0, z=None, dg=P)):
        assert grad(**bad) == ARG, bad
    assert grad(dz=None) == 0
    assert lib.wf_linear_backward_input(P, 32, P, 64, P, 63, 4, 32, 64, 1, None) == ARG
    assert lib.wf_linear_backward_input(P, 33, P, 64, P, 64, 4, 32, 64, 1, None) == ARG
    assert lib.wf_linear_backward_input(P, 32, P, 64, P, 64, 4, 32, 64, 2, None) == UNSUPPORTED
    assert lib.wf_linear_backward_weight(P, 32, P + 4, 64, P, 64, 4, 32, 64, 1, None) == ARG
    assert lib.wf_linear_backward_weight(P, 32, P, 64, None, 64, 4, 32, 64, 1, None) == ARG
    assert lib.wf_copy_rows16(P, 4, P, 8, 3, 5, None) == ARG and lib.wf_copy_rows16(P, 8, P, 8, 0, 5, None) == 0
    assert lib.wf_linear_status(ctypes.POINTER(ctypes.c_int)()) == ARG


def test_c_layer_norm_refuses():
    lib = wf("_ext").lib()

    def norm(x=P, ldx=64, w=P, b=P, wt=1, y=P, ldy=64, mean=None, rstd=None, rows=4, d=64, rpg=4, eps=1e-6, type=1):
        return lib.wf_layer_norm(x, ldx, w, b, wt, y, ldy, mean, rstd, rows, d, rpg, eps, type, None)
    assert norm(type=5) == UNSUPPORTED and norm(wt=0) == UNSUPPORTED and norm(type=2, wt=1) == UNSUPPORTED
    for bad in (dict(rows=-1), dict(d=0), dict(ldx=63), dict(ldy=63), dict(rpg=0), dict(eps=-1.0), dict(eps=float("nan")),
                dict(mean=P), dict(x=None), dict(y=P + 1), dict(w=P + 1)):
        assert norm(**bad) == ARG, bad
    assert norm(rows=0) == 0

    def back(dy=P, x=P, mean=P, rstd=P, dx=P, lddx=64, dw=None, db=None, rows=4, d=64, rpg=4, type=1, ws=None, size=0):
        return lib.wf_layer_norm_backward(dy, 64, x, 64, P, 1, mean, rstd, dx, lddx, dw, db, rows, d, rpg, type, ws, size, None)
    for bad in (dict(dy=None), dict(mean=None), dict(rows=0), dict(lddx=8), dict(dw=P), dict(dw=P, ws=P, size=16), dict(rpg=0)):
        assert back(**bad) == ARG, bad
    assert back(dx=None) == 0
