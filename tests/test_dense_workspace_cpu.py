"""How much workspace the dense linear layer's backward pass asks for, without a GPU."""

import itertools
import random

import pytest

import dense_cabi
from conftest import wf

P = 4096  # an aligned address that nothing reads
FIELDS = ("dy x w z gate dx dw db dg ws lddy ldx ldw ldz lddx lddw rpg size m n k act type zt reserved").split()


def _needs(**kw):
    d = dict.fromkeys(FIELDS, 0)
    d.update(dy=P, x=P, w=P, rpg=1, type=1)
    d.update(kw)
    return wf("_ext").lib().wf_linear_backward_needs(dense_cabi.LINEAR_GRAD_ARGS.pack(*d.values()))


def test_only_what_the_call_uses():
    m, n = 4096, 2048
    size = dict(m=m, n=n, k=512, lddy=n, rpg=m)
    assert _needs(**size, dx=P, dw=P) == 0                                    # the products read dy
    assert _needs(**size, dx=P, dw=P, act=3, z=P) == m * n * 2                # dz
    assert _needs(**size, dx=P, gate=P) == m * n * 2
    assert _needs(**{**size, "lddy": n + 3}, dx=P) == m * n * 2               # dy that TMA cannot read
    assert _needs(**size, db=P, act=3, z=P) == _needs(**size, db=P) > 0       # partial sums alone
    assert _needs(**size, db=P) < m * n // 4
    one_row = {**size, "rpg": 1}
    assert _needs(**one_row, dx=P, gate=P, act=3, z=P) == m * n * 2           # a gate row a row, and no gradient of it
    assert _needs(**one_row, dg=P, gate=P, z=P) == m * n * 4
    assert wf("_ext").lib().wf_linear_backward_needs(None) == 0
    assert _needs(**{**size, "m": 0}) == 0 and _needs(**{**size, "rpg": 0}) == 0


def test_never_more_than_the_sizes_allow():
    lib, rng = wf("_ext").lib(), random.Random(3)
    for _ in range(3000):
        m, n = int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 14))
        rpg = rng.choice([1, 2, 7, max(1, m // 3), m, m + 5, rng.randint(1, m)])
        most = lib.wf_linear_backward_workspace(m, n, rpg)
        for db, dg, gate, dx in itertools.product((0, P), repeat=4):
            if dg and not gate:
                continue
            got = _needs(m=m, n=n, k=64, lddy=n, rpg=rpg, db=db, dg=dg, gate=gate, dx=dx, act=3, z=P)
            assert got <= most, (m, n, rpg, db, dg, gate, dx)


@pytest.mark.parametrize("short", [1, 16])
def test_a_smaller_workspace_is_refused(short):
    d = dict.fromkeys(FIELDS, 0)
    d.update(dy=P, x=P, w=P, z=P, dx=P, db=P, ws=P, rpg=300, type=1, act=3, m=300, n=72, k=64, lddy=72, ldx=64, ldw=64, ldz=72,
             lddx=64)
    ext = wf("_ext")
    need = ext.lib().wf_linear_backward_needs(dense_cabi.LINEAR_GRAD_ARGS.pack(*d.values()))
    d["size"] = need - short
    assert ext.lib().wf_linear_backward(dense_cabi.LINEAR_GRAD_ARGS.pack(*d.values()), None) == -1
