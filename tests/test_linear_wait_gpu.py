"""A pipeline wait of the dense linear layer made to run out on purpose: with the limit shortened to 1 ns (the library's test
hook) the kernels stop issuing, drain the copies and MMAs that they started, and leave NaN where no result is; the host
learns of it."""

import ctypes

import pytest

from conftest import wf

pytestmark = pytest.mark.gpu


def _limit(ns):
    ext = wf("_ext")
    ext.check(ext.lib().wf_linear_set_wait_limit(ctypes.c_uint64(ns)), "wf_linear_set_wait_limit")


# one CTA a tile, tiles shared by a cluster, CTA pairs, CTA pairs with outputs of an odd width: long contractions, so that some
# wait does not end at its first try
@pytest.mark.parametrize("m,k,n", [(16, 16384, 20480), (24, 32768, 1024), (4096, 8192, 2048), (4096, 8192, 2041)])
@pytest.mark.parametrize("kind", ["none", "gelu"])
def test_expired_waits_leave_nan_and_are_reported(cuda, m, k, n, kind):
    import torch
    fl = wf("enhancers.fused_linear")
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn((m, k), device="cuda", generator=g).bfloat16().requires_grad_()
    w = (torch.randn((n, k), device="cuda", generator=g) * 0.02).bfloat16().requires_grad_()
    dy = torch.ones((m, n), device="cuda", dtype=torch.bfloat16)
    assert fl.status() == 0
    want = fl.linear(x, w, activation=kind)
    grads = torch.autograd.grad(want, (x, w), dy, retain_graph=True)
    torch.cuda.synchronize()
    # forward
    _limit(1)
    try:
        y = fl.linear(x, w, activation=kind).detach()
        torch.cuda.synchronize()
    finally:
        _limit(0)
    bad = torch.isnan(y)
    assert bool(bad.any()) and torch.equal(y[~bad], want.detach()[~bad])
    with pytest.raises(RuntimeError, match="ran out of time"):
        fl.linear(x, w, activation=kind)
    with pytest.raises(RuntimeError, match="ran out of time"):
        torch.autograd.grad(want, (x, w), dy, retain_graph=True)
    assert fl.status() in (1, 2, 3) and fl.status() == 0
    # one product of the backward pass
    _limit(1)
    try:
        dx, = torch.autograd.grad(want, x, dy, retain_graph=True)
        torch.cuda.synchronize()
    finally:
        _limit(0)
    bad = torch.isnan(dx)
    assert torch.equal(dx[~bad], grads[0][~bad])
    assert bool(bad.any()) == (fl.status() in (1, 2, 3))
    # and everything works again
    assert torch.equal(fl.linear(x, w, activation=kind), want)
    for a, b in zip(torch.autograd.grad(want, (x, w), dy), grads):
        assert torch.equal(a, b)
    assert fl.status() == 0


def test_first_call_inside_a_capture(cuda):
    """The word that the host looks at is allocated by a process's first call, a captured one too."""
    import os
    import subprocess
    import sys
    from conftest import REPO
    code = """
import sys; sys.path.insert(0, "tests")
import torch
from conftest import wf
x, w = torch.ones((40, 64), device="cuda").bfloat16(), torch.ones((72, 64), device="cuda").bfloat16()
fl = wf("enhancers.fused_linear")
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    y = fl.linear(x, w)
graph.replay()
torch.cuda.synchronize()
assert bool((y == 64).all()) and fl.status() == 0
print("ok")
"""
    res = subprocess.run(["timeout", "-k", "10", "200", sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True,
                         env=dict(os.environ))
    assert res.returncode == 0 and res.stdout.endswith("ok\n"), res.stdout[-1000:] + res.stderr[-2000:]


@pytest.mark.parametrize("m,k,n", [(24, 32768, 1024), (4096, 8192, 2048), (4096, 8192, 2041)])
@pytest.mark.parametrize("z_name", ["float16", "float32"])
def test_expired_waits_leave_nan_in_the_kept_values(cuda, m, k, n, z_name):
    """z, too, is what a whole run leaves or NaN."""
    import torch
    import dense_cabi
    x = torch.randn((m, k), device="cuda").bfloat16()
    w = (torch.randn((n, k), device="cuda") * 0.02).bfloat16()
    up = (n + 7) // 8 * 8

    def run():
        y = torch.full((m, n), -7.0, device="cuda", dtype=torch.bfloat16)
        z = torch.full((m, up), -7.0, device="cuda", dtype=getattr(torch, z_name))
        dense_cabi.launch("wf_linear", dense_cabi.LINEAR_ARGS.pack(
            x.data_ptr(), w.data_ptr(), 0, 0, 0, y.data_ptr(), z.data_ptr(), k, k, 0, n, up, 1, m, n, k, 3, 1,
            {"float16": 0, "float32": 2}[z_name], 0))
        torch.cuda.synchronize()
        return y, z[:, :n]
    want = run()
    _limit(1)
    try:
        got = run()
    finally:
        _limit(0)
    assert wf("enhancers.fused_linear").status() in (1, 2, 3)
    for a, b in zip(got, want):
        bad = torch.isnan(a)
        assert bool(bad.any()) and torch.equal(a[~bad], b[~bad])
