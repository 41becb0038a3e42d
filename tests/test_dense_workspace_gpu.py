"""The dense linear layer's backward pass stays inside the workspace that it asks for, and takes no more of the device."""

import math

import pytest

import dense_cabi
from conftest import wf
from dense_reference import assert_within, linear_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,rpg", [(300, 72, 300), (300, 72, 100), (301, 61, 7), (2000, 264, 1), (4096, 1024, 4096)])
@pytest.mark.parametrize("results", ["dx dw db dg", "dg", "db", "db dg", "dx dg", "dw"])
def test_exact_workspace(cuda, m, n, rpg, results):
    """Results as in a call with every result, bit for bit, and nothing written behind the last byte."""
    import torch
    lib = wf("_ext").lib()
    k, groups = 64, -(-m // rpg)
    g = torch.Generator(device="cuda").manual_seed(m + n + rpg)

    def normal(*shape, s=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * s).to(torch.bfloat16)
    x, w, gate, dy = normal(m, k), normal(n, k, s=1 / math.sqrt(k)), normal(groups, n), normal(m, n)
    z = (x.double() @ w.double().t()).float()
    want = linear_reference(x, w, torch.zeros(n, device="cuda").bfloat16(), "silu", None, gate, rpg, dy)
    out = {"dx": torch.empty_like(x), "dw": torch.empty_like(w), "db": torch.empty_like(w[:, 0]), "dg": torch.empty_like(gate)}
    p = {nm: t.data_ptr() if nm in results.split() else 0 for nm, t in out.items()}

    def pack(ws, size):
        return dense_cabi.LINEAR_GRAD_ARGS.pack(
            dy.data_ptr(), x.data_ptr(), w.data_ptr(), z.data_ptr(), gate.data_ptr(), p["dx"], p["dw"], p["db"], p["dg"], ws, n, k, k,
            n, k, k, rpg, size, m, n, k, 2, 1, 2, 0)
    need = lib.wf_linear_backward_needs(pack(0, 0))
    work = torch.full((need + 4096,), 113, device="cuda", dtype=torch.uint8)
    dense_cabi.launch("wf_linear_backward", pack(work.data_ptr(), need))
    assert bool((work[need:] == 113).all())
    for nm, key in (("dx", "x"), ("dw", "weight"), ("db", "bias"), ("dg", "gate")):
        if p[nm]:
            assert_within(out[nm], want[key], nm)


def test_memory_of_a_step(cuda):
    """Without an activation the products read dy: dx and dw are all that a backward pass takes. A gate row for each row, without a
    gradient of its own, costs dz alone."""
    import torch
    linear = wf("enhancers.fused_linear").linear
    m, k, n = 8192, 64, 2048
    x, w = (torch.ones(s, device="cuda").bfloat16().requires_grad_() for s in ((m, k), (n, k)))
    dy, gate = torch.ones((m, n), device="cuda").bfloat16(), torch.ones((m, n), device="cuda").bfloat16()
    for g, most in ((None, 0), (gate, 2 * m * n)):
        y = linear(x, w, gate=g)
        torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        torch.autograd.grad(y, (x, w), dy)
        grads = 2 * (m * k + n * k)
        assert torch.cuda.max_memory_allocated() - before <= grads + most + (4 << 20)
