"""The dense operators' gradients can be taken once: every way of differentiating them again raises, whichever operand it asks for
and whether or not unused operands are allowed."""

import pytest

from conftest import wf

pytestmark = pytest.mark.gpu


def _operands(torch, op):
    g = torch.Generator(device="cuda").manual_seed(2)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).bfloat16().requires_grad_()
    if op == "linear":
        leaves = [normal(6, 16), normal(24, 16), normal(24), normal(6, 24), normal(2, 24)]
        return leaves, lambda x, w, b, r, gate: wf("enhancers.fused_linear").linear(x, w, b, "gelu", r, gate), 3
    leaves = [normal(6, 16), normal(2, 16), normal(2, 16)]
    return leaves, lambda x, w, b: wf("enhancers.fused_norm").layer_norm(x, w, b), None


@pytest.mark.parametrize("op", ["linear", "norm"])
def test_again_for_every_operand(cuda, op):
    import torch
    leaves, call, resid = _operands(torch, op)
    y = call(*[t * 1 for t in leaves])
    dy = torch.randn_like(y).requires_grad_()
    grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for i, first in enumerate(grads):
        for second in [*leaves, dy]:
            if i == resid:  # dy itself
                got, = torch.autograd.grad(first.sum(), second, retain_graph=True, allow_unused=True)
                assert torch.equal(got, torch.ones_like(dy)) if second is dy else got is None
            else:
                with pytest.raises(RuntimeError, match="differentiated again"):
                    torch.autograd.grad(first.sum(), second, retain_graph=True, allow_unused=True)


@pytest.mark.parametrize("op", ["linear", "norm"])
def test_again_by_the_functional_forms(cuda, op):
    import torch
    leaves, call, _ = _operands(torch, op)
    x, rest = leaves[0].detach(), [t.detach() for t in leaves[1:]]
    f = torch.autograd.functional
    with pytest.raises(RuntimeError, match="differentiated again"):
        f.jvp(lambda t: call(t, *rest), x, torch.ones_like(x))
    with pytest.raises(RuntimeError, match="differentiated again"):
        f.hvp(lambda t: call(t, *rest).float().square().sum(), x, torch.ones_like(x))


@pytest.mark.parametrize("op", ["linear", "norm"])
def test_recorded_gradients_have_their_values(cuda, op):
    """create_graph changes nothing of the first derivatives, and a use of them that is not differentiated again is free."""
    import torch
    leaves, call, _ = _operands(torch, op)
    y = call(*leaves)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    penalty = sum(t.detach().float().square().sum() for t in got)
    assert bool(torch.isfinite(penalty))
