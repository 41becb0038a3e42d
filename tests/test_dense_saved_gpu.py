"""The dense operators' saved tensors: hooks that return them with strides of their own, and what comes back changed."""

import math

import pytest

from conftest import wf
from dense_reference import assert_within, norm_reference

pytestmark = pytest.mark.gpu


def _hooks(torch):
    saved_tensors_hooks = torch.autograd.graph.saved_tensors_hooks

    def apart(t):  # rows twice as far apart
        out = torch.empty_strided(t.shape, [2 * s + (s > 1) for s in t.stride()], dtype=t.dtype, device=t.device) \
            if t.dim() == 2 and t.stride(1) == 1 else torch.empty_like(t)
        return out.copy_(t)
    return {
        "save_on_cpu": lambda: torch.autograd.graph.save_on_cpu(),
        "contiguous": lambda: saved_tensors_hooks(lambda t: t, lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)),
        "transposed": lambda: saved_tensors_hooks(lambda t: t.t().contiguous() if t.dim() == 2 else t,
                                                  lambda t: t.t() if t.dim() == 2 else t),
        "apart": lambda: saved_tensors_hooks(lambda t: t, apart),
    }


def _calls(torch):
    """(name, call, leaves): operands of every layout that is read in place or copied."""
    fl, fn = wf("enhancers.fused_linear"), wf("enhancers.fused_norm")
    g = torch.Generator(device="cuda").manual_seed(5)

    def normal(*shape, dtype=torch.bfloat16, s=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * s).to(dtype)
    for m, k, n in ((40, 120, 88), (1, 120, 88), (300, 68, 61), (70, 61, 264)):
        wide, wbig, gate = normal(m, 256), normal(n + 5, 200, s=1 / math.sqrt(k)), normal(2 if m > 1 else 1, 2 * n)
        for name, x, w in (("slices", wide[:, :k], wbig[5:, :k]), ("odd slices", wide[:, 3:3 + k], wbig[5:, 1:1 + k]),
                           ("whole", wide[:, :k].contiguous(), wbig[5:, :k].contiguous())):
            for kind, gated in (("gelu", False), ("relu", True), ("none", True)):
                yield (f"linear {m} {k} {n} {name} {kind} {gated}",
                       lambda x, w, g, kind=kind, gated=gated: fl.linear(x, w, activation=kind, gate=g if gated else None),
                       (x, w, gate[:, :n]))
    for m, d in ((40, 120), (1, 120), (33, 61), (700, 1024)):
        for dtype in (torch.bfloat16, torch.float32):
            wide, w = normal(m, 2 * d, dtype=dtype), normal(d, 2, dtype=dtype)
            for name, x in (("slice", wide[:, :d]), ("odd slice", wide[:, 3:3 + d]), ("whole", wide[:, :d].contiguous())):
                yield f"norm {m} {d} {dtype} {name}", lambda x, w: fn.layer_norm(x, w), (x, w[:, 0])


def _dy(torch, y):
    return torch.linspace(-1, 1, y.numel(), device="cuda").to(y.dtype).view(y.shape)


def _grads(torch, call, leaves, hook=None):
    leaves = [t.detach().requires_grad_() for t in leaves]
    if hook is None:
        y = call(*leaves)
    else:
        with hook():
            y = call(*leaves)
    return [t for t in torch.autograd.grad(y, leaves, _dy(torch, y), allow_unused=True) if t is not None]


@pytest.mark.parametrize("hook", ["save_on_cpu", "contiguous", "transposed", "apart"])
def test_hooks_that_return_other_strides(cuda, hook):
    """The linear layer's gradients have the bits that they have without a hook; layer norm's, whose kernels differ by layout,
    are within their bounds of the definition."""
    import torch
    make = _hooks(torch)[hook]
    for name, call, leaves in _calls(torch):
        got = _grads(torch, call, leaves, make)
        if name.startswith("linear"):
            want = _grads(torch, call, leaves)
            assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(want, got)), name
        else:
            x, w = leaves
            want = norm_reference(x, w.view(1, -1), None, 1e-6, 1 << 30, _dy(torch, x))
            assert_within(got[0], want["x"], name + " x")
            assert_within(got[1].view(1, -1), want["weight"], name + " weight")


def test_checkpointed_step(cuda):
    import torch
    from torch.utils.checkpoint import checkpoint
    for name, call, leaves in _calls(torch):
        want = _grads(torch, call, leaves)
        got = _grads(torch, lambda *a: checkpoint(call, *a, use_reentrant=False), leaves)
        assert all(torch.equal(a, b) for a, b in zip(want, got)), name


@pytest.mark.parametrize("change", [lambda t: t[:-1], lambda t: t.float() if t.dtype.itemsize == 2 else t.half(), lambda t: t.cpu()])
def test_changed_saved_tensors_are_refused(cuda, change):
    """A hook that returns another shape, type or device: an error, and nothing is launched."""
    import torch
    for name, call, leaves in _calls(torch):
        if leaves[0].shape[0] == 1:
            continue
        with pytest.raises(RuntimeError, match="came back as"):
            _grads(torch, call, leaves, lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, change))
