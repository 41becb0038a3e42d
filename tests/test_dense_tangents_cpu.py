"""The dense operators refuse, before they look at the device, what they would drop without a word: forward-mode tangents and an
active tracer."""

import pytest

from conftest import wf


def _leaves():
    import torch
    x, w = torch.randn(4, 16).bfloat16(), torch.randn(8, 16).bfloat16()
    return x, w, torch.randn(8).bfloat16(), torch.randn(4, 8).bfloat16(), torch.randn(2, 8).bfloat16()


def _linear(x, w, b, r, g):
    return wf("enhancers.fused_linear").linear(x, w, b, residual=r, gate=g)


def _norm(x, w, b):
    return wf("enhancers.fused_norm").layer_norm(x, w, b)


def _dual_error(call, leaves, which, **kw):
    import torch
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        args = [fw.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(leaves)]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*args)
    args = [t.detach().requires_grad_() for t in leaves]
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*args)


@pytest.mark.parametrize("which", range(5))
def test_linear_refuses_tangents(which):
    _dual_error(_linear, _leaves(), which)


@pytest.mark.parametrize("which", range(3))
def test_layer_norm_refuses_tangents(which):
    x, w, _, _, _ = _leaves()
    _dual_error(_norm, (x, w[0].clone(), w[1].clone()), which)


def test_tangents_that_are_off_are_none():
    """A primal taken out of its dual, and forward mode switched off, are ordinary calls (refused here for the CPU alone)."""
    import torch
    fw = torch.autograd.forward_ad
    x, w, b, r, g = _leaves()
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="CUDA device"):
            _linear(fw.unpack_dual(dual).primal, w, b, r, g)
        with fw._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA device"):
            _linear(dual, w, b, r, g)


def test_tracer_is_refused():
    import torch
    x, w, b, r, g = _leaves()
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(lambda t: _linear(t, w, b, r, g), x)
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(lambda t: _norm(t, w[0], w[1]), x)
