"""The dense operators refuse PyTorch's graph tracers (make_fx on real and on fake tensors), which would record the empty output
and not the launch; modes that only watch are none."""

import pytest

from conftest import wf


def _calls():
    import torch
    x, w, nw = torch.randn(4, 16).bfloat16(), torch.randn(8, 16).bfloat16(), torch.ones(16).bfloat16()
    return x, (lambda t: wf("enhancers.fused_linear").linear(t, w), lambda t: wf("enhancers.fused_norm").layer_norm(t, nw))


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_graph_tracers_are_refused(mode):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, calls = _calls()
    for call in calls:
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call, tracing_mode=mode)(x)


def test_watching_modes_are_ordinary():
    from torch.utils.flop_counter import FlopCounterMode
    x, calls = _calls()
    for call in calls:
        with FlopCounterMode(display=False), pytest.raises(ValueError, match="CUDA device"):
            call(x)
