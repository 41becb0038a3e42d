"""The operators together, as they are used: the streamed stack's blocks with the fused dense linear layer
(WEIGHTFERRY_FUSED_LINEAR=1) against the block-level oracle, and a block's MLP sub-layer -- adaLN norm, input layer with
GELU, output layer with the gated residual -- as a training step against float64, eager and captured."""

import importlib
import math
import os
import subprocess
import sys

import pytest

from conftest import REPO, wf

pytestmark = pytest.mark.gpu


def test_stack_blocks_with_fused_linear_match_block_oracle(cuda, monkeypatch):
    """The bounds of the unfused blocks (tests/test_block_oracle_gpu.py): the fused path rounds at fewer places."""
    import torch
    monkeypatch.setenv("WEIGHTFERRY_FUSED_LINEAR", "1")
    ob = importlib.import_module("oracle.block")
    cb, stk, fl = wf("streaming.cosmos_block"), wf("streaming.stack"), wf("enhancers.fused_linear")
    calls = []
    real = fl.linear
    monkeypatch.setattr(fl, "linear", lambda *a, **kw: calls.append(kw) or real(*a, **kw))
    cfg = cb.CosmosConfig(hidden=1024, heads=8, mlp=4096, ctx_dim=512, lora=64)
    batch, T, H, W, S = 2, 1, 8, 8, 32
    tokens = T * H * W
    g = torch.Generator(device="cuda").manual_seed(41)
    x = torch.randn((batch * tokens, cfg.hidden), device="cuda", generator=g).to(torch.bfloat16)
    emb = (torch.randn((batch, cfg.hidden), device="cuda", generator=g) * 0.5).to(torch.bfloat16)
    lora = (torch.randn((batch, 3 * cfg.hidden), device="cuda", generator=g) * 0.05).to(torch.bfloat16)
    ctx = torch.randn((batch, S, cfg.ctx_dim), device="cuda", generator=g).to(torch.bfloat16)
    rope = cb.rope3d_table(T, H, W, device="cuda")
    stack = stk.StreamedStack(cfg, 2, "cuda", seed=505, num_slots=2)
    y = stack.forward(x, emb, ctx, rope, batch, tokens, lora)
    torch.cuda.synchronize()
    assert len(calls) == 8 and sum(c.get("activation") == "gelu" for c in calls) == 2
    ref = x.cpu().to(torch.float64)
    for b in range(2):
        Wb = ob.dequant_block(stack.host_flats[b], stack.layout)
        ref = ob.block_forward(ref, emb.cpu(), ctx.cpu(), rope.cpu(), Wb, cfg.heads, cfg.eps, batch, tokens, lora.cpu())
    stack.close()
    y64, x64 = y.cpu().to(torch.float64), x.cpu().to(torch.float64)
    d = (y64 - ref).abs()
    row = ref.pow(2).mean(dim=1, keepdim=True).sqrt()
    assert bool(torch.isfinite(y64).all())
    assert bool((d / row).max() <= 0.12) and bool(d.mean() <= 0.006 * row.mean())
    assert float(((y64 - x64) - (ref - x64)).norm() / (ref - x64).norm()) <= 1e-2


def _sublayer(x, nw, nb, w1, b1, w2, gate, norm, linear):
    n = norm(x, nw, nb)
    return linear(linear(n, w1, b1, activation="gelu"), w2, residual=x, gate=gate)


def test_mlp_sublayer_training_step(cuda):
    """Two groups of rows. The reference repeats the 16-bit roundings between the operators (they are the path's, not the
    operators'), so that what is left is each operator's own error: bounded in norm by the roundings that a gradient goes
    through, each off by at most half a step relative to its value, with a factor 2 for their accumulation."""
    import torch
    fl, fn = wf("enhancers.fused_linear"), wf("enhancers.fused_norm")
    m, d, hid, groups = 600, 256, 1024, 2
    for dtype in (torch.bfloat16, torch.float16):
        g = torch.Generator(device="cuda").manual_seed(7)

        def normal(*shape, s=1.0, o=0.0):
            return (torch.randn(shape, device="cuda", generator=g) * s + o).to(dtype)
        data = [normal(m, d), normal(groups, d, s=0.2, o=1.0), normal(groups, d, s=0.2), normal(hid, d, s=1 / math.sqrt(d)),
                normal(hid, s=0.1), normal(d, hid, s=1 / math.sqrt(hid)), normal(groups, d, s=0.3, o=0.3)]
        dy = normal(m, d)

        class Round(torch.autograd.Function):  # to dtype and back, straight through in both directions
            @staticmethod
            def forward(ctx, t):
                return t.to(dtype).double()

            @staticmethod
            def backward(ctx, t):
                return t.to(dtype).double()
        rows = torch.arange(m, device="cuda") // (m // groups)

        def norm64(x, w, b):
            return Round.apply(torch.nn.functional.layer_norm(x, (d,), None, None, 1e-6) * w[rows] + b[rows])

        def linear64(x, w, b=None, activation="none", residual=None, gate=None):
            h = x @ w.t()
            h = torch.nn.functional.gelu(h + b) if b is not None else h
            return Round.apply(h if residual is None else residual + gate[rows] * h)
        leaves64 = [t.double().requires_grad_() for t in data]
        y64 = _sublayer(*leaves64, norm64, linear64)
        want = torch.autograd.grad(y64, leaves64, dy.double())

        def step():
            leaves = [t.clone().requires_grad_() for t in data]
            y = _sublayer(*leaves, fn.layer_norm, fl.linear)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))
        got = step()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            replayed = step()
        graph.replay()
        torch.cuda.synchronize()
        half = torch.finfo(dtype).eps / 2
        for i, (a, r, b) in enumerate(zip(got, replayed, (y64.detach(), *want))):
            assert torch.equal(a.view(torch.int16), r.view(torch.int16)), i
            # the most roundings on the way to a gradient: y, z, dz, h (twice), dz again, the norm's input gradient, the sum
            assert float((a.double() - b).norm()) <= 2 * 8 * half * float(b.norm()), i


@pytest.mark.parametrize("kernel", ["0", "1"])
def test_each_kernel_alone_covers_every_size(cuda, kernel):
    """WEIGHTFERRY_LINEAR_PAIR is read once a process: the tile kernel alone, and the pair kernel alone."""
    env = {**os.environ, "WEIGHTFERRY_LINEAR_PAIR": kernel}
    res = subprocess.run(["timeout", "-k", "10", "300", sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu",
                          os.path.join(REPO, "tests", "test_linear_gpu.py"), "-k", "forward or gradients or groups or memory"],
                         cwd=REPO, capture_output=True, text=True, env=env)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]
