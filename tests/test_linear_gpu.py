"""The dense linear layer (enhancers/fused_linear.py): outputs and gradients against float64 within derived bounds, on
every kernel variant's sizes; layouts, groups, streams, graphs, empty inputs."""

import math

import pytest

import dense_cabi
from conftest import wf
from dense_reference import ACTS, act, assert_within, linear_reference

pytestmark = pytest.mark.gpu

# (m, k, n): one row to many tiles; widths that no vector access fits; contractions below and past a stage
SIZES = [(1, 16, 8), (1, 1, 1), (1, 2048, 520), (2, 256, 384), (3, 64, 5), (7, 8, 129), (16, 68, 130), (17, 1001, 1013),
         (33, 40, 256), (64, 520, 200), (65, 1024, 64), (129, 72, 136), (300, 520, 264), (333, 256, 1280), (513, 1024, 768),
         (1000, 264, 1001)]


def _data(torch, m, k, n, dtype, bias=True, groups=0, seed=0, rpg=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 131 * m + 17 * k + n)

    def normal(*shape, s=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * s).to(dtype)
    d = {"x": normal(m, k), "weight": normal(n, k, s=1 / math.sqrt(k)), "bias": normal(n) if bias else None,
         "residual": normal(m, n, s=2.0) if groups else None, "gate": normal(groups, n) if groups else None}
    return d, normal(m, n)


def _call(d, kind, rpg=None):
    return wf("enhancers.fused_linear").linear(d["x"], d["weight"], d["bias"], activation=kind, residual=d["residual"],
                                               gate=d["gate"], rows_per_group=rpg)


def _reference(d, kind, dy=None, rpg=None):
    m = d["x"].shape[0]
    groups = 1 if d["gate"] is None else d["gate"].shape[0]
    return linear_reference(d["x"], d["weight"], d["bias"], kind, d["residual"], d["gate"], rpg or max(1, m // groups), dy)


def _train(torch, d, kind, dy, rpg=None):
    names = [nm for nm, t in d.items() if t is not None]
    for nm in names:
        d[nm].requires_grad_(True)
    y = _call(d, kind, rpg)
    return y, dict(zip(names, torch.autograd.grad(y, [d[nm] for nm in names], dy)))


@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward(cuda, m, k, n):
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        d, _ = _data(torch, m, k, n, dtype, bias=False)
        assert_within(_call(d, "none"), _reference(d, "none")["y"], f"plain {dtype}")
        d, _ = _data(torch, m, k, n, dtype, groups=1)
        assert_within(_call(d, "gelu"), _reference(d, "gelu")["y"], f"everything {dtype}")


@pytest.mark.parametrize("kind", ACTS)
def test_activations(cuda, kind):
    import torch
    d, dy = _data(torch, 200, 96, 264, torch.bfloat16)
    d["bias"] = (torch.linspace(-30, 30, 264, device="cuda")).to(torch.bfloat16)  # far into both tails
    want = _reference(d, kind, dy)
    y, grads = _train(torch, d, kind, dy)
    for nm, got in {"y": y.detach(), **grads}.items():
        assert_within(got, want[nm], f"{kind} {nm}")


@pytest.mark.parametrize("m,k,n", SIZES)
def test_gradients(cuda, m, k, n):
    import torch
    for dtype, kind, groups in ((torch.bfloat16, "gelu", 0), (torch.float16, "silu", 1), (torch.bfloat16, "none", 1),
                                (torch.bfloat16, "none", 0)):
        d, dy = _data(torch, m, k, n, dtype, bias=kind != "none" or groups == 0, groups=groups)
        want = _reference(d, kind, dy)
        y, grads = _train(torch, d, kind, dy)
        for nm, got in {"y": y.detach(), **grads}.items():
            assert_within(got, want[nm], f"{dtype} {kind} groups {groups}: {nm}")


@pytest.mark.parametrize("m,rpg", [(12, 1), (100, 10), (100, 33), (4096, 2), (1000, 999), (257, 256), (50, 70)])
def test_gate_groups(cuda, m, rpg):
    """One row a group, groups that end inside tiles, a short last group."""
    import torch
    groups = -(-m // rpg)
    d, dy = _data(torch, m, 40, 72, torch.bfloat16, groups=groups)
    want = _reference(d, "silu", dy, rpg)
    y, grads = _train(torch, d, "silu", dy, rpg)
    for nm, got in {"y": y.detach(), **grads}.items():
        assert_within(got, want[nm], nm)


def test_gradients_against_differences(cuda):
    """The directional derivative of sum(y dy) in float64, by central differences of the definition, against the
    gradients' inner products with the direction."""
    import torch
    d, dy = _data(torch, 24, 32, 40, torch.float16, groups=2)
    y, grads = _train(torch, {nm: t.clone() for nm, t in d.items()}, "gelu_tanh", dy)
    want = _reference(d, "gelu_tanh", dy)
    g = torch.Generator(device="cuda").manual_seed(3)

    def value(shift):
        v = {nm: t.double() + shift.get(nm, 0) for nm, t in d.items()}
        h, _ = act(v["x"] @ v["weight"].t() + v["bias"], "gelu_tanh")
        rows = torch.arange(24, device="cuda") // 12
        return float(((v["residual"] + v["gate"][rows] * h) * dy.double()).sum())
    for nm in d:
        way = torch.randn(d[nm].shape, device="cuda", generator=g, dtype=torch.float64)
        step = 1e-5
        slope = (value({nm: step * way}) - value({nm: -step * way})) / (2 * step)
        got = float((grads[nm].double() * way).sum())
        # the differences' own error: third derivatives times step^2 and float64's cancellation, both below 1e-6 here
        assert abs(got - slope) <= float((want[nm][1] * way.abs()).sum()) + 1e-6 * (1 + abs(slope)), nm


def test_layouts(cuda):
    """Leading dimensions, slices, transposes, expanded rows, unaligned starts: the same bits as contiguous copies."""
    import torch
    fl = wf("enhancers.fused_linear")
    g = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
    big, wbig = normal(6, 7, 200), normal(300, 120)
    w = normal(88, 120)
    cases = [
        (big[:, :, 40:160], w), (big[:, 1:5, 3:123], w), (big[..., :120].transpose(0, 1), w),
        (normal(1, 120).expand(9, 120), w), (normal(120, 31).t(), w), (normal(120), w), (normal(2, 3, 120), wbig[5:93]),
        (normal(5, 120), wbig[::3]), (normal(5, 120), normal(120, 88).t()), (normal(4, 1), normal(7, 1)),
        (normal(4, 240)[:, ::2], w), (normal(40, 1).expand(40, 16), normal(24, 16)),
    ]
    for i, (x, wt) in enumerate(cases):
        n = wt.shape[0]
        res = normal(*x.shape[:-1], 2 * n)[..., :n]
        gate = normal(n, 1).expand(n, 2).t()[:1]
        want = fl.linear(x.contiguous(), wt.contiguous(), residual=res.contiguous(), gate=gate.contiguous())
        got = fl.linear(x, wt, residual=res, gate=gate)
        assert got.is_contiguous() and got.shape == (*x.shape[:-1], n)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), i
        xa, wa = x.detach().requires_grad_(True), wt.detach().requires_grad_(True)
        xb, wb = x.contiguous().requires_grad_(True), wt.contiguous().requires_grad_(True)
        dy = normal(*x.shape[:-1], n)
        for a, b in zip(torch.autograd.grad(fl.linear(xa, wa, activation="gelu"), (xa, wa), dy),
                        torch.autograd.grad(fl.linear(xb, wb, activation="gelu"), (xb, wb), dy)):
            assert torch.equal(a.contiguous().view(torch.int16), b.view(torch.int16)), i
        for a, b in zip(torch.autograd.grad(fl.linear(xa, wa).sum(), (xa, wa)),  # dy expanded from one value
                        torch.autograd.grad(fl.linear(xb, wb), (xb, wb), torch.ones_like(dy))):
            assert torch.equal(a.contiguous().view(torch.int16), b.view(torch.int16)), i


def test_only_what_is_needed(cuda):
    """Any subset of the operands may need a gradient; the others get none, and the values do not depend on the subset."""
    import itertools
    import torch
    fl = wf("enhancers.fused_linear")
    d, dy = _data(torch, 40, 64, 48, torch.bfloat16, groups=2)
    _, full = _train(torch, {nm: t.clone() for nm, t in d.items()}, "none", dy)
    for r in (1, 2, 3):
        for names in itertools.combinations(d, r):
            leaves = {nm: t.clone().requires_grad_(nm in names) for nm, t in d.items()}
            y = fl.linear(leaves["x"], leaves["weight"], leaves["bias"], residual=leaves["residual"], gate=leaves["gate"])
            y.backward(dy)
            for nm, t in leaves.items():
                assert (t.grad is not None) == (nm in names)
                if t.grad is not None:
                    assert torch.equal(t.grad.view(torch.int16), full[nm].view(torch.int16)), (names, nm)


def test_empty(cuda):
    import torch
    fl = wf("enhancers.fused_linear")
    for m, n in ((0, 16), (5, 0), (0, 0)):
        d, dy = _data(torch, m, 24, n, torch.bfloat16)
        y, grads = _train(torch, d, "gelu", dy)
        assert y.shape == (m, n)
        for nm, got in grads.items():
            assert got.shape == d[nm].shape and not bool(got.any())
    assert fl.linear(torch.empty((3, 0, 24), device="cuda", dtype=torch.float16),
                     torch.zeros((8, 24), device="cuda", dtype=torch.float16)).shape == (3, 0, 8)


def test_nonfinite_rows_stay_in_their_rows(cuda):
    import torch
    for m in (5, 300):
        d, _ = _data(torch, m, 64, 72, torch.bfloat16, bias=False)
        clean = _call(d, "silu")
        d["x"][1, 3] = float("nan")
        d["x"][3, 5] = float("inf")
        y = _call(d, "silu")
        assert bool(torch.isnan(y[1]).all()) and not bool(torch.isfinite(y[3]).any())
        keep = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(y[keep].view(torch.int16), clean[keep].view(torch.int16))


def test_neighbouring_memory_is_left_alone(cuda):
    """The C entry points write rows of n values and nothing between or behind them."""
    import torch
    ext = wf("_ext")
    for m, n, k, ld in ((5, 72, 64, 80), (130, 70, 64, 77), (300, 264, 128, 272), (2000, 1000, 64, 1008), (2000, 1001, 64, 1003)):
        x = torch.ones((m, k), device="cuda", dtype=torch.bfloat16)
        w = torch.ones((n, k), device="cuda", dtype=torch.bfloat16)
        dy = torch.ones((m, n), device="cuda", dtype=torch.bfloat16)
        y = torch.full((m + 3, ld), -7.0, device="cuda", dtype=torch.bfloat16)
        z = torch.full((m + 3, ld), -7.0, device="cuda", dtype=torch.float16)
        dense_cabi.launch("wf_linear", dense_cabi.LINEAR_ARGS.pack(x.data_ptr(), w.data_ptr(), 0, 0, 0, y.data_ptr(), z.data_ptr(), k, k, 0,
                                                     ld, ld, 1, m, n, k, 1, 1, 0, 0))
        for t in (y, z):
            assert bool((t[:m, :n] == k).all()) and bool((t[:m, n:] == -7).all()) and bool((t[m:] == -7).all())
        dx = torch.full((m + 3, k + 8), -7.0, device="cuda", dtype=torch.bfloat16)
        dw = torch.full((n + 3, k + 8), -7.0, device="cuda", dtype=torch.bfloat16)
        db = torch.full((n + 8,), -7.0, device="cuda", dtype=torch.bfloat16)
        size = ext.lib().wf_linear_backward_workspace(m, n, m)
        work = torch.full((size + 64,), 113, device="cuda", dtype=torch.uint8)
        dense_cabi.launch("wf_linear_backward", dense_cabi.LINEAR_GRAD_ARGS.pack(
            dy.data_ptr(), x.data_ptr(), w.data_ptr(), 0, 0, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), 0, work.data_ptr(), n,
            k, k, 0, k + 8, k + 8, m, size, m, n, k, 0, 1, 0, 0))
        assert bool((work[size:] == 113).all())
        n16, m16 = (float(torch.tensor(float(v)).to(torch.bfloat16)) for v in (n, m))
        assert bool((dx[:m, :k] == n16).all()) and bool((dx[:m, k:] == -7).all()) and bool((dx[m:] == -7).all())
        assert bool((dw[:n, :k] == m16).all()) and bool((dw[:n, k:] == -7).all()) and bool((dw[n:] == -7).all())
        assert bool((db[:n] == m16).all()) and bool((db[n:] == -7).all())


@pytest.mark.parametrize("m,k,n", [(1, 512, 2048), (5, 72, 61), (300, 1024, 520), (700, 64, 1001), (3000, 256, 1280), (5001, 72, 2048)])
def test_output_over_residual(cuda, m, k, n):
    """y may be resid: the bits of a call with an output of its own."""
    import torch
    d, _ = _data(torch, m, k, n, torch.bfloat16, groups=1)
    want = _call(d, "gelu")
    y = d["residual"].clone()
    dense_cabi.launch("wf_linear", dense_cabi.LINEAR_ARGS.pack(
        d["x"].data_ptr(), d["weight"].data_ptr(), d["bias"].data_ptr(), d["gate"].data_ptr(), y.data_ptr(), y.data_ptr(), 0, k, k, n,
        n, n, m, m, n, k, 3, 1, 0, 0))
    assert torch.equal(y, want)


def test_streams_graphs_and_repeats(cuda):
    """A side stream, a captured training step replayed on new values, and a second run give the same bits."""
    import torch
    for m, k, n in ((1, 256, 384), (100, 264, 520), (700, 512, 768)):
        d, dy = _data(torch, m, k, n, torch.bfloat16, groups=1)
        y0, g0 = _train(torch, d, "gelu", dy)
        y1, g1 = _train(torch, d, "gelu", dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2, g2 = _train(torch, d, "gelu", dy)
        torch.cuda.synchronize()
        leaves = {nm: t.detach().clone().mul_(0.5) for nm, t in d.items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y3, g3 = _train(torch, leaves, "gelu", dy)
        with torch.no_grad():
            for nm, t in d.items():
                leaves[nm].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for y, g in ((y1, g1), (y2, g2), (y3, g3)):
            assert torch.equal(y.detach().view(torch.int16), y0.detach().view(torch.int16))
            for nm in g0:
                assert torch.equal(g[nm].view(torch.int16), g0[nm].view(torch.int16)), nm
    assert wf("enhancers.fused_linear").status() == 0


def test_second_derivative_is_refused(cuda):
    import torch
    d, dy = _data(torch, 4, 16, 16, torch.bfloat16)
    d["x"].requires_grad_(True)
    (gx,) = torch.autograd.grad(_call(d, "gelu"), d["x"], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
