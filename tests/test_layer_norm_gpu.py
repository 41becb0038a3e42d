"""Layer norm (enhancers/fused_norm.py): outputs and gradients against float64 within derived bounds, over widths, types,
groups and layouts."""

import pytest

import dense_cabi
from conftest import wf
from dense_reference import assert_within, norm_reference

pytestmark = pytest.mark.gpu

WIDTHS = [1, 2, 7, 8, 31, 40, 255, 256, 257, 264, 1000, 1001, 1024, 2048, 2056, 5120, 8192, 8200, 12289, 16384, 20480, 33000]


def _data(torch, m, d, dtype, wdtype, groups=1, offset=0.5, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * m + d)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)
    x = (normal(m, d) * torch.exp(normal(d)) + offset).to(dtype)
    w = (1 + 0.3 * normal(groups, d)).to(wdtype) if groups else None
    b = (0.3 * normal(groups, d)).to(wdtype) if groups else None
    return {"x": x, "weight": w, "bias": b}, normal(m, d).to(dtype)


def _train(torch, d, dy, eps=1e-6, rpg=None):
    names = [nm for nm, t in d.items() if t is not None]
    for nm in names:
        d[nm].requires_grad_(True)
    y = wf("enhancers.fused_norm").layer_norm(d["x"], d["weight"], d["bias"], eps, rpg)
    return y, dict(zip(names, torch.autograd.grad(y, [d[nm] for nm in names], dy)))


def _compare(torch, d, dy, eps=1e-6, rpg=None):
    m = d["x"].shape[0]
    groups = 1 if d["weight"] is None else d["weight"].shape[0]
    want = norm_reference(d["x"], d["weight"], d["bias"], eps, rpg or max(1, m // groups), dy)
    with torch.no_grad():
        plain = wf("enhancers.fused_norm").layer_norm(d["x"], d["weight"], d["bias"], eps, rpg)
    y, grads = _train(torch, d, dy, eps, rpg)
    assert torch.equal(plain, y.detach())
    for nm, got in {"y": y.detach(), **grads}.items():
        assert_within(got, want[nm], nm)


@pytest.mark.parametrize("d", WIDTHS)
def test_widths(cuda, d):
    import torch
    for m, dtype, wdtype in ((1, torch.bfloat16, torch.bfloat16), (37, torch.float16, torch.float32),
                             (9, torch.float32, torch.float32), (19, torch.bfloat16, torch.float32)):
        _compare(torch, *_data(torch, m, d, dtype, wdtype))


@pytest.mark.parametrize("m,d", [(5000, 64), (3001, 520), (700, 2048), (40000, 8), (2100, 1001), (4001, 24), (3000, 120),
                                 (650, 1000), (650, 2816), (650, 4096), (650, 5120), (650, 6144), (650, 6152), (600, 8200)])
def test_many_rows(cuda, m, d):
    import torch
    for dtype, wdtype in ((torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float16, torch.float16)):
        _compare(torch, *_data(torch, m, d, dtype, wdtype))


@pytest.mark.parametrize("m,rpg", [(12, 1), (100, 10), (100, 33), (4096, 2), (1000, 999), (257, 256), (50, 70)])
@pytest.mark.parametrize("d", [48, 1001, 1024, 17000])
def test_groups(cuda, m, rpg, d):
    import torch
    data, dy = _data(torch, m, d, torch.bfloat16, torch.bfloat16, groups=-(-m // rpg))
    _compare(torch, data, dy, rpg=rpg)


@pytest.mark.parametrize("m,rpg", [(1, 1), (300, 75), (301, 300), (64, 3)])
@pytest.mark.parametrize("d", [8193, 8200, 9999, 12288, 12296, 16383, 16384, 16391, 16392])
def test_rows_shared_by_clusters(cuda, m, rpg, d):
    import torch
    for wdtype in (torch.float16, torch.float32):
        data, dy = _data(torch, m, d, torch.float16, wdtype, groups=-(-m // rpg))
        _compare(torch, data, dy, rpg=rpg)
    _compare(torch, *_data(torch, m, d, torch.float32, torch.float32, groups=-(-m // rpg)), rpg=rpg)
    # the gradients of w and b alone take no exchange
    fn, want = wf("enhancers.fused_norm"), norm_reference(data["x"], data["weight"], data["bias"], 1e-6, rpg, dy)
    y = fn.layer_norm(data["x"].detach(), data["weight"], data["bias"], 1e-6, rpg)
    for nm, got in zip(("weight", "bias"), torch.autograd.grad(y, (data["weight"], data["bias"]), dy)):
        assert_within(got, want[nm], nm)


@pytest.mark.parametrize("d", [3, 31, 33, 63, 65, 127, 129, 250, 300, 2045, 2049, 5119, 5121, 8191, 16389, 24575, 24577])
def test_odd_widths(cuda, d):
    import torch
    for m, dtype, wdtype in ((1, torch.float32, torch.float32), (95, torch.bfloat16, torch.float32), (701, torch.float16, torch.float16),
                             (700, torch.float32, torch.float32)):
        _compare(torch, *_data(torch, m, d, dtype, wdtype))
    data, dy = _data(torch, 75, d, torch.bfloat16, torch.bfloat16, groups=8)
    _compare(torch, data, dy, rpg=10)


def test_without_weight_or_bias(cuda):
    import torch
    for d in (40, 1001, 2048):
        data, dy = _data(torch, 33, d, torch.bfloat16, torch.bfloat16)
        for drop in (("weight",), ("bias",), ("weight", "bias")):
            _compare(torch, {nm: None if nm in drop else t.detach().clone() for nm, t in data.items()}, dy)


def test_far_mean_and_constant_rows(cuda):
    """A mean a thousand spreads away costs no digits beyond the bound; a constant row gives the bias, with any eps > 0."""
    import torch
    _compare(torch, *_data(torch, 64, 1024, torch.float32, torch.float32, offset=1000.0))
    data, dy = _data(torch, 8, 512, torch.bfloat16, torch.bfloat16)
    data["x"][3] = 2.5
    y, grads = _train(torch, data, dy, eps=1e-5)
    assert torch.equal(y[3].detach(), data["bias"][0].detach())
    assert bool(torch.isfinite(grads["x"].float()).all()) and bool(torch.isfinite(grads["weight"].float()).all())


def test_nonfinite_rows_stay_in_their_rows(cuda):
    import torch
    fn = wf("enhancers.fused_norm")
    for d in (64, 1000, 2048, 17000):
        data, _ = _data(torch, 20, d, torch.bfloat16, torch.bfloat16)
        clean = fn.layer_norm(**data)
        data["x"][3, d // 2] = float("nan")
        data["x"][11, 0] = float("inf")
        y = fn.layer_norm(**data)
        assert bool(torch.isnan(y[[3, 11]]).all())
        keep = [i for i in range(20) if i not in (3, 11)]
        assert torch.equal(y[keep].view(torch.int16), clean[keep].view(torch.int16))


@pytest.mark.parametrize("d", [5, 77, 1001, 4097, 8193, 9999, 12288, 17777])
def test_nonfinite_rows_leave_their_neighbours(cuda, d):
    """A row shares its first and last 16 bytes with its neighbours where the width is odd: y and dx of other rows keep their bits."""
    import torch
    for dtype in (torch.bfloat16, torch.float32):
        data, dy = _data(torch, 23, d, dtype, dtype)
        y, grads = _train(torch, {nm: t.clone() for nm, t in data.items()}, dy)
        bad = {nm: t.clone() for nm, t in data.items()}
        bad["x"][4] = float("nan")
        bad["x"][10, -1] = float("inf")
        bad_dy = dy.clone()
        bad_dy[17, 0] = float("nan")
        y1, grads1 = _train(torch, bad, bad_dy)
        keep = [i for i in range(23) if i not in (4, 10, 17)]
        assert torch.equal(y1[keep], y[keep]) and torch.equal(y1[17], y[17])
        assert torch.equal(grads1["x"][keep], grads["x"][keep])
        assert bool(torch.isnan(y1[[4, 10]]).all()) and bool(torch.isnan(grads1["x"][[4, 17]]).all())


def test_gradients_against_differences(cuda):
    """Central differences of the definition in float64 against the gradients' inner products with a direction."""
    import torch
    data, dy = _data(torch, 24, 72, torch.float32, torch.float32, groups=3)
    want = norm_reference(data["x"], data["weight"], data["bias"], 1e-6, 8, dy)
    _, grads = _train(torch, {nm: t.clone() for nm, t in data.items()}, dy)
    g = torch.Generator(device="cuda").manual_seed(3)

    def value(shift):
        v = {nm: t.double() + shift.get(nm, 0) for nm, t in data.items()}
        rows = torch.arange(24, device="cuda") // 8
        y = torch.nn.functional.layer_norm(v["x"], (72,), None, None, 1e-6) * v["weight"][rows] + v["bias"][rows]
        return float((y * dy.double()).sum())
    for nm in data:
        way = torch.randn(data[nm].shape, device="cuda", generator=g, dtype=torch.float64)
        step = 1e-5
        slope = (value({nm: step * way}) - value({nm: -step * way})) / (2 * step)
        got = float((grads[nm].double() * way).sum())
        assert abs(got - slope) <= float((want[nm][1] * way.abs()).sum()) + 1e-6 * (1 + abs(slope)), nm


def test_layouts(cuda):
    """Leading dimensions, slices, transposes, expanded rows, unaligned starts: within the bounds of contiguous copies."""
    import torch
    fn = wf("enhancers.fused_norm")
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in (torch.bfloat16, torch.float32):
        def normal(*shape):
            return torch.randn(shape, device="cuda", generator=g).to(dtype)
        for x in (normal(4, 5, 600)[:, :, 8:520], normal(4, 5, 600)[:, 1:3, 3:515], normal(512, 30).t(), normal(512),
                  normal(5, 7, 512).transpose(0, 1), normal(1, 512).expand(6, 512), normal(6, 1024)[:, ::2]):
            w, b = normal(1024)[1:513], normal(512, 2)[:, 0]
            xa, wa, ba = (t.detach().requires_grad_(True) for t in (x, w, b))
            y = fn.layer_norm(xa, wa, ba)
            dy = normal(512, y.numel() // 512).t().reshape(y.shape)
            want = norm_reference(x.reshape(-1, 512), w.view(1, -1), b.reshape(1, -1), 1e-6, 1 << 30, dy.reshape(-1, 512))
            assert y.shape == x.shape and y.is_contiguous()
            assert_within(y.detach().reshape(-1, 512), want["y"], "y")
            dx, dw, db = torch.autograd.grad(y, (xa, wa, ba), dy)
            assert_within(dx.reshape(-1, 512), want["x"], "x")
            assert_within(dw.view(1, -1), want["weight"], "weight")
            assert_within(db.view(1, -1), want["bias"], "bias")


def test_only_what_is_needed(cuda):
    import itertools
    import torch
    for d in (48, 1024, 17000):
        data, dy = _data(torch, 60, d, torch.bfloat16, torch.float32, groups=2)
        _, full = _train(torch, {nm: t.clone() for nm, t in data.items()}, dy)
        for r in (1, 2):
            for names in itertools.combinations(data, r):
                leaves = {nm: t.clone().requires_grad_(nm in names) for nm, t in data.items()}
                wf("enhancers.fused_norm").layer_norm(**leaves).backward(dy)
                for nm, t in leaves.items():
                    assert (t.grad is not None) == (nm in names)
                    assert t.grad is None or torch.equal(t.grad, full[nm]), (names, nm)


def test_empty(cuda):
    import torch
    data, dy = _data(torch, 0, 40, torch.bfloat16, torch.float32)
    y, grads = _train(torch, data, dy)
    assert y.shape == (0, 40) and grads["x"].shape == (0, 40)
    assert not bool(grads["weight"].any()) and not bool(grads["bias"].any())


def test_neighbouring_memory_is_left_alone(cuda):
    import torch
    ext = wf("_ext")
    for m, d, ld in ((5, 48, 56), (5, 45, 47), (9, 1024, 1032), (9, 1001, 1003), (3, 17000, 17002)):
        x = torch.randn((m, d), device="cuda")
        y = torch.full((m + 2, ld), -7.0, device="cuda")
        stats = torch.full((2, m + 2), -7.0, device="cuda")
        dense_cabi.launch("wf_layer_norm", dense_cabi.LAYER_NORM_ARGS.pack(x.data_ptr(), 0, 0, y.data_ptr(), stats.data_ptr(),
                                                             stats[1].data_ptr(), d, ld, m, d, m, 1e-6, 2, 2, 0))
        assert bool((y[:m, d:] == -7).all()) and bool((y[m:] == -7).all()) and bool((stats[:, m:] == -7).all())
        dx = torch.full((m + 2, ld), -7.0, device="cuda")
        dense_cabi.launch("wf_layer_norm_backward", dense_cabi.LAYER_NORM_GRAD_ARGS.pack(
            x.data_ptr(), x.data_ptr(), 0, stats.data_ptr(), stats[1].data_ptr(), dx.data_ptr(), 0, 0, 0, d, d, ld, m, d, m, 0,
            2, 2))
        assert bool((dx[:m, d:] == -7).all()) and bool((dx[m:] == -7).all()) and not bool((dx[:m, :d] == -7).any())


@pytest.mark.parametrize("d", [5, 64, 77, 250, 1001, 2048, 5119, 5120, 8191, 8192, 9999, 12288, 17777, 33000])
def test_output_over_input(cuda, d):
    """y may be x: the bits of a call with an output of its own."""
    import torch
    for dtype, code in ((torch.float16, 0), (torch.float32, 2)):
        for m in (3, 900):
            data, _ = _data(torch, m, d, dtype, dtype)
            want = wf("enhancers.fused_norm").layer_norm(**data)
            x, w, b = data["x"], data["weight"], data["bias"]
            dense_cabi.launch("wf_layer_norm", dense_cabi.LAYER_NORM_ARGS.pack(
                x.data_ptr(), w.data_ptr(), b.data_ptr(), x.data_ptr(), 0, 0, d, d, m, d, m, 1e-6, code, code, 0))
            assert torch.equal(x, want), (dtype, m)


def test_streams_graphs_and_repeats(cuda):
    import torch
    for m, d in ((3, 64), (300, 1001), (500, 2048), (20, 17000)):
        data, dy = _data(torch, m, d, torch.bfloat16, torch.bfloat16)
        y0, g0 = _train(torch, data, dy)
        y1, g1 = _train(torch, data, dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y2, g2 = _train(torch, data, dy)
        torch.cuda.synchronize()
        leaves = {nm: t.detach().clone().mul_(0.5) for nm, t in data.items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y3, g3 = _train(torch, leaves, dy)
        with torch.no_grad():
            for nm, t in data.items():
                leaves[nm].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for y, gr in ((y1, g1), (y2, g2), (y3, g3)):
            assert torch.equal(y.detach(), y0.detach())
            for nm in g0:
                assert torch.equal(gr[nm], g0[nm]), nm
