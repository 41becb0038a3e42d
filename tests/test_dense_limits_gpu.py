"""The dense linear layer and layer norm where calls meet limits: more than 2^31 values, allocations that fail, arguments
that are one tensor, changed saved tensors, several threads at once."""

import math
import threading

import pytest

from conftest import wf
from dense_reference import assert_within, linear_reference, norm_reference

pytestmark = pytest.mark.gpu


def _normal(torch, *shape, s=1.0, dtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(shape, device="cuda", generator=g, dtype=dtype or torch.bfloat16) * s


def test_linear_of_more_than_2_31_outputs(cuda):
    import torch
    m, k, n = 70_001, 64, 32_776
    x, w, b = _normal(torch, m, k), _normal(torch, n, k, s=1 / math.sqrt(k)), _normal(torch, n)
    dy = _normal(torch, m, n)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = wf("enhancers.fused_linear").linear(x, w, b, "gelu_tanh")
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    rows = torch.tensor([0, 1, 40_000, 65_519, 65_520, 65_536, m - 257, m - 1], device="cuda")  # 2^31 lies in row 65520
    want = linear_reference(x[rows], w, b, "gelu_tanh", None, None, 1, dy[rows])
    assert_within(y[rows].detach(), want["y"], "y")
    assert_within(dx[rows], want["x"], "x")
    cols = torch.tensor([0, 255, 256, n - 9, n - 1], device="cuda")
    want = linear_reference(x, w[cols], b[cols], "gelu_tanh", None, None, 1, dy[:, cols])
    assert_within(dw[cols], want["weight"], "weight")
    assert_within(db[cols], want["bias"], "bias")


@pytest.mark.parametrize("m,d", [(1_060_001, 2048), (2_160_001, 1001), (8_600_001, 250), (8_400_001, 256), (270_001, 8200)])
def test_layer_norm_of_more_than_2_31_values(cuda, m, d):
    import torch
    x, dy, w, b = _normal(torch, m, d), _normal(torch, m, d, seed=1), _normal(torch, d), _normal(torch, d, seed=1)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = wf("enhancers.fused_norm").layer_norm(*leaves)
    dx, _, _ = torch.autograd.grad(y, leaves, dy)
    split = 2 ** 31 // d
    rows = torch.tensor([0, 1, m // 2, split - 1, split, split + 1, m - 2, m - 1], device="cuda")
    want = norm_reference(x[rows], w.view(1, -1), b.view(1, -1), 1e-6, m, dy[rows])
    assert_within(y[rows].detach(), want["y"], "y")
    assert_within(dx[rows], want["x"], "x")


def test_failed_allocation_keeps_its_type(cuda):
    """An output of 16 TB: the allocator's own error, and the next call works."""
    import torch
    linear = wf("enhancers.fused_linear").linear
    x, w = _normal(torch, 1, 16), _normal(torch, 65_536, 16)
    with pytest.raises(torch.OutOfMemoryError):
        linear(x.expand(1 << 27, 16), w)
    with pytest.raises(torch.OutOfMemoryError):
        wf("enhancers.fused_norm").layer_norm(x.expand(1 << 39, 16))
    assert_within(linear(x, w), linear_reference(x, w, None, "none", None, None, 1)["y"], "y")


def test_one_tensor_for_several_arguments(cuda):
    import torch
    x = _normal(torch, 72, 72)
    want = linear_reference(x, x, x[0], "silu", x, x[:1], 72, x)
    a = x.clone().requires_grad_()
    y = wf("enhancers.fused_linear").linear(a, a, a[0], "silu", a, a[:1])
    assert_within(y.detach(), want["y"], "y")
    got, = torch.autograd.grad(y, a, x)
    # PyTorch adds the five gradients in bfloat16: a rounding each
    value, bound = (want["x"][i] + want["weight"][i] + want["residual"][i] for i in (0, 1))
    size = sum(want[nm][0].abs() + want[nm][1] for nm in ("x", "weight", "residual"))
    for nm in ("bias", "gate"):
        value[0] += want[nm][0].reshape(-1)
        bound[0] += want[nm][1].reshape(-1)
        size[0] += want[nm][0].reshape(-1).abs() + want[nm][1].reshape(-1)
    assert_within(got, (value, bound + 5 * size * torch.finfo(torch.bfloat16).eps / 2 * 1.02), "all")


def test_changed_saved_tensors_are_noticed(cuda):
    import torch
    linear, norm = wf("enhancers.fused_linear").linear, wf("enhancers.fused_norm").layer_norm
    for call, saved in ((lambda x, p: linear(x, p), "p"), (lambda x, p: linear(x, p, None, "gelu"), "x"),
                        (lambda x, p: linear(x, x.detach(), None, "none", None, p[0]), "p"),
                        (lambda x, p: norm(x, p[0]), "p"), (lambda x, p: norm(x, p[0]), "x")):
        x, p = _normal(torch, 64, 64).requires_grad_(), _normal(torch, 64, 64, seed=1).requires_grad_()
        y = call(x, p)
        with torch.no_grad():
            (x if saved == "x" else p).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_threads_and_streams_at_once(cuda):
    """Four threads, each on a stream of its own, train the same layers: the bits of one thread alone."""
    import torch
    linear, norm = wf("enhancers.fused_linear").linear, wf("enhancers.fused_norm").layer_norm
    shapes = [(300, 264), (40, 1024), (513, 520), (2, 61)]
    params = {k: (_normal(torch, k), _normal(torch, k), _normal(torch, 300, k, s=0.1), _normal(torch, 300)) for _, k in shapes}

    def step(i):
        m, k = shapes[i]
        w, b, weight, bias = (t.detach().requires_grad_() for t in params[k])
        x = _normal(torch, m, k, seed=7).requires_grad_()
        y = linear(norm(x, w, b), weight, bias, "gelu")
        return [y.detach(), *torch.autograd.grad(y, (x, w, b, weight, bias), torch.ones_like(y))]

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = step(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
