"""What the dense linear layer keeps for its backward pass (the pre-activation z), through the C entry points: every way
in which y and z leave the kernels."""

import math

import pytest

import dense_cabi
from conftest import wf
from dense_reference import U, act, assert_within, half_step

pytestmark = pytest.mark.gpu

ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
CODE = {"float16": 0, "bfloat16": 1, "float32": 2}


def _forward(torch, x, w, kind, z_type, ldy, ldz):
    """(y, z) of x w^T with row pitches ldy and ldz."""
    m, k = x.shape
    n = w.shape[0]
    y = torch.full((m, ldy), -7.0, device="cuda", dtype=x.dtype)
    z = torch.full((m, ldz), -7.0, device="cuda", dtype=z_type)
    code = CODE[str(x.dtype).rsplit(".", 1)[1]]
    dense_cabi.launch("wf_linear", dense_cabi.LINEAR_ARGS.pack(
        x.data_ptr(), w.data_ptr(), 0, 0, 0, y.data_ptr(), z.data_ptr(), k, k, 0, ldy, ldz, 1, m, n, k, ACT[kind], code,
        CODE[str(z_type).rsplit(".", 1)[1]], 0))
    return y, z


@pytest.mark.parametrize("m,n,k", [(5001, 2041, 72), (5001, 2048, 72), (300, 1001, 520), (3, 61, 64)])
@pytest.mark.parametrize("kind,z_name", [("gelu", "float16"), ("gelu", "float32"), ("none", "bfloat16")])
def test_kept_values_in_every_layout(cuda, m, n, k, kind, z_name):
    """y and z each at a pitch of 16-byte pieces and at an odd one: z within a rounding of its definition, y within the
    float32 sums' error and a rounding, and the same bits in every repeat (several tiles a block, so that each buffer of an
    epilogue warp is used again)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = torch.randn((m, k), device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn((n, k), device="cuda", generator=g) / math.sqrt(k)).to(torch.bfloat16)
    z_type = getattr(torch, z_name)
    want = x.double() @ w.double().t()
    e = 2 * U * k * (x.double().abs() @ w.double().abs().t())
    h, _ = act(want, kind)
    # 1.13 is the steepest slope of gelu; 8e-6 and 2e-7 its own float32 evaluation
    ey = 1.13 * e + 8e-6 * h.abs() + 2e-7 * want.abs() + half_step(h, x.dtype) * (1 + 1e-3)
    ez = e + half_step(want, z_type) * (1 + 1e-3)
    up = (n + 7) // 8 * 8
    for ldy, ldz in ((up, up), (up, up + 3), (up + 3, up), (up + 3, up + 3)):
        first = None
        for _ in range(4):
            y, z = _forward(torch, x, w, kind, z_type, ldy, ldz)
            if first is None:
                first = y, z
                assert_within(y[:, :n], (h, ey), f"y {ldy} {ldz}")
                assert_within(z[:, :n], (want, ez), f"z {ldy} {ldz}")
            else:
                assert torch.equal(y[:, :n], first[0][:, :n]) and torch.equal(z[:, :n], first[1][:, :n]), (ldy, ldz)
    assert wf("enhancers.fused_linear").status() == 0


def _exact_step(torch, dtype, kind, m, k, n, xs, ws, ds):
    """A training step on small integers times powers of two (x: xs, weight: ws, dy: ds), whose products and sums float32 holds
    exactly: (z, dy, dx, dw) in float64 for a slope that is 1 above 0, 0 below, and half of both at 0 but for relu; and the
    step's own dx and dw."""
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def integers(*shape, s):
        return (torch.randint(-3, 4, shape, device="cuda", generator=g) * s).to(dtype)
    x, w, dy = integers(m, k, s=xs).requires_grad_(), integers(n, k, s=ws).requires_grad_(), integers(m, n, s=ds)
    y = wf("enhancers.fused_linear").linear(x, w, activation=kind)
    got = torch.autograd.grad(y, (x, w), dy)
    x, w, dy = x.detach().double(), w.detach().double(), dy.double()
    z = x @ w.t()
    dz = dy * torch.where(z > 0, 1.0, torch.where(z < 0, 0.0, 0.0 if kind == "relu" else 0.5)).double()
    return z, (dz @ w, dz.t() @ x), got


@pytest.mark.parametrize("m,n", [(24, 512), (300, 61), (3000, 2048), (3000, 2041)])
def test_relu_of_small_values(cuda, m, n):
    """z of a few steps of 2^-40, far below what f16 holds: the slope is 1 wherever z is above 0."""
    import torch
    z, want, got = _exact_step(torch, torch.bfloat16, "relu", m, 72, n, 2.0 ** -20, 2.0 ** -20, 1.0)
    assert bool((z.abs() < 2.0 ** -25).all())
    for nm, a, b in zip(("dx", "dw"), got, want):
        assert torch.equal(a, b.to(torch.bfloat16)), nm


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,n", [(24, 512), (300, 61), (3000, 2048), (3000, 2041)])
def test_f16_values_past_its_range(cuda, kind, m, n):
    """An f16 layer whose z are multiples of 2^13, most of them past 65504: the slopes are 0 and 1 out there (1/2 at 0), and
    the gradients finite."""
    import torch
    z, want, got = _exact_step(torch, torch.float16, kind, m, 72, n, 2.0 ** 8, 2.0 ** 5, 2.0 ** -8)
    assert bool((z > 65504).any()) and bool((z < -65504).any())
    for nm, a, b in zip(("dx", "dw"), got, want):
        assert torch.equal(a, b.to(torch.float16)), nm


@pytest.mark.parametrize("m,n", [(24, 512), (300, 61), (3000, 2048), (3000, 2041)])
def test_f16_relu_of_small_values(cuda, m, n):
    """z of a few steps of 2^-28 in an f16 layer, which itself rounds most of them to 0: their slope is 1 all the same."""
    import torch
    z, want, got = _exact_step(torch, torch.float16, "relu", m, 72, n, 2.0 ** -14, 2.0 ** -14, 1.0)
    assert bool((z[z > 0] <= 2.0 ** -25).any())
    for nm, a, b in zip(("dx", "dw"), got, want):
        assert torch.equal(a, b.to(torch.float16)), nm


def test_nan_stays_nan(cuda):
    """A NaN on the way into z is one in the gradient of its row and of its inputs' column, for every smooth slope."""
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        for m, n in ((24, 512), (3000, 2048)):
            for kind in ("silu", "gelu", "gelu_tanh"):
                x = torch.ones((m, 72), device="cuda", dtype=dtype)
                x[5, 3] = float("nan")
                w = torch.ones((n, 72), device="cuda", dtype=dtype)
                x.requires_grad_(), w.requires_grad_()
                y = wf("enhancers.fused_linear").linear(x, w, activation=kind)
                dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
                assert bool(torch.isnan(dx[5]).all()) and bool(torch.isfinite(dx[6]).all()) and bool(torch.isnan(dw).all())


@pytest.mark.parametrize("m,n", [(24, 512), (300, 61), (3000, 2048), (3000, 2041)])
def test_f16_gate_of_values_past_its_range(cuda, m, n):
    """residual + gate * z is finite where z is not, in f16: so is the gate's gradient, the sum of dy z, and rows of dy = 0
    count nothing in it."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def integers(*shape, s):
        return (torch.randint(-3, 4, shape, device="cuda", generator=g) * s).half()
    x, w, dy = integers(m, 72, s=2.0 ** 8), integers(n, 72, s=2.0 ** 5), integers(m, n, s=2.0 ** -12)
    dy[m // 2:] = 0
    residual = integers(m, n, s=1.0)
    gate = torch.full((n,), 2.0 ** -10, device="cuda", dtype=torch.float16, requires_grad=True)
    y = wf("enhancers.fused_linear").linear(x, w, residual=residual, gate=gate)
    dg, = torch.autograd.grad(y, gate, dy)
    z = x.double() @ w.double().t()
    assert bool((z.abs() > 65504).any()) and bool(torch.isfinite(y).all())
    assert torch.equal(dg, (dy.double() * z).sum(0).half())  # the float32 sums are exact: multiples of 2, below 2^25


@pytest.mark.parametrize("m,n,k", [(5001, 2041, 72), (5001, 2044, 72), (700, 61, 64), (3, 61, 64)])
def test_columns_behind_the_rows_are_left_alone(cuda, m, n, k):
    """Widths that are no multiple of 8 at pitches that are: y, z past its next multiple of 8, dx and dw write nothing else."""
    import torch
    x = torch.ones((m, k), device="cuda", dtype=torch.bfloat16)
    w = torch.ones((n, k), device="cuda", dtype=torch.bfloat16)
    up = (n + 7) // 8 * 8
    for ld in (up, up + 8, up + 64):
        for z_type in (torch.float16, torch.float32):
            y, z = _forward(torch, x, w, "relu", z_type, ld, ld)
            assert bool((y[:, :n] == k).all()) and bool((y[:, n:] == -7).all()), ld
            assert bool((z[:, :n] == k).all()) and bool((z[:, n if ld > up else up:] == -7).all()), ld
        # a product of m x n and n x k with the widths' parts exchanged: dx [m, n] = dy [m, k] w [k, n], dw [k, n]
        xw = torch.ones((m, up), device="cuda", dtype=torch.bfloat16)
        wk = torch.ones((k, up), device="cuda", dtype=torch.bfloat16)
        dx = torch.full((m, ld), -7.0, device="cuda", dtype=torch.bfloat16)
        dw = torch.full((k, ld), -7.0, device="cuda", dtype=torch.bfloat16)
        size = wf("_ext").lib().wf_linear_backward_workspace(m, k, m)
        work = torch.empty((size,), device="cuda", dtype=torch.uint8)
        dense_cabi.launch("wf_linear_backward", dense_cabi.LINEAR_GRAD_ARGS.pack(
            x.data_ptr(), xw.data_ptr(), wk.data_ptr(), 0, 0, dx.data_ptr(), dw.data_ptr(), 0, 0, work.data_ptr(), k, up, up, 0, ld,
            ld, m, size, m, k, n, 0, 1, 0, 0))
        assert bool((dx[:, :n] == k).all()) and bool((dx[:, n:] == -7).all()), ld
        assert bool((dw[:, :n] == float(torch.tensor(float(m)).bfloat16())).all()) and bool((dw[:, n:] == -7).all()), ld
