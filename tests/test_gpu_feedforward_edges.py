"""The linear layers of a feed-forward block where types, sizes and rules end, against 64 bits."""

import pytest
import torch

import feedforward_ref as ref
from conftest import bits_equal
from test_gpu_feedforward import BF, DEV, F16, F32, K, _on_lines, _pair, _randn, _takes, bands, without_bands  # noqa: F401  (bands: every output between sentinels)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ gradients in f16
def _f16_grads(dh, x, w, p, name):
    """(dx, tolerance, dw, tolerance) as feedforward_ref.gated_grads derives them, but for dP, which f16 holds by rows for dx and by columns for dw: scaled so
    that the largest of a row (column) lies in [2^14, 2^15), an element is off by 2^-11 of itself or half a step of the subnormals, 2^-25, which is
    2^-39 of the largest."""
    dh, x, w, p = dh.double(), x.double(), w.double(), p.double()
    F = w.shape[0] // 2
    g, u = p[:, :F], p[:, F:]
    a, s = ref.act(g, name), ref.slope(g, name)
    dp = torch.cat([dh * u * s, dh * a], 1)
    fn = torch.cat([2.0**-18 * dh.abs() * u.abs() * (1 + g.abs().clamp(max=30)), ref.act_error(g, name, F16) * dh.abs() * a.abs()], 1)
    ddp = ref.U[F16] * dp.abs() + fn
    by_row, by_col = (ddp + 2.0**-39 * dp.abs().amax(d, keepdim=True) for d in (1, 0))
    dx, dw = dp @ w, dp.t() @ x
    tx = ref.U[F16] * dx.abs() + by_row @ w.abs() + ref.sum_error(2 * F, F16) * (dp.abs() @ w.abs())
    tw = ref.U[F16] * dw.abs() + by_col.t() @ x.abs() + ref.sum_error(x.shape[0], F16) * (dp.abs().t() @ x.abs())
    return dx, 1.001 * tx + ref.TINY[F16], dw, 1.001 * tw + ref.TINY[F16]


def _spread(n, low, high):
    return torch.logspace(low, high, n, base=2.0, device=DEV).unsqueeze(1)


F16_SIZES = [(1, 64, 8), (5, 64, 24), (70, 136, 72), (64, 2048, 700), (130, 1000, 520), (300, 267, 333), (777, 520, 1003), (40, 60, 4000)]


@pytest.mark.parametrize("size", F16_SIZES, ids=str)
@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
def test_gradients_in_f16_where_those_of_the_projections_leave_its_range(size, name):
    """dP of up to 2^22, where f16 ends at 65504, and of 2^-30, where it ends at 2^-24, with operands that bring both gradients back."""
    M, k, F = size
    # large: up projections of 2^12, gradients of 2^-6 to 2^6 from row to row; w and x take 2^-12 of it back
    dh = (_randn(M, F, dtype=F32, seed=3) * _spread(M, -6, 6)).half()
    p = torch.cat([_randn(M, F, dtype=F32, seed=4), _randn(M, F, dtype=F32, seed=5) * 2.0**12], 1)
    x, w = _randn(M, k, dtype=F16, std=2.0**-12, seed=1), _randn(2 * F, k, dtype=F16, std=2.0**-12, seed=2)
    for what, xs, ws in (("rows", x, w), ("turned", x.t().contiguous().t(), w.t().contiguous().t())):
        dx, tx, dw, tw = _f16_grads(dh, x, w, p, name)
        assert dx.abs().max() < 65504 and dw.abs().max() < 65504
        gx, gw = K.gated_linear_backward(dh, xs, ws, p, name)
        ref.assert_within(gx, dx, tx, f"large, {what}: dx")
        ref.assert_within(gw, dw, tw, f"large, {what}: dw")
        assert bits_equal(K.gated_linear_backward(dh, xs, ws, p, name, [True, False])[0], gx) and bits_equal(K.gated_linear_backward(dh, xs, ws, p, name, [False, True])[1], gw)
    # small: projections of 2^-12, gradients of 2^-12 to 2^-4; w and x bring it back by 2^14
    dh = (_randn(M, F, dtype=F32, seed=3) * _spread(M, -12, -4)).half()
    p = _randn(M, 2 * F, dtype=F32, seed=4) * 2.0**-12
    x, w = _randn(M, k, dtype=F16, std=2.0**8, seed=1), _randn(2 * F, k, dtype=F16, std=2.0**8, seed=2)
    dx, tx, dw, tw = _f16_grads(dh, x, w, p, name)
    gx, gw = K.gated_linear_backward(dh, x, w, p, name)
    ref.assert_within(gx, dx, tx, "small: dx")
    ref.assert_within(gw, dw, tw, "small: dw")


def test_what_is_not_finite_in_f16_gradients_stays_in_its_rows_and_columns():
    M, k, F = 200, 264, 304
    x, w = _pair(M, k, F, F16)
    dh = _randn(M, F, dtype=F16, seed=3)
    _, p = K.gated_linear_train(x, w)
    cx, cw = K.gated_linear_backward(dh, x, w, p)
    dh[7] = 0.0
    dh[33, 20], dh[50, 9] = float("inf"), float("nan")
    gx, gw = K.gated_linear_backward(dh, x, w, p)
    rows, ups = [i for i in range(M) if i not in (7, 33, 50)], [i for i in range(2 * F) if i % F not in (9, 20)]
    assert not gx[[33, 50]].isfinite().any() and not gx[7].any() and bits_equal(gx[rows], cx[rows])
    assert not gw[[9, 20, F + 9, F + 20]].isfinite().any() and gw[ups].isfinite().all()


@without_bands
def test_f16_gradients_captured_and_replayed():
    """Two graphs of the same call, replayed with new contents of other magnitudes: the maxima are found anew."""
    M, k, F = 150, 200, 96
    x, w = _pair(M, k, F, F16)
    dh, p = _randn(M, F, dtype=F16, seed=3), _randn(M, 2 * F, dtype=F32, seed=4)
    K.gated_linear_backward(dh, x, w, p)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = K.gated_linear_backward(dh, x, w, p)
        graphs.append((g, out))
    for step in (12, -12, 0):
        p.copy_(_randn(M, 2 * F, dtype=F32, seed=10 + step) * 2.0**step)
        want = K.gated_linear_backward(dh, x, w, p)
        for g, out in graphs:
            g.replay()
            assert all(bits_equal(a, b) for a, b in zip(out, want)), step


# ------------------------------------------------------------------ where the exponential of a gate leaves fp32
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "sigmoid"])
def test_gates_whose_exponential_is_at_the_end_of_fp32(name, dtype):
    """e^-y between 2^116 and 2^148: 1 + e^-y passes 2^126 (where a fast quotient ends) and 2^128, the activation is 2^-148 or more all
    the same, and an up projection of 2^100 brings it back. Beside the relative errors, e^y is off by two steps of the subnormals at
    most, 2^-148, where it is one."""
    g = torch.arange(-10.625, -9.5, 1 / 16) if name == "gelu_tanh" else torch.arange(-102.0, -80.0, 0.5)
    n = g.numel()
    up = 2.0**100
    for M, k in ((2, 64), (300, 64), (128, 1024)):
        F = 256
        g64 = g.double().to(DEV).repeat((F + n - 1) // n)[:F]
        x = torch.zeros(M, k, device=DEV, dtype=dtype)
        x[:, 0] = 1
        w = torch.zeros(2 * F, k, device=DEV, dtype=dtype)
        w[:F, 0], w[F:, 0] = g64.to(dtype), up
        want = ref.act(g64, name) * up
        tol = (ref.U[dtype] + ref.act_error(g64, name, dtype)) * want.abs() + 2.0**-148 * (1 + g64.abs()) * up
        assert want.abs().min() > 2.0**-48
        for h in (K.gated_linear(x, w, name), K.gated_linear_train(x, w, name)[0]):
            ref.assert_within(h, want.expand(M, F), 1.001 * tol.expand(M, F), f"{M} rows")
    # the slope, by a weight that hands dP on as it is: dx = [dh u act'(g) | dh act(g)]
    g64 = g.double().to(DEV)
    p = torch.stack([g64, torch.ones_like(g64)], 1).float()
    dh = torch.full((n, 1), up, device=DEV, dtype=dtype)
    dx, _ = K.gated_linear_backward(dh, torch.zeros(n, 2, device=DEV, dtype=dtype), torch.eye(2, device=DEV, dtype=dtype), p, name)
    for got, value in ((dx[:, 0], ref.slope(g64, name)), (dx[:, 1], ref.act(g64, name))):
        # a slope has another factor of up to 1 + 1.6 |g| (1 + 0.14 g^2), of a dozen roundings
        tol = (ref.U[dtype] + ref.act_error(g64, name, dtype) + 16 * 2.0**-24) * value.abs() + 2.0**-148 * (1 + 1.6 * g64.abs() * (1 + 0.14 * g64.square()))
        ref.assert_within(got, value * up, 1.001 * tol * up, "dP")
