"""The linear layers of a feed-forward block where types, sizes and rules end, against 64 bits."""

import pytest
import torch

import feedforward_ref as ref
from backendbench_b200 import _abi, feedforward, ops
from conftest import bits_equal
from test_gpu_feedforward import BF, DEV, F16, F32, K, _pair, _randn, bands, without_bands  # noqa: F401  (bands: every output between sentinels)

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


# ------------------------------------------------------------------ fp32: sizes and rules
def _check_f32(M, k, F, name="silu"):
    """Both passes elementwise and by the norm (see test_large_products_in_32_bits_are_as_exact_as_their_sums)."""
    x, w = _pair(M, k, F, F32)
    h, th, p, tp = ref.gated(x, w, name, F32)
    out, projections = K.gated_linear_train(x, w, name)
    ref.assert_within(projections, p, tp, "projections")
    ref.assert_within(out, h, th, "h")
    assert (projections.double() - p).norm() <= 1e-6 * p.norm() and (out.double() - h).norm() <= 2e-6 * h.norm()
    dh = _randn(M, F, dtype=F32, seed=3) * _spread(M, -8, 8)  # (columns of dP, which are rows of a product, hold all magnitudes)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, name, F32)
    gx, gw = K.gated_linear_backward(dh, x, w, projections, name)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dw")
    assert (gx.double() - dx).norm() <= 1e-6 * dx.norm() and (gw.double() - dw).norm() <= 1e-6 * dw.norm()


def _joint(M, k, F):
    return feedforward.lib().b200_linear_f32_grads_scratch_bytes(M, 2 * F, k) >= 0


@pytest.mark.parametrize("size", [(70, 97, 7003), (13401, 73, 71), (261, 2190, 6844), (13850, 2199, 129)], ids=str)
def test_fp32_operands_that_lie_across_long_contractions(size):
    """Contractions of more than 13,312 (eight CTAs' shared memory) are read twice where they lie across: the weight for dx, dP and x for dw; by
    products of their own and in the joint launch."""
    M, k, F = size
    assert max(M, 2 * F) > 8 * 26 * 64 and _joint(M, k, F) == (k > 2000)
    _check_f32(M, k, F)


@pytest.mark.parametrize("size", [(33, 4096, 300), (40, 2048, 1001), (57, 1030, 701), (64, 4100, 257)], ids=str)
def test_fp32_products_of_33_to_64_rows(size):
    M, k, F = size
    assert feedforward.lib().b200_linear_f32_scratch_bytes(M, 2 * F, k) > 0
    _check_f32(M, k, F, "gelu")


def test_fp32_products_take_planes_from_33_rows_and_enough_work():
    planes = lambda *a: feedforward.lib().b200_linear_f32_scratch_bytes(*a)
    assert planes(32, 4096, 4096) == planes(4096, 32, 4096) == planes(4096, 4096, 31) == planes(0, 1, 1) == 0
    assert planes(33, 4096, 4096) > 0 and planes(4096, 33, 4096) > 0 and planes(4096, 4096, 32) > 0 and planes(64, 4096, 4096) > 0
    assert planes(256, 512, 512) > 0 and planes(256, 512, 511) == 0  # 2^26 multiply-adds


@pytest.mark.parametrize("size", [(300, 700, 333), (777, 520, 1003), (583, 477, 145), (856, 237, 219), (1049, 841, 84), (1475, 570, 647)], ids=str)
def test_both_gradients_of_fp32_come_from_one_launch(size):
    """Sizes that take it, the longer contraction on either side."""
    M, k, F = size
    assert _joint(M, k, F)
    _check_f32(M, k, F)


@pytest.mark.parametrize("size", [(200, 512, 300), (2752, 640, 400)], ids=str)
def test_both_gradients_of_fp32_come_from_two_launches(size):
    M, k, F = size
    assert not _joint(M, k, F)
    _check_f32(M, k, F)


@pytest.mark.parametrize("M", [32, 33])
def test_what_a_row_of_one_large_element_leaves_of_the_others_in_fp32(M):
    """Planes (from 33 rows on) resolve an element to 2^-22 of itself or 2^-39 of its row's largest, which shows where the largest meets a
    zero; the products below keep every element to 2^-22. (The largest is scaled to 2^14 at least, where both planes end in steps of 2^-24: half
    a step is 2^-25 = 2^-39 * 2^14. Rows whose largest is a power of two, as here, are those that come to 2^14.)"""
    k, F = 2048, 512
    x, w = torch.zeros(M, k, device=DEV), torch.zeros(2 * F, k, device=DEV)
    large = 2.0 ** torch.arange(M, device=DEV, dtype=torch.float64) * 2.0**10  # beside 1.2345..: 2^10 to 2^42
    x[:, 0], x[:, 1] = large.float(), 1.2345678
    w[:, 1] = 0.7654321
    _, p = K.gated_linear_train(x, w, "relu")
    want = (x.double() @ w.double().t())
    tol = 2.0**-22 * want.abs() * 3  # both operands' elements and the sum
    if M > 32:
        tol = tol + 2.0**-39 * large.unsqueeze(1) * 0.7654321
    ref.assert_within(p, want, tol, "projections")


def test_the_gates_gradient_as_a_c_entry():
    """b200_gate_backward is b200_gate_backward_rows without a gap between rows."""
    lib = feedforward.lib()
    for M, F in ((5, 24), (70, 129), (300, 1000)):
        for dtype, code in ((BF, _abi.BF16), (F16, _abi.F16), (F32, _abi.F32)):
            dh, p = _randn(M, F, dtype=dtype, seed=3), _randn(M, 2 * F, dtype=F32, seed=4)
            wide, tight = ops._new((M, 2 * F + 8), dtype, p.device), ops._new((M, 2 * F), dtype, p.device)
            assert lib.b200_gate_backward(dh.data_ptr(), p.data_ptr(), tight.data_ptr(), M, F, 1, code, ops._stream_handle()) == 0
            assert lib.b200_gate_backward_rows(dh.data_ptr(), p.data_ptr(), wide.data_ptr(), 2 * F + 8, M, F, 1, code, ops._stream_handle()) == 0
            d, g, u = dh.double(), p[:, :F].double(), p[:, F:].double()
            want = torch.cat([d * u * ref.slope(g, "gelu"), d * ref.act(g, "gelu")], 1)
            fn = 2.0**-18 if dtype != F32 else 2.0**-20
            tol = ref.U[dtype] * want.abs() + torch.cat([fn * (d * u).abs() * (1 + g.abs()), ref.act_error(g, "gelu", dtype) * (d * ref.act(g, "gelu")).abs()], 1) + ref.TINY[dtype]
            ref.assert_within(tight, want, 1.001 * tol, f"{M} x {F}")
            assert bits_equal(wide[:, : 2 * F], tight)


def _same_where_not_finite(got, want, what):
    """Infinities of the same sign, NaN where NaN, nothing else that is not finite (want is in 64 bits, which holds every finite value here)."""
    got = got.double()
    bad = ~((got == want) | (got.isnan() & want.isnan()) | (got.isfinite() & want.isfinite()))
    assert not bad.any(), f"{what}: {int(bad.sum())} differ, first {got[bad][0].item()} for {want[bad][0].item()}"


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(20, 64, 40), (300, 512, 300), (129, 1030, 1001), (64, 4100, 257), (1531, 1027, 205)], ids=str)
def test_infinities_are_those_of_the_formula(size, dtype):
    """One infinity in a row or column makes its products infinite with their signs; one that meets a zero, or another of the other sign, NaN."""
    M, k, F = size
    x, w = _pair(M, k, F, dtype)
    inf = float("inf")
    x[2, 3], x[5, 1], x[7, [4, 9]], w[7, 2], w[9, 3], w[F + 4, k - 1], w[11, 3] = inf, -inf, inf, inf, -inf, inf, 0.0
    for what, xs, ws in (("rows", x, w), ("turned", x.t().contiguous().t(), w.t().contiguous().t())):
        out, projections = K.gated_linear_train(xs, ws, "relu")
        p = x.double() @ w.double().t()
        _same_where_not_finite(projections, p, what + ": projections")
        h = ref.act(p[:, :F], "relu") * p[:, F:]
        _same_where_not_finite(out, h, what + ": h")
    x, w = _pair(M, k, F, dtype)
    dh = _randn(M, F, dtype=dtype, seed=3)
    _, projections = K.gated_linear_train(x, w)
    dh[3, 5], dh[6, 7], dh[6, 8], w[5, 2] = inf, -inf, inf, 0.0
    p = projections.double()
    dp = torch.cat([dh.double() * p[:, F:] * ref.slope(p[:, :F], "silu"), dh.double() * ref.act(p[:, :F], "silu")], 1)
    for what, xs, ws in (("rows", x, w), ("turned", x.t().contiguous().t(), w.t().contiguous().t())):
        gx, gw = K.gated_linear_backward(dh, xs, ws, projections)
        _same_where_not_finite(gx, dp @ w.double(), what + ": dx")
        _same_where_not_finite(gw, dp.t() @ x.double(), what + ": dw")


@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
def test_both_gradients_of_a_linear_layer_as_a_c_entry(dtype):
    """dx = g w and dw = g^T x of a 16-bit g as it is, both and each by itself."""
    lib, (M, J, k) = feedforward.lib(), (300, 664, 520)
    g, x, w = _randn(M, J, dtype=dtype, seed=1), _randn(M, k, dtype=dtype, seed=2), _randn(J, k, dtype=dtype, seed=3)
    need = lib.b200_linear_grads_scratch_bytes(g.data_ptr(), x.data_ptr(), w.data_ptr(), M, J, k, J, k, 1, k, 1)
    assert need >= 0
    scratch = ops._scratch(g.device, max(need, 1))
    g64, x64, w64 = g.double(), x.double(), w.double()
    want = g64 @ w64, g64.t() @ x64
    tol = [ref.U[dtype] * v.abs() + ref.sum_error(n, dtype) * m + ref.TINY[dtype] for v, n, m in zip(want, (J, M), (g64.abs() @ w64.abs(), g64.abs().t() @ x64.abs()))]
    for wanted in ((0, 1), (0,), (1,)):
        out = [ops._new(v.shape, dtype, g.device) if i in wanted else None for i, v in enumerate(want)]
        rc = lib.b200_linear_grads(
            g.data_ptr(), x.data_ptr(), w.data_ptr(), *(o.data_ptr() if o is not None else None for o in out), M, J, k, J, k, k, ops._dt(dtype),
            scratch.data_ptr(), need, ops._status(g.device).data_ptr(), ops._stream_handle(),
        )
        assert rc == 0
        for i in wanted:
            ref.assert_within(out[i], want[i], 1.001 * tol[i], ("dx", "dw")[i])
