"""The linear layers of a feed-forward block on a GPU, against 64 bits (feedforward_ref.py derives the tolerances)."""

import pytest
import torch

import feedforward_ref as ref
from backendbench_b200 import feedforward, ops
from conftest import GuardBands, bits_equal

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    import backendbench_b200.custom_ops  # noqa: F401  (registers torch.ops.b200)
K = torch.ops.b200
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def without_bands(test):
    """For tests that capture graphs or hold gigabytes."""
    test.without_bands = True
    return test


@pytest.fixture(autouse=True)
def bands(request):
    """Every output and scratch buffer between sentinel bands, checked when the test ends."""
    if not torch.cuda.is_available() or getattr(request.function, "without_bands", False):
        yield
        return
    guard = GuardBands()
    ops._allocator = guard
    try:
        yield guard
        guard.verify()
    finally:
        ops._allocator = None
    ops.check_device_status()


def _randn(*shape, dtype, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7919 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _pair(M, k, F, dtype):
    return _randn(M, k, dtype=dtype, seed=1), _randn(2 * F, k, dtype=dtype, seed=2, std=k**-0.5)


# ------------------------------------------------------------------ gated projections
SIZES = [
    (1, 64, 8), (1, 8, 1), (1, 1, 1), (2, 1000, 300), (1, 4096, 1500), (3, 17, 5), (7, 512, 80), (16, 128, 40), (17, 72, 129), (53, 2048, 704),
    (64, 640, 2368), (100, 96, 24), (127, 200, 129), (128, 256, 256), (129, 320, 64), (129, 328, 65), (130, 1000, 520), (255, 384, 130), (257, 2056, 200), (300, 64, 7),
    (512, 512, 1024), (700, 1027, 333), (1000, 4096, 96), (2048, 448, 1376),
    (4096, 320, 2104), (4096, 328, 1001), (5000, 64, 1504), (40, 11008, 1024), (60, 4096, 4096),
]


@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gated_linear_16_bits(size, dtype):
    M, k, F = size
    x, w = _pair(M, k, F, dtype)
    name = ref.ACTS[(M + k + F) % 5]
    h, th, p, tp = ref.gated(x, w, name, dtype)
    ref.assert_within(K.gated_linear(x, w, name), h, th, f"{name} h")
    out, projections = K.gated_linear_train(x, w, name)
    ref.assert_within(out, h, th, f"{name} h of the training form")
    ref.assert_within(projections, p, tp, "projections")


@pytest.mark.parametrize("name", ref.ACTS)
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
def test_every_activation_with_large_and_small_gates(name, dtype):
    """Gates from -80 to 80, up projections of 1: what saturates does so as in 64 bits."""
    F, k = 1024, 64
    x = torch.zeros(2, k, device=DEV, dtype=dtype)
    x[:, 0] = 1
    x[1, 1] = -1
    w = torch.zeros(2 * F, k, device=DEV, dtype=dtype)
    w[:F, 0] = torch.linspace(-80, 80, F, device=DEV).to(dtype)
    w[:F, 1] = torch.linspace(-1, 1, F, device=DEV).to(dtype)
    w[F:, 0] = 1
    h, th, p, _ = ref.gated(x, w, name, dtype)
    out, projections = K.gated_linear_train(x, w, name)
    ref.assert_within(out, h, th, name)
    dh = _randn(2, F, dtype=dtype)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, name, dtype)
    gx, gw = K.gated_linear_backward(dh, x, w, projections, name)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dw")


F32_LARGE = [(65, 11008, 200), (100, 2048, 512), (200, 4096, 300), (129, 1030, 1001), (2048, 1024, 1104), (1000, 64, 4000), (1531, 1027, 1365), (3000, 200, 190), (66, 4100, 3001)]


@pytest.mark.parametrize("size", [(1, 64, 8), (3, 17, 5), (130, 1000, 520), (300, 260, 301), (1531, 1027, 205)] + F32_LARGE, ids=str)
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_gated_linear_32_bits(size, name):
    M, k, F = size
    x, w = _pair(M, k, F, F32)
    h, th, p, tp = ref.gated(x, w, name, F32)
    ref.assert_within(K.gated_linear(x, w, name), h, th, "h")
    out, projections = K.gated_linear_train(x, w, name)
    ref.assert_within(projections, p, tp, "projections")
    ref.assert_within(out, h, th, "h of the training form")


@pytest.mark.parametrize("size", F32_LARGE, ids=str)
def test_large_products_in_32_bits_are_as_exact_as_their_sums(size):
    """Against 64 bits by the norm, where errors that always have one sign would show: two f16 planes are off by 2^-23 of an element or so,
    a sum rounded to nearest slab by slab by 2^-24 of what it has reached, at random: 1e-6 holds an order of magnitude."""
    M, k, F = size
    x, w = _pair(M, k, F, F32)
    x = x.abs()  # sums that grow all the way
    out, projections = K.gated_linear_train(x, w)
    h, _, p, _ = ref.gated(x, w, "silu", F32)
    assert (projections.double() - p).norm() <= 1e-6 * p.norm() and (out.double() - h).norm() <= 2e-6 * h.norm()
    dh = _randn(M, F, dtype=F32, seed=3)
    dx, _, dw, _ = ref.gated_grads(dh, x, w, projections, "silu", F32)
    gx, gw = K.gated_linear_backward(dh, x, w, projections)
    assert (gx.double() - dx).norm() <= 1e-6 * dx.norm() and (gw.double() - dw).norm() <= 1e-6 * dw.norm()


def test_rows_of_any_magnitude_in_32_bits():
    """Rows and columns from the subnormals to the largest numbers, rows of zeros, one large element in a row; what is not finite spoils its
    own row or column alone."""
    M, k, F = 300, 512, 256
    x, w = _pair(M, k, F, F32)
    x *= torch.logspace(-38, 20, M, device=DEV, dtype=F32)[:, None]
    w *= torch.logspace(-15, 10, 2 * F, device=DEV, dtype=F32)[torch.randperm(2 * F, device=DEV)][:, None]
    x[5], x[6, 1:], w[7], x[8] = 0.0, 0.0, 0.0, 1e-42
    x[9, 3], x[290] = 1e6 * x[9].abs().max(), 3.0e38 / 512**2
    w[11, 5] *= 1e4
    _, projections = K.gated_linear_train(x, w, "relu")
    _, _, p, tp = ref.gated(x, w, "relu", F32)
    fine = p.abs() < 3.0e38
    ref.assert_within(projections[fine], p[fine], tp[fine] + 2.0**-149, "projections")
    assert not projections[p.abs() > 3.5e38].isfinite().any()
    x, w = _pair(M, k, F, F32)
    _, clean = K.gated_linear_train(x, w)
    x[20, 100], x[21, 7], w[30, 9] = float("nan"), -float("inf"), float("inf")
    _, spoilt = K.gated_linear_train(x, w)
    rows, cols = [i for i in range(M) if i not in (20, 21)], [i for i in range(2 * F) if i != 30]
    assert not spoilt[[20, 21]].isfinite().any() and not spoilt[:, 30].isfinite().any()
    assert bits_equal(spoilt[rows][:, cols], clean[rows][:, cols])


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(1, 64, 8), (3, 17, 5), (64, 256, 96), (200, 512, 136), (257, 130, 77), (1024, 768, 640), (777, 520, 1001), (130, 4096, 300)], ids=str)
def test_gated_linear_backward(size, dtype):
    M, k, F = size
    x, w = _pair(M, k, F, dtype)
    name = ref.ACTS[(M + k + F) % 5]
    dh = _randn(M, F, dtype=dtype, seed=3)
    _, projections = K.gated_linear_train(x, w, name)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, name, dtype)
    gx, gw = K.gated_linear_backward(dh, x, w, projections, name)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dw")
    only = K.gated_linear_backward(dh, x, w, projections, name, [False, True])
    assert only[0] is None and bits_equal(only[1], gw)


@pytest.mark.parametrize("seed", range(6))
def test_products_of_drawn_sizes(seed):
    """Tiles of every width, clusters of every size and pairs, as the plan takes them for sizes nobody chose."""
    import random

    rng = random.Random(seed)
    for _ in range(14):
        M, k, F = (int(2 ** rng.uniform(0, top)) for top in (11, 13, 11.5))
        if rng.random() < 0.5:
            k, F = (k + 15) // 16 * 16, (F + 7) // 8 * 8
        dtype, name = rng.choice((BF, F16)), rng.choice(ref.ACTS)
        for dtype in (dtype, F32):
            x, w = _pair(M, k, F, dtype)
            h, th, p, tp = ref.gated(x, w, name, dtype)
            out, projections = K.gated_linear_train(x, w, name)
            ref.assert_within(out, h, th, f"{M} x {k} x {F}: h")
            ref.assert_within(projections, p, tp, f"{M} x {k} x {F}: projections")
        a, b = _int8(M, k), _int8(F, k, seed=1)
        _check_int8(a, b.t(), rng.choice((BF, F16, F32)), what=f"{M} x {k} x {F}: 8 bits")


def _layouts(M, k, F, dtype):
    x, w = _pair(M, k, F, dtype)
    wide = _randn(M, k + 24, dtype=dtype)
    yield "rows apart", wide[:, 8 : 8 + k], w
    yield "rows apart, off the grid", _randn(M, k + 3, dtype=dtype)[:, 1 : 1 + k], w
    yield "base off the grid", _randn(M * k + 1, dtype=dtype)[1:].view(M, k), w
    yield "x transposed", x.t().contiguous().t(), w
    yield "weight transposed", x, w.t().contiguous().t()
    yield "every second column", _randn(M, 2 * k, dtype=dtype)[:, ::2], _randn(2 * F, 2 * k, dtype=dtype, std=k**-0.5)[:, ::2]
    yield "one row for all", x[:1].expand(M, k), w
    yield "weight rows apart", x, _randn(2 * F, k + 8, dtype=dtype, std=k**-0.5)[:, :k]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(5, 64, 24), (150, 328, 72), (260, 520, 400)], ids=str)
def test_gated_linear_of_any_layout(size, dtype):
    M, k, F = size
    for what, x, w in _layouts(M, k, F, dtype):
        h, th, _, _ = ref.gated(x, w, "silu", dtype)
        ref.assert_within(K.gated_linear(x, w), h, th, what)
        out, projections = K.gated_linear_train(x, w)
        dh = _randn(M, F, dtype=dtype, seed=5).t().contiguous().t()
        dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, "silu", dtype)
        gx, gw = K.gated_linear_backward(dh, x, w, projections)
        ref.assert_within(gx, dx, tx, what + ": dx")
        ref.assert_within(gw, dw, tw, what + ": dw")


def test_gated_linear_of_more_and_fewer_dimensions():
    w = _randn(48, 40, dtype=BF, std=0.2)
    x = _randn(3, 4, 5, 40, dtype=BF)
    h = K.gated_linear(x, w)
    assert h.shape == (3, 4, 5, 24) and bits_equal(h.view(60, 24), K.gated_linear(x.view(60, 40), w))
    assert bits_equal(K.gated_linear(x.transpose(0, 2), w), h.transpose(0, 2).contiguous())
    assert bits_equal(K.gated_linear(x[0, 0, 0], w), h[0, 0, 0])
    _, projections = K.gated_linear_train(x, w)
    dx, dw = K.gated_linear_backward(h, x, w, projections)
    assert dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_gated_linear_of_nothing(dtype):
    w = _randn(16, 8, dtype=dtype)
    assert K.gated_linear(_randn(0, 8, dtype=dtype), w).shape == (0, 8)
    assert K.gated_linear(_randn(2, 0, 8, dtype=dtype), w).shape == (2, 0, 8)
    assert K.gated_linear(_randn(3, 8, dtype=dtype), w[:0]).shape == (3, 0)
    out, projections = K.gated_linear_train(torch.empty(3, 0, device=DEV, dtype=dtype), torch.empty(16, 0, device=DEV, dtype=dtype))
    assert out.shape == (3, 8) and not out.any() and projections.shape == (3, 16) and not projections.any()
    x = _randn(0, 8, dtype=dtype)
    out, projections = K.gated_linear_train(x, w)
    dx, dw = K.gated_linear_backward(out, x, w, projections)
    assert dx.shape == (0, 8) and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("M", [5, 300])
def test_a_row_that_is_not_finite_stays_by_itself(M):
    x, w = _pair(M, 512, 136, BF)
    clean = K.gated_linear(x, w)
    x[2, 7], x[4, 100] = float("nan"), float("inf")
    out = K.gated_linear(x, w)
    others = [i for i in range(M) if i not in (2, 4)]
    assert out[2].isnan().all() and not out[4].isfinite().any()
    assert bits_equal(out[others], clean[others])


def test_gradients_against_differences():
    """The gradients of a sum, in fp32, against central differences of the 64-bit formula along random directions."""
    x, w = _pair(9, 33, 14, F32)
    dh = _randn(9, 14, dtype=F32, seed=4)
    for name in ref.ACTS:
        _, projections = K.gated_linear_train(x, w, name)
        dx, dw = K.gated_linear_backward(dh, x, w, projections, name)
        loss = lambda a, b: (ref.gated(a, b, name, F32)[0] * dh.double()).sum()
        for seed in range(3):
            vx, vw, e = _randn(9, 33, dtype=F32, seed=seed).double(), _randn(28, 33, dtype=F32, seed=seed).double(), 1e-6
            want = (loss(x.double() + e * vx, w.double() + e * vw) - loss(x.double() - e * vx, w.double() - e * vw)) / (2 * e)
            have = (dx.double() * vx).sum() + (dw.double() * vw).sum()
            scale = (dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum()
            assert abs(have - want) <= 1e-5 * scale, (name, have, want)


# ------------------------------------------------------------------ dropout
def _state(seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device=DEV)


def _check_dropout(x, p, seed, offset, residual, sub):
    keep = ref.kept(tuple(x.shape), p, seed, offset, sub).to(DEV)
    scale = 1 / (1 - p) if p < 1 else 0.0
    y = torch.where(keep, x.double() * scale, 0.0)
    r = residual.double() if residual is not None else torch.zeros_like(y)
    want = y + r
    # fp32: the scale, the product and the sum are each off by half a step at most; then the rounding to the type
    tol = lambda of, terms: ref.U[x.dtype] * of.abs() + 2.0**-22 * terms + ref.TINY[x.dtype]
    ref.assert_within(K.dropout(x, p, _state(seed, offset), residual, subsequence=sub), want, tol(want, y.abs() + r.abs()), "dropout")
    ref.assert_within(K.dropout_backward(x, p, _state(seed, offset), subsequence=sub), y, tol(y, y.abs()), "its gradient")


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7,), (8,), (1, 1000), (16, 256), (129, 77), (5, 3, 33), (700, 2933)], ids=str)
def test_dropout(shape, dtype):
    x, r = _randn(*shape, dtype=dtype), _randn(*shape, dtype=dtype, seed=9)
    for i, (p, residual) in enumerate([(0.1, r), (0.5, None), (0.0, r), (0.9, r)]):
        _check_dropout(x, p, -(2**63) + 12345 * i if i % 2 else 2**62 + i, 2**35 * i + 3, residual, i * (2**33 + 1))


def test_dropout_of_everything_and_of_what_is_not_finite():
    x = _randn(64, 40, dtype=BF)
    r = _randn(64, 40, dtype=BF, seed=3)
    x[3], x[5] = float("inf"), float("nan")
    assert not K.dropout(x, 1.0, _state(1, 2)).any()
    assert bits_equal(K.dropout(x, 1.0, _state(1, 2), r), r)
    assert bits_equal(K.dropout(x, 0.0, _state(1, 2)), x)
    keep = ref.kept((64, 40), 0.5, 1, 2).to(DEV)
    y = K.dropout(x, 0.5, _state(1, 2))
    assert not y[~keep].any() and y[3][keep[3]].isinf().all() and y[5][keep[5]].isnan().all()


def test_dropout_counts_elements_in_the_order_of_the_shape():
    x = _randn(60, 44, dtype=F16)
    want = K.dropout(x, 0.3, _state(7, 9))
    assert bits_equal(K.dropout(x.t().contiguous().t(), 0.3, _state(7, 9)), want)
    assert bits_equal(K.dropout(_randn(60 * 44 + 1, dtype=F16)[1:].copy_(x.view(-1)).view(60, 44), 0.3, _state(7, 9)), want)
    wide = torch.zeros(60, 50, dtype=F16, device=DEV)
    wide[:, 3:47] = x
    assert bits_equal(K.dropout(wide[:, 3:47], 0.3, _state(7, 9), subsequence=0), want)
    assert bits_equal(K.dropout(x.view(2, 30, 44), 0.3, _state(7, 9)).view(60, 44), want)
    one = torch.ones(1, dtype=F16, device=DEV).expand(60, 44)
    assert bits_equal(K.dropout(one, 0.3, _state(7, 9)) != 0, ref.kept((60, 44), 0.3, 7, 9).to(DEV))
    strided = torch.tensor([7, 0, 9, 0], device=DEV)[::2]
    assert bits_equal(K.dropout(x, 0.3, strided), want)
    assert K.dropout(x[:0], 0.3, _state(7, 9)).shape == (0, 44)
    assert K.dropout(x[0, 0], 0.0, _state(7, 9)).shape == ()


def test_the_counter_wraps_and_subsequences_differ():
    x = torch.ones(4000, device=DEV)
    for offset in (2**32 - 3, 2**63 - 2, -2):  # across 32 bits, the sign and 64 bits
        assert bits_equal(K.dropout(x, 0.5, _state(5, offset)) != 0, ref.kept((4000,), 0.5, 5, offset).to(DEV))
    a, b = (K.dropout(x, 0.5, _state(5, 0), subsequence=s) for s in (0, 1))
    assert 1500 < int((a != b).sum()) < 2500


# ------------------------------------------------------------------ 8 bits
def _quantized(x):
    """The definition in fp32, operation by operation (every one is correctly rounded on both sides; torch takes reciprocals in
    place of quotients by or of a number, so those are formed in 64 bits and rounded once)."""
    x = x.float()
    most = x.abs().amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1], device=x.device)
    inv = torch.where(most >= 2.0**-118, (127.0 / most.double()).float(), 0.0)
    return torch.round(x * inv.unsqueeze(-1)).to(torch.int8), torch.where(most >= 2.0**-118, (most.double() / 127.0).float(), 0.0)


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 17), (5, 128), (33, 520), (64, 4104), (2, 9000), (2, 40000), (4, 11007), (2, 3, 64), (300, 8)], ids=str)
def test_quantize_rows(shape, dtype):
    x = _randn(*shape, dtype=dtype)
    x.view(-1, shape[-1])[0] *= 100
    q, scale = K.quantize_rows(x)
    want_q, want_scale = _quantized(x)
    assert torch.equal(q, want_q) and torch.equal(scale, want_scale)
    off = (q.double() * scale.double().unsqueeze(-1) - x.double()).abs()
    assert (off <= scale.double().unsqueeze(-1) * 0.50002).all()  # half a step, and what fp32 adds


def test_quantize_rows_layouts_zeros_and_what_is_not_finite():
    x = _randn(40, 96, dtype=BF)
    want = K.quantize_rows(x)
    wide = torch.zeros(40, 130, dtype=BF, device=DEV)
    for at in (8, 5):
        wide.zero_()[:, at : at + 96] = x
        got = K.quantize_rows(wide[:, at : at + 96])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = K.quantize_rows(x.t().contiguous().t())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert K.quantize_rows(x[0])[1].shape == () and torch.equal(K.quantize_rows(x[0])[0], want[0][0])
    assert K.quantize_rows(x[:0])[0].shape == (0, 96)
    q, scale = K.quantize_rows(x[:, :0])
    assert q.shape == (40, 0) and not scale.any()
    x = x.float()
    x[0], x[1, 3], x[2, 5], x[3], x[4] = 0.0, float("nan"), -float("inf"), 1e-37, torch.finfo(F32).max
    x[1, 4] = float("inf")
    q, scale = K.quantize_rows(x)
    assert not q[:4].any() and scale[0] == 0 and scale[1].isnan() and scale[2].isinf() and scale[3] == 0
    assert (q[4] == 127).all() and torch.equal(q[5:], want[0][5:])


def _int8(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def _check_int8(a, b, dtype, bias=None, what=""):
    M, N = a.shape[0], b.shape[1]
    sa, sb = _randn(M, dtype=F32, seed=1).abs() + 0.1, _randn(N, dtype=F32, seed=2) * 1e-3
    prod = (a.double() @ b.double()) * sa.double()[:, None] * sb.double()
    want = prod + (bias.double() if bias is not None else 0)
    # the sum is exact; its rounding to fp32, two products, a sum: four half steps; then the rounding to the type
    mag = prod.abs() + (bias.double().abs() if bias is not None else 0)
    tol = ref.U[dtype] * want.abs() + 2.0**-21 * mag + ref.TINY[dtype]
    ref.assert_within(K.mm_int8(a, b, sa, sb, bias, out_dtype=dtype), want, tol, what)


INT8_SIZES = [
    (1, 1, 1), (1, 16, 16), (1, 4096, 1504), (2, 17, 3), (5, 128, 16), (16, 256, 40), (33, 1000, 130), (64, 11008, 512), (100, 144, 2400), (128, 512, 256), (129, 640, 128),
    (130, 656, 129), (255, 1024, 264), (257, 1027, 515), (300, 100, 20), (1000, 2048, 96), (700, 4096, 1000), (2537, 1027, 301), (1024, 1040, 2048),
    (4096, 384, 2112), (6000, 64, 1501), (24, 8192, 3001), (300, 8192, 520),
]


@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", INT8_SIZES, ids=str)
def test_mm_int8(size, dtype):
    M, k, N = size
    a, w = _int8(M, k), _int8(N, k, seed=1)
    _check_int8(a, w.t(), dtype)
    _check_int8(a, w.t(), dtype, _randn(N, dtype=dtype), "with a bias")


def test_mm_int8_of_any_layout():
    for M, k, N in ((7, 80, 24), (200, 784, 130)):
        a, w = _int8(M, k), _int8(N, k, seed=1)
        _check_int8(a, w.t().contiguous(), BF, what="B along N")
        _check_int8(a.t().contiguous().t(), w.t(), BF, what="A along M")
        _check_int8(_int8(M, k + 16)[:, :k], _int8(N, k + 7)[:, 3 : 3 + k].t(), BF, what="rows apart")
        _check_int8(_int8(M * k + 1)[1:].view(M, k), w.t(), BF, what="base off the grid")
        _check_int8(_int8(M, 2 * k)[:, ::2], w.t(), BF, what="every second column")
        _check_int8(a[:1].expand(M, k), w[:1].expand(N, k).t(), BF, what="one row for all")
        bias = _randn(2 * N, dtype=F16)[::2]
        _check_int8(a, w.t(), F16, bias, "a strided bias")
        sa, sb = torch.rand(M, device=DEV), torch.rand(N, device=DEV)
        want = K.mm_int8(a, w.t(), sa, sb)
        assert want.dtype == BF and bits_equal(K.mm_int8(a, w.t(), sa[:, None], sb[None]), want)
        off = torch.rand(N + 1, device=DEV)[1:].copy_(sb)
        assert bits_equal(K.mm_int8(a, w.t(), sa.repeat_interleave(2)[::2], off), want)


def test_mm_int8_extremes():
    """The largest sums that 32 bits hold, both ways, and no contraction at all."""
    k = feedforward.INT8_MAX_K
    a, one = torch.full((2, k), -128, dtype=torch.int8, device=DEV), torch.ones(2, device=DEV)
    a[1, ::2] = 127
    b = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    b[1] = 127
    want = (a.double() @ b.double().t()).float()
    assert torch.equal(K.mm_int8(a, b.t(), one, torch.ones(3, device=DEV), out_dtype=F32), want)
    bias = _randn(3, dtype=F16)
    e = torch.empty(2, 0, dtype=torch.int8, device=DEV)
    assert torch.equal(K.mm_int8(e, torch.empty(0, 3, dtype=torch.int8, device=DEV), one, torch.ones(3, device=DEV), bias), bias.expand(2, 3))
    assert not K.mm_int8(e, torch.empty(0, 3, dtype=torch.int8, device=DEV), one, torch.ones(3, device=DEV)).any()
    assert K.mm_int8(a[:0], b.t(), one[:0], torch.ones(3, device=DEV)).shape == (0, 3)
    assert K.mm_int8(a, b[:0].t(), one, torch.ones(0, device=DEV)).shape == (2, 0)


def test_scales_that_are_not_finite_spoil_their_row_alone():
    x = _randn(40, 256, dtype=BF)
    w, ws = _int8(48, 256), torch.rand(48, device=DEV) + 0.1
    clean = K.mm_int8(*(lambda q, s: (q, w.t(), s, ws))(*K.quantize_rows(x)))
    x[3, 9] = float("inf")
    q, s = K.quantize_rows(x)
    out = K.mm_int8(q, w.t(), s, ws)
    assert not out[3].isfinite().any() and bits_equal(out[4:], clean[4:]) and bits_equal(out[:3], clean[:3])


# ------------------------------------------------------------------ as they are used
def _block(x, w, wd, bd, state, name, p):
    h = K.gated_linear(x, w, name)
    y = K.mm(h.view(-1, h.shape[-1]), wd.t()).view(x.shape) if not wd.requires_grad else torch.mm(h.view(-1, h.shape[-1]), wd.t()).view(x.shape)
    return K.dropout(y, p, state, x, subsequence=1)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_a_block_forward_and_backward(dtype):
    """y = x + dropout(gated(x) Wd^T) and its gradients through autograd, against the same block in 64 bits; errors are judged by the
    norm: half a dozen roundings of up to U each on the way, none amplified (all weights are of norm about 1)."""
    B, T, d, F, p = 3, 50, 192, 320, 0.2
    x, w = _randn(B, T, d, dtype=dtype).requires_grad_(), _randn(2 * F, d, dtype=dtype, std=d**-0.5).requires_grad_()
    wd, dy = _randn(d, F, dtype=dtype, std=F**-0.5).requires_grad_(), _randn(B, T, d, dtype=dtype, seed=8)
    state = _state(11, 5)
    y = _block(x, w, wd, None, state, "silu", p)
    got = torch.autograd.grad(y, (x, w, wd), dy)
    x64, w64, wd64 = (t.detach().double().requires_grad_() for t in (x, w, wd))
    pr = x64 @ w64.t()
    h = torch.nn.functional.silu(pr[..., :F]) * pr[..., F:]
    y64 = x64 + ref.kept((B, T, d), p, 11, 5, 1).to(DEV) * (h @ wd64.t()) / (1 - p)
    want = torch.autograd.grad(y64, (x64, w64, wd64), dy.double())
    for g, r in zip((y, *got), (y64, *want)):
        assert (g.double() - r).norm() <= 6 * ref.U[dtype] * r.norm() + 2.0**-20 * r.norm()


def test_gradients_flow_only_where_they_are_wanted():
    x, w = _pair(10, 64, 24, BF)
    s = _state(1, 1)
    w.requires_grad_()
    h = K.gated_linear(x, w)
    h.sum().backward()
    assert w.grad is not None and x.grad is None
    w.grad = None
    with torch.no_grad():
        assert not K.gated_linear(x, w).requires_grad
    r = torch.zeros_like(x).requires_grad_()
    y = K.dropout(x, 0.5, s, r)
    y.sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))
    x = x.requires_grad_()
    (g,) = torch.autograd.grad(K.gated_linear(x, w.detach()).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g.sum().backward()
    y = K.dropout(x, 0.5, s)
    s += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@without_bands
@pytest.mark.parametrize("name", sorted(feedforward.OPERATORS))
def test_operators_hold_up_to_torchs_own_checks(name):
    """Schema, fake kernel, autograd registration and tracing, as torch.library.opcheck looks at them."""
    x, w = _pair(4, 64, 8, BF)
    x, w, s, q, one = x.requires_grad_(), w.requires_grad_(), _state(1, 2), _int8(8, 64), torch.ones(8, device=DEV)
    plain, p = x.detach(), _randn(4, 16, dtype=F32)
    args = {
        "gated_linear": ((x, w, "gelu"), {}),
        "gated_linear_train": ((x, w), {}),
        "gated_linear_backward": ((_randn(4, 8, dtype=BF), plain, w.detach(), p, "silu", [True, False]), {}),
        "dropout": ((x, 0.3, s, x), {"subsequence": 2}),
        "dropout_backward": ((plain, 0.3, s), {}),
        "quantize_rows": ((plain,), {}),
        "mm_int8": ((q, q.t(), one, one, _randn(8, dtype=F16)), {"out_dtype": F16}),
    }[name]
    torch.library.opcheck(getattr(K, name).default, *args)


def test_gradients_of_broadcast_inputs():
    """x and its gradient's memory shared along rows: the gradient sums over them, whatever the strides say."""
    w = _randn(48, 64, dtype=F32, std=0.125)
    row = _randn(1, 64, dtype=F32).requires_grad_()
    K.gated_linear(row.expand(30, 64), w).sum().backward()  # dh: one value for all, strides of zero
    many = row.detach().repeat(30, 1).requires_grad_()
    K.gated_linear(many, w).backward(torch.ones(30, 24, device=DEV))
    assert torch.allclose(row.grad, many.grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_the_8_bit_layers_in_a_row():
    """tokens -> 8 bits -> product -> gate by mul and relu -> 8 bits -> product, each step against the 64-bit form of its own inputs."""
    x, w1, w2 = _randn(37, 512, dtype=BF), _int8(640, 512), _int8(512, 320, seed=2)
    s1, s2 = torch.rand(640, device=DEV) * 1e-3, torch.rand(512, device=DEV) * 1e-3
    q, s = K.quantize_rows(x)
    p = K.mm_int8(q, w1.t(), s, s1)
    h = K.mul(K.relu(p[:, :320]), p[:, 320:])
    q2, t = K.quantize_rows(h)
    y = K.mm_int8(q2, w2.t(), t, s2, out_dtype=F32)
    want_q, want_s = _quantized(x)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)
    want_q2, want_t = _quantized(h)
    assert torch.equal(q2, want_q2) and torch.equal(t, want_t)
    want = (q2.double() @ w2.double().t()) * t.double()[:, None] * s2.double()
    ref.assert_within(y, want, 2.0**-21 * want.abs() + 1e-37, "second product")


def _all_calls(x, w, q, w8, sa, sb, dh, state):
    h, projections = K.gated_linear_train(x, w)
    return (K.gated_linear(x, w), h, projections, *K.gated_linear_backward(dh, x, w, projections), K.dropout(x, 0.1, state, x), *K.quantize_rows(x), K.mm_int8(q, w8.t(), sa, sb))


def _all_args(M=70, k=136, F=72, odd=0, dtype=BF):
    k += odd
    x, w = _pair(M, k, F, dtype)
    return x, w, _int8(M, k), _int8(96, k), torch.rand(M, device=DEV), torch.rand(96, device=DEV), _randn(M, F, dtype=dtype), _state(3, 4)


@pytest.mark.parametrize("odd", [0, 3])
@pytest.mark.parametrize("dtype", [BF, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(70, 136, 72), (300, 600, 200)], ids=str)
def test_native_calls_give_what_the_wrappers_give(dtype, odd, size, bands):
    """With the bands' allocator in place every call goes through the wrappers; without it plain ones come from native code."""
    M, k, F = size[0], size[1] + odd, size[2]
    x, w = _pair(M, k, F, dtype)
    q, w8, sa, sb, bias = _int8(M, k), _int8(96, k), torch.rand(M, device=DEV), torch.rand(96, device=DEV), _randn(96, dtype=dtype)
    dh, s, r = _randn(M, F, dtype=dtype), _state(3, 4), _randn(M, k, dtype=dtype, seed=6)
    wide = _randn(M, k + 8, dtype=dtype)

    def calls():
        for v in (x, wide[:, :k], x.t().contiguous().t(), x.view(2, M // 2, k)):
            h, projections = K.gated_linear_train(v, w, "gelu")
            g = dh.view(h.shape)
            yield from (K.gated_linear(v, w), h, projections)
            yield from K.gated_linear_backward(g, v, w, projections, "gelu")
            yield K.gated_linear_backward(g, v, w, projections, "gelu", [True, False])[0]
            yield from (K.dropout(v, 0.3, s, r.view(v.shape), subsequence=9), K.dropout(v, 0.3, s), K.dropout_backward(v, 0.3, s, subsequence=9))
            yield from K.quantize_rows(v)
        yield from (K.mm_int8(q, w8.t(), sa, sb), K.mm_int8(q, w8.t(), sa[:, None], sb[None], bias), K.mm_int8(q, w8.t(), sa, sb, out_dtype=dtype), K.mm_int8(q, w8.t().contiguous(), sa, sb))

    want = list(calls())
    assert bands.allocations > 50
    ops._allocator = None
    count = bands.allocations
    got = list(calls())
    assert bands.allocations == count
    assert len(got) == len(want) and all(a.dtype == b.dtype and a.shape == b.shape and bits_equal(a, b) for a, b in zip(got, want))


def test_refusals_come_back_as_the_wrappers_raise_them(bands):
    ops._allocator = None
    x, w = _pair(4, 64, 8, BF)
    s, q, one = _state(1, 2), _int8(4, 64), torch.ones(4, device=DEV)
    for call, error, match in (
        (lambda: K.gated_linear(x, w, "tanh"), ValueError, "not one of"),
        (lambda: K.gated_linear(x, w[:5]), RuntimeError, "5 rows"),
        (lambda: K.gated_linear(x, w.half()), RuntimeError, "same dtype"),
        (lambda: K.gated_linear(x, w.cpu()), ops.UnsupportedByB200, "no CPU path"),
        (lambda: K.gated_linear_backward(x, x, w, x), RuntimeError, "do not go with"),
        (lambda: K.dropout(x, 2.0, s), ValueError, "between 0 and 1"),
        (lambda: K.dropout(x, 0.1, s, x[:1]), RuntimeError, "like the input"),
        (lambda: K.dropout(x, 0.1, s.cpu()), ops.UnsupportedByB200, "no CPU path"),
        (lambda: K.quantize_rows(q), ops.UnsupportedByB200, "int8"),
        (lambda: K.mm_int8(q, q.t(), one, one[:3]), RuntimeError, "fp32 values"),
        (lambda: K.mm_int8(q, q, one, one), RuntimeError, "cannot be multiplied"),
    ):
        with pytest.raises(error, match=match):
            call()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode|jvp"):
            K.gated_linear(torch.autograd.forward_ad.make_dual(x, x), w)


@pytest.mark.parametrize("args", [{}, {"odd": 3}, {"M": 300, "k": 1000, "F": 200, "dtype": F32}], ids=str)
def test_calls_repeat_bit_for_bit_on_other_streams_and_side_by_side(args):
    args = _all_args(**args)
    want = _all_calls(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [_all_calls(*args) for _ in range(4)]
    torch.cuda.synchronize()
    for g in got:
        assert all(bits_equal(a, b) for a, b in zip(g, want))


@without_bands
@pytest.mark.parametrize("args", [{}, {"odd": 3}, {"M": 300, "k": 1000, "F": 200, "dtype": F32}], ids=str)
def test_captured_calls_replay_with_new_contents(args):
    """Two graphs of the same calls, replayed in turn on two streams with new inputs and a new offset; each owns what its calls used."""
    args = _all_args(**args)
    _all_calls(*args)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _all_calls(*args)
        graphs.append((g, out, torch.cuda.Stream()))
    for step in range(3):
        args[0].copy_(_randn(*args[0].shape, dtype=args[0].dtype, seed=20 + step))
        args[7][1] = 1000 * step
        torch.cuda.synchronize()
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = _all_calls(*args)
        for _, out, _ in graphs:
            assert all(bits_equal(a, b) for a, b in zip(out, want)), step


@without_bands
def test_a_captured_training_step_beside_an_eager_one():
    """Forward and backward captured through the explicit operators while an eager autograd graph of the same leaves lives."""
    x, w = _pair(64, 128, 48, BF)
    x.requires_grad_(), w.requires_grad_()
    eager = K.gated_linear(x, w)
    dh = torch.ones_like(eager)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad():
        K.gated_linear_backward(dh, x, w, K.gated_linear_train(x, w)[1])
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            h, projections = K.gated_linear_train(x, w)
            dx, dw = K.gated_linear_backward(dh, x, w, projections)
    g.replay()
    eager.backward(dh)
    assert bits_equal(h, eager) and bits_equal(dx, x.grad) and bits_equal(dw, w.grad)


@without_bands
def test_offsets_beyond_32_bits():
    """Results of more than 2^31 elements: the last rows are those of a call on these rows alone."""
    M, k, F = 200_003, 64, 11008
    x, w = _randn(M, k, dtype=BF), _randn(2 * F, k, dtype=BF, std=0.125)
    h = K.gated_linear(x, w)
    assert h.numel() > 2**31
    for rows in (slice(0, 130), slice(100_000, 100_130), slice(M - 130, M)):
        want, tol, _, _ = ref.gated(x[rows], w, "silu", BF)
        ref.assert_within(h[rows], want, tol, str(rows))
    state, at = _state(9, 2**40), (M - 130) * F // 4 * 4
    y = K.dropout(h, 0.25, state)
    tail = K.dropout(h.view(-1)[at:], 0.25, _state(9, 2**40 + at // 4))
    assert bits_equal(y.view(-1)[at:], tail)
    del y, tail
    q, s = K.quantize_rows(h)
    want_q, want_s = _quantized(h[-130:])
    assert torch.equal(q[-130:], want_q) and torch.equal(s[-130:], want_s)
    w8 = _int8(8, F)
    out = K.mm_int8(q, w8.t(), s, torch.ones(8, device=DEV), out_dtype=F32)
    want = (q[-130:].double() @ w8.double().t()) * s[-130:].double()[:, None]
    ref.assert_within(out[-130:], want, 2.0**-22 * want.abs() + 1e-30, "int8")


# ------------------------------------------------------------------ rows that lie across lines, threads, captured gradients
def _on_lines(t, offset):
    """The values of t in rows a multiple of 128 bytes apart, the first `offset` bytes behind a line."""
    size = t.element_size()
    wide = torch.empty(t.shape[0], (t.shape[1] * size + offset + 127) // 128 * 128 // size, dtype=t.dtype, device=t.device)
    return wide[:, offset // size : offset // size + t.shape[1]].copy_(t)


@pytest.mark.parametrize("size", [(4000, 1000, 2500), (1000, 1000, 6000), (8000, 1000, 520), (300, 200, 96)], ids=["both", "input", "weight", "neither"])
def test_rows_across_lines_of_memory(size):
    """Rows on the 16-byte grid that start anywhere in a line are copied where many tiles read them: the same bits either way."""
    M, k, F = size
    x, w = _pair(M, k, F, BF)
    h, th, _, _ = ref.gated(x[-200:], w, "silu", BF)
    want = K.gated_linear(_on_lines(x, 0), _on_lines(w, 0))
    ref.assert_within(want[-200:], h, th, "h")
    assert bits_equal(K.gated_linear(x, w), want)
    assert bits_equal(K.gated_linear(_on_lines(x, 16), _on_lines(w, 48)), want)
    k8 = 2 * k + 16  # 2016 and 416 bytes
    a, b, sa, sb = _int8(M, k8), _int8(2 * F, k8), torch.rand(M, device=DEV) + 0.5, torch.rand(2 * F, device=DEV) + 0.5
    want = K.mm_int8(_on_lines(a, 0), _on_lines(b, 0).t(), sa, sb, out_dtype=F32)
    exact = (a[-200:].double() @ b.double().t()) * sa[-200:].double()[:, None] * sb.double()
    ref.assert_within(want[-200:], exact, 2.0**-22 * exact.abs() + 1e-30, "int8")  # three roundings of 2^-24
    assert bits_equal(K.mm_int8(a, b.t(), sa, sb, out_dtype=F32), want)
    assert bits_equal(K.mm_int8(_on_lines(a, 16), _on_lines(b, 112).t(), sa, sb, out_dtype=F32), want)


@without_bands
def test_calls_of_several_threads_at_once():
    """Four threads, each on a stream of its own, with calls that need scratch and calls of other sizes in between."""
    import threading

    cases = [_all_args(odd=3), _all_args(), _all_args(M=300, k=1000, F=200, dtype=F32), _all_args(M=70, k=264, F=88)]
    wants = [_all_calls(*args) for args in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [(i % 4, _all_calls(*cases[i % 4])) for i in range(first, first + 12)]
                torch.cuda.current_stream().synchronize()
            wrong.extend(i for i, g in got if not all(bits_equal(a, b) for a, b in zip(g, wants[i])))
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@without_bands
def test_gradients_captured_through_autograd():
    """A forward and backward pass through the autograd formulas in one graph, replayed with new contents."""
    x, w = _pair(96, 128, 48, BF)
    x.requires_grad_(), w.requires_grad_()
    state, dy = _state(3, 0), _randn(96, 48, dtype=BF, seed=5)

    def step():
        y = K.dropout(K.gated_linear(x, w), 0.25, state)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(2):
        with torch.no_grad():
            x.copy_(_randn(96, 128, dtype=BF, seed=30 + seed))
        state[1] = 1000 * seed
        graph.replay()
        torch.cuda.synchronize()
        assert all(bits_equal(a, b) for a, b in zip(out, step())), seed


# ------------------------------------------------------------------ both gradients in one launch
def _takes(M, F, x, w):
    J, k = 2 * F, x.shape[1]
    dp = torch.empty(M, (J + 63) // 64 * 64, dtype=x.dtype, device=DEV)
    return feedforward.lib().b200_linear_grads_scratch_bytes(dp.data_ptr(), x.data_ptr(), w.data_ptr(), M, J, k, dp.stride(0), x.stride(0), x.stride(1), w.stride(0), w.stride(1)) >= 0


@pytest.mark.parametrize("dtype", [BF, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", [(129, 72, 68), (130, 1000, 520), (256, 256, 128), (300, 267, 1000), (777, 520, 1003), (2500, 512, 300), (2000, 1000, 400), (513, 4096, 2752), (2752, 2048, 1280), (1536, 2048, 2048)], ids=str)
def test_both_gradients_in_one_launch(size, dtype):
    """dx and dW against 64 bits, sizes whose tiles are ragged, of one part alone, with the longer contraction on either side."""
    M, k, F = size
    x, w = _pair(M, k, F, dtype)
    if k % 2 == 0:
        x, w = _on_lines(x, 0), _on_lines(w, 16)  # (an odd K is copied to the grid)
    dh = _randn(M, F, dtype=dtype, seed=3)
    _, projections = K.gated_linear_train(x, w)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, "silu", dtype)
    assert _takes(M, F, x, w)
    gx, gw = K.gated_linear_backward(dh, x, w, projections)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dW")
    again = K.gated_linear_backward(dh, x, w, projections)
    assert bits_equal(gx, again[0]) and bits_equal(gw, again[1])
    # one gradient at a time is the same; operands that the launch does not take have products of their own
    one, other = K.gated_linear_backward(dh, x, w, projections, "silu", [True, False])[0], K.gated_linear_backward(dh, x, w, projections, "silu", [False, True])[1]
    assert bits_equal(one, gx) and bits_equal(other, gw)
    wt = w.t().contiguous().t()
    assert not _takes(M, F, x, wt)
    ref.assert_within(K.gated_linear_backward(dh, x, wt, projections)[0], dx, tx, "dx of a turned weight")


def test_gradients_that_are_not_finite_stay_in_their_rows():
    M, k, F = 400, 264, 304
    x, w = _pair(M, k, F, BF)
    dh = _randn(M, F, dtype=BF, seed=3)
    _, projections = K.gated_linear_train(x, w)
    assert _takes(M, F, x, w)
    cx, cw = K.gated_linear_backward(dh, x, w, projections)
    dh[33, 20] = float("nan")
    gx, gw = K.gated_linear_backward(dh, x, w, projections)
    rows, ups = [i for i in range(M) if i != 33], [i for i in range(2 * F) if i not in (20, F + 20)]
    assert gx[33].isnan().all() and bits_equal(gx[rows], cx[rows])
    assert gw[[20, F + 20]].isnan().all() and bits_equal(gw[ups], cw[ups])


@pytest.mark.parametrize("size", [(200, 512, 300), (300, 700, 333), (777, 520, 1003), (1531, 1027, 1365), (2752, 640, 400), (513, 2048, 2752)], ids=str)
def test_both_gradients_of_fp32_in_one_launch(size):
    M, k, F = size
    x, w = _pair(M, k, F, F32)
    dh = _randn(M, F, dtype=F32, seed=3)
    _, projections = K.gated_linear_train(x, w)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, "silu", F32)
    gx, gw = K.gated_linear_backward(dh, x, w, projections)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dW")
    assert (gx.double() - dx).norm() <= 1e-6 * dx.norm() and (gw.double() - dw).norm() <= 1e-6 * dw.norm()
    one, other = K.gated_linear_backward(dh, x, w, projections, "silu", [True, False])[0], K.gated_linear_backward(dh, x, w, projections, "silu", [False, True])[1]
    assert bits_equal(one, gx) and bits_equal(other, gw)
    turned = K.gated_linear_backward(dh, x.t().contiguous().t(), w.t().contiguous().t(), projections)
    assert bits_equal(turned[0], gx) and bits_equal(turned[1], gw)


@pytest.mark.parametrize("size", [(1, 72, 68), (1, 1000, 500), (17, 520, 333), (64, 2048, 700), (128, 300, 512)], ids=str)
def test_both_gradients_of_few_rows_in_one_launch(size):
    M, k, F = size
    x, w = _pair(M, k, F, BF)
    dh = _randn(M, F, dtype=BF, seed=3)
    _, projections = K.gated_linear_train(x, w)
    dx, tx, dw, tw = ref.gated_grads(dh, x, w, projections, "silu", BF)
    assert _takes(M, F, x, w)
    gx, gw = K.gated_linear_backward(dh, x, w, projections)
    ref.assert_within(gx, dx, tx, "dx")
    ref.assert_within(gw, dw, tw, "dW")
    one, other = K.gated_linear_backward(dh, x, w, projections, "silu", [True, False])[0], K.gated_linear_backward(dh, x, w, projections, "silu", [False, True])[1]
    assert bits_equal(one, gx) and bits_equal(other, gw)
