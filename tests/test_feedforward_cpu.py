"""The linear layers of a feed-forward block without a GPU: schemas, shapes, refusals, and the reference formulas themselves."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import feedforward_ref as ref
from backendbench_b200 import _abi, custom_ops, feedforward, ops

K = torch.ops.b200


def test_the_generator_gives_its_published_vectors():
    """Known answers that go with the paper's reference implementation: counter and key all zeros, all ones, and the digits of pi."""
    assert [int(w) for w in ref.words(4, 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(w) for w in ref.words(4, -1, -1, -1)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert [int(w) for w in ref.words(4, 0x299F31D0A4093822, 0x85A308D3243F6A88, 0x0370734413198A2E)] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("name", ref.ACTS)
def test_slopes_are_those_of_the_activations(name):
    g = torch.linspace(-6, 6, 4001, dtype=torch.float64) + 1e-4  # off relu's corner
    e = 1e-5
    assert torch.allclose(ref.slope(g, name), (ref.act(g + e, name) - ref.act(g - e, name)) / (2 * e), atol=1e-9)


def test_operators_are_registered_with_their_schemas():
    for name, (schema, _, _) in feedforward.OPERATORS.items():
        op = custom_ops.operator(name)
        assert op._schema.name == f"b200::{name}"
        assert len(op._schema.arguments) == len([a for a in schema.split(") -> ")[0].strip("(").replace("*, ", "").split(", ") if " " in a])
    assert not set(feedforward.OPERATORS) & set(custom_ops.OPERATORS)


def test_fake_kernels_and_gradients_by_shape():
    with FakeTensorMode():
        x = torch.empty(3, 5, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(64, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        h = K.gated_linear(x, w, "gelu")
        assert h.shape == (3, 5, 32) and h.dtype == torch.bfloat16 and h.requires_grad
        assert not K.gated_linear(x.detach(), w.detach()).requires_grad
        out, projections = K.gated_linear_train(x, w)
        assert out.requires_grad and projections.shape == (3, 5, 64) and projections.dtype == torch.float32 and not projections.requires_grad
        dx, dw = K.gated_linear_backward(h.detach(), x.detach(), w.detach(), projections, "gelu", [True, False])
        assert dx.shape == x.shape and dw is None
        state = torch.empty(2, dtype=torch.int64, device="cuda")
        y = K.dropout(h, 0.1, state, h, subsequence=3)
        assert y.shape == h.shape and y.requires_grad
        q, scale = K.quantize_rows(x.detach())
        assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (3, 5) and scale.dtype == torch.float32
        w8 = torch.empty(40, 16, device="cuda", dtype=torch.int8)
        y = K.mm_int8(q.view(15, 16), w8.t(), scale.view(15), torch.empty(40, device="cuda"), out_dtype=torch.float16)
        assert y.shape == (15, 40) and y.dtype == torch.float16
        with pytest.raises(RuntimeError, match="cannot be multiplied"):
            K.gated_linear(x, torch.empty(64, 17, device="cuda", dtype=torch.bfloat16))


def test_there_is_no_host_path():
    x, s = torch.randn(4, 8), torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(4, 8, dtype=torch.int8)
    for call in (lambda: K.gated_linear(x, torch.randn(6, 8)), lambda: K.dropout(x, 0.1, s), lambda: K.quantize_rows(x), lambda: K.mm_int8(q, q.t(), torch.ones(4), torch.ones(4))):
        with pytest.raises(ops.UnsupportedByB200, match="no CPU path"):
            call()


@pytest.fixture
def anywhere(monkeypatch):
    """The wrappers' own checks, which come before anything touches a device."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(feedforward, "lib", lambda: pytest.fail("a refused call reached the library"))
    return feedforward


def _bad(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_refusals(anywhere):
    f, x, w = anywhere, torch.randn(4, 8), torch.randn(6, 8)
    _bad(lambda: f.gated_linear(x, w, "tanh"), ValueError, "not one of")
    _bad(lambda: f.gated_linear(x, w, None), ValueError, "not one of")
    _bad(lambda: f.gated_linear(x, w[:5]), RuntimeError, "5 rows")
    _bad(lambda: f.gated_linear(x, w[:, :7]), RuntimeError, "cannot be multiplied")
    _bad(lambda: f.gated_linear(x, w[0]), RuntimeError, "a weight of two")
    _bad(lambda: f.gated_linear(x[0, 0], w), RuntimeError, "one dimension or more")
    _bad(lambda: f.gated_linear(x, w.half()), RuntimeError, "same dtype")
    _bad(lambda: f.gated_linear(x.double(), w.double()), ops.UnsupportedByB200, "float64")
    h, p = torch.randn(4, 3), torch.randn(4, 6)
    _bad(lambda: f.gated_linear_backward(h[:, :2], x, w, p), RuntimeError, "do not go with")
    _bad(lambda: f.gated_linear_backward(h, x, w, p[:, :4]), RuntimeError, "do not go with")
    _bad(lambda: f.gated_linear_backward(h.half(), x, w, p), RuntimeError, "like the input and fp32")
    _bad(lambda: f.gated_linear_backward(h.half(), x.half(), w.half(), p.half()), RuntimeError, "fp32 projections")
    assert f.gated_linear_backward(h, x, w, p, "silu", [False, False]) == (None, None)
    s = torch.zeros(2, dtype=torch.int64)
    for p_drop in (-0.1, 1.1, float("nan")):
        _bad(lambda: f.dropout(x, p_drop, s), ValueError, "between 0 and 1")
    _bad(lambda: f.dropout(x, 0.1, s.int()), RuntimeError, "two int64")
    _bad(lambda: f.dropout(x, 0.1, s[:1]), RuntimeError, "two int64")
    _bad(lambda: f.dropout(x, 0.1, s, x[:1]), RuntimeError, "like the input")
    _bad(lambda: f.dropout(x, 0.1, s, x.half()), RuntimeError, "like the input")
    _bad(lambda: f.dropout(s, 0.1, s), ops.UnsupportedByB200, "int64")
    _bad(lambda: f.quantize_rows(s), ops.UnsupportedByB200, "int64")
    _bad(lambda: f.quantize_rows(x[0, 0]), RuntimeError, "one dimension or more")
    q, b, r, c = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(8, 3, dtype=torch.int8), torch.ones(4), torch.ones(3)
    _bad(lambda: f.mm_int8(q, b[:7], r, c), RuntimeError, "cannot be multiplied")
    _bad(lambda: f.mm_int8(q[0], b, r, c), RuntimeError, "must be matrices")
    _bad(lambda: f.mm_int8(q, b.to(torch.uint8), r, c), ops.UnsupportedByB200, "uint8")
    _bad(lambda: f.mm_int8(q, b, c, c), RuntimeError, "4 fp32 values, one to each row")
    _bad(lambda: f.mm_int8(q, b, r, r), RuntimeError, "3 fp32 values, one to each column")
    _bad(lambda: f.mm_int8(q, b, r.double(), c), RuntimeError, "fp32 values")
    _bad(lambda: f.mm_int8(q, b, r, c, c[:2]), RuntimeError, "bias must be")
    _bad(lambda: f.mm_int8(q, b, r, c, c, out_dtype=torch.float16), RuntimeError, "bias must be")
    _bad(lambda: f.mm_int8(q, b, r, c, out_dtype=torch.int32), ops.UnsupportedByB200, "out_dtype")
    long = torch.zeros(1, dtype=torch.int8).expand(1, 131072)
    _bad(lambda: f.mm_int8(long, long.t(), r[:1], c[:1]), ops.UnsupportedByB200, "overflow")


def test_the_library_refuses_what_the_wrappers_would(monkeypatch):
    lib, BF, F32 = _abi.lib(), _abi.BF16, _abi.F32
    g = lambda *a: lib.b200_gated_linear(None, None, None, None, *a, None, 0, None, None)
    assert g(-1, 4, 4, 4, 1, 4, 1, 0, BF) == -1 and g(4, 4, 4, 4, 1, 4, 1, 5, BF) == -1 and g(4, 4, 4, 4, 1, 4, 1, -1, BF) == -1
    assert g(4, 4, 4, 4, 1, 4, 1, 0, F32) == -2 and g(4, 4, 4, 4, 1, 4, 1, 0, BF) == -1 and g(0, 4, 4, 4, 1, 4, 1, 0, BF) == 0
    base = 1 << 20  # an aligned address that nobody looks behind
    assert lib.b200_gated_linear_scratch_bytes(base, base, 4, 8, 64, 64, 1, 64, 1) == 0
    assert lib.b200_gated_linear_scratch_bytes(base, base, 4, 8, 63, 63, 1, 63, 1) >= 4 * 64 * 2 + 16 * 64 * 2
    assert lib.b200_mm_int8_scratch_bytes(base, base, 4, 8, 64, 64, 1, 1, 64) == 0  # B as the transpose of rows along K
    assert lib.b200_mm_int8_scratch_bytes(base, base, 4, 8, 64, 64, 1, 8, 1) >= 8 * 64
    m = lambda *a: lib.b200_mm_int8(None, None, None, None, None, None, *a, None, 0, None, None)
    assert m(4, 4, 131072, 4, 1, 4, 1, BF) == -1 and m(4, 4, 4, 4, 1, 4, 1, _abi.I32) == -2 and m(4, 0, 4, 4, 1, 4, 1, BF) == 0 and m(4, 4, 4, 4, 1, 4, 1, BF) == -1
    f = lambda *a: lib.b200_linear_f32(None, None, None, *a, None, 0, None, None)
    assert f(4, 4, 4, 4, 1, 4, 1) == -1 and f(0, 4, 4, 4, 1, 4, 1) == -1
    assert lib.b200_linear_f32(base, base, base, 128, 128, 128, 128, 1, 128, 1, None, 0, None, None) == -4
    assert lib.b200_gated_linear_f32(base, base, base, None, 128, 128, 128, 128, 1, 128, 1, 7, None, 0, None, None) == -1
    assert lib.b200_linear_f32_scratch_bytes(64, 4096, 4096) == lib.b200_linear_f32_scratch_bytes(128, 128, 128) == lib.b200_linear_f32_scratch_bytes(0, 1, 1) == 0
    assert lib.b200_dropout(None, None, None, 4, 1.5, None, 0, BF, None) == -1 and lib.b200_dropout(None, None, None, 0, 0.5, None, 0, BF, None) == 0
    assert lib.b200_dropout(None, None, None, 4, 0.5, None, 0, _abi.I8, None) == -2 and lib.b200_dropout(None, None, None, 4, 0.5, None, 0, BF, None) == -1
    assert lib.b200_gate(None, None, 4, 4, 9, None) == -1 and lib.b200_gate_backward(None, None, None, 4, 4, 0, _abi.I32, None) == -2
    assert lib.b200_quantize_rows(None, None, None, 4, 4, 4, BF, None) == -1 and lib.b200_quantize_rows(None, None, None, 0, 4, 4, BF, None) == 0
