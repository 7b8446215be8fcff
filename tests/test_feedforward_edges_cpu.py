"""Refusals of the C entries for f16 gradients, without a GPU."""

from backendbench_b200 import _abi

BASE = 1 << 20  # an aligned address that nobody looks behind


def test_entries_for_f16_gradients_refuse_bad_arguments():
    lib, BF, F16 = _abi.lib(), _abi.BF16, _abi.F16
    gate = lambda *a: lib.b200_gate_backward_scaled(*a, None)
    assert gate(BASE, BASE, BASE, BASE, BASE, 7, 4, 4, 0) == -1  # rows of 8 elements, 7 apart
    assert gate(BASE, BASE, BASE, BASE, BASE, 8, -1, 4, 0) == -1 and gate(BASE, BASE, BASE, BASE, BASE, 8, 4, 4, 5) == -1
    assert gate(BASE, BASE, None, None, BASE, 8, 4, 4, 0) == -1 and gate(BASE, BASE, BASE, None, None, 8, 4, 4, 0) == -1 and gate(None, BASE, BASE, None, BASE, 8, 4, 4, 0) == -1
    assert gate(None, None, None, None, None, 8, 0, 4, 0) == 0 and gate(None, None, None, None, None, 0, 4, 0, 0) == 0
    product = lambda a, most, b, out, *s: lib.b200_linear_scaled(a, most, b, out, *s, None, 0, None, None)
    assert product(BASE, None, BASE, BASE, 4, 8, 64, 64, 1, 1, 64) == -1 and product(BASE, BASE, BASE, None, 4, 8, 64, 64, 1, 1, 64) == -1
    assert product(BASE, BASE, BASE, BASE, -1, 8, 64, 64, 1, 1, 64) == -1 and product(BASE, BASE, BASE, BASE, 4, 8, 0, 1, 1, 1, 1) == -1
    assert product(None, None, None, None, 0, 8, 64, 64, 1, 1, 64) == 0
    assert lib.b200_linear_scaled_scratch_bytes(BASE, BASE, 4, 8, 64, 64, 1, 1, 64) == 0  # B as the transpose of rows along K
    assert lib.b200_linear_scaled_scratch_bytes(BASE, BASE, 4, 8, 64, 64, 1, 8, 1) >= 8 * 64 * 2
    grads = lambda *operands: lib.b200_linear_grads_scaled(*operands, 256, 256, 256, 256, 256, 256, None, 0, None, None)
    assert grads(BASE, BASE, None, BASE, BASE, BASE, BASE) == -1  # without the magnitudes
    assert grads(BASE, None, BASE, BASE, BASE, BASE, BASE) == -1 and grads(None, BASE, BASE, BASE, BASE, BASE, BASE) == -1
    assert grads(BASE, BASE, BASE, BASE, BASE, None, None) == -1 and grads(BASE, BASE, BASE, None, BASE, BASE, BASE) == -1
    plain = lambda g, dx, dw, dtype: lib.b200_linear_grads(g, BASE, BASE, dx, dw, 256, 256, 256, 256, 256, 256, dtype, None, 0, None, None)
    assert plain(None, BASE, BASE, BF) == -1 and plain(BASE, None, None, F16) == -1 and plain(BASE, BASE, BASE, _abi.F32) == -2
