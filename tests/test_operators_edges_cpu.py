"""Refusals of the operators at the edges of their arguments' ranges, at the C ABI (no GPU: every check comes before the device is touched)."""
import pytest

from test_operators_cpu import ALL, GRAD, Attn, Rows


@pytest.mark.parametrize("scale", [2.0 ** 127, 3.0e38])
def test_scales_without_exponentials_are_refused(U, scale):
    """finite in 32 bits, but not times log2(e)"""
    a = Attn(U, scale=scale)
    assert a.forward() == -2 and a.backward() == -2
    for call in ALL:
        assert getattr(Rows(U, scale=scale), call)() == -2, call


@pytest.mark.parametrize("scale", [1e-46, 2.0 ** -150, 1e39, 3.3e38, 1e400, 2 ** 200, -1e-46, 0.0, 0, float("nan")])
def test_scales_that_32_bits_do_not_hold_are_refused(U, scale):
    with pytest.raises(ValueError):
        U.operators._scale("call", "scale", scale)
    for fine in (1, 1e-44, 0.7, 1.6e38):
        assert U.operators._scale("call", "scale", fine) == fine


@pytest.mark.parametrize("stride", [1 << 59, 1 << 61, 1 << 62, (1 << 63) - 1, -(1 << 61), -(1 << 63)])
def test_rows_whose_offsets_do_not_fit_64_bits_are_refused(U, stride):
    """the check that a gradient overlaps nothing multiplies strides by rows and bytes: a product that wraps around would let it pass"""
    for call in ALL:
        assert getattr(Rows(U, row_stride=stride), call)() == -2, call
    for call in GRAD:
        assert getattr(Rows(U, ds=stride), call)() == -2, call
