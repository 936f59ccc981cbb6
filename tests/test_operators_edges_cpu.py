"""Refusals of the operators at the edges of their arguments' ranges, at the C ABI (no GPU: every check comes before the device is touched)."""
import ctypes

import numpy as np
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


def test_match_log_probs_targets_that_are_no_32_bit_integers(U, monkeypatch):
    """an index beyond 32 bits is none of the candidates (it wrapped around to one), and a fraction no index at all"""
    seen = []

    class Library:
        def urf_sg_match_log_probs(self, h, targets, *rest):
            seen.append(np.ctypeslib.as_array(ctypes.cast(targets, ctypes.POINTER(ctypes.c_int)), (3,)).tolist())
            return 0

    monkeypatch.setattr(U._lib, "lib", lambda: Library())
    sg = U.frontend.SuperGlue.__new__(U.frontend.SuperGlue)
    sg._h, sg._n0 = None, 3
    for given in (np.array([3, (1 << 32) + 3, -(1 << 32) + 3]), [3, 1 << 40, -5], np.array([3, (1 << 63) + 3, 1 << 32], np.uint64)):
        sg.match_log_probs(given)
        assert seen[-1][0] == 3 and all(t < 0 or t > 1024 for t in seen[-1][1:]), seen[-1]
    sg.match_log_probs(np.array([1, -1, 70], np.int32))
    assert seen[-1] == [1, -1, 70]
    for given in (np.array([0.5, 1.0, 2.0]), [1.0, 2.0, 3.0], np.array(["1", "2", "3"]), np.array([1, 2])):
        with pytest.raises(ValueError):
            sg.match_log_probs(given)
