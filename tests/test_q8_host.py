"""Host side of the rotation plan (shannon_prime_q8.h): phases against the
formula, the pairs' axes, and what is refused.  No GPU."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest


def _plan(**kw):
    import spb200
    return spb200.RopeAxes(**kw).plan


def test_phases_match_the_ladder(built_lib):
    import math
    p = _plan(head_dim=128, sections=[64], theta=10000.0)
    for i in range(64):
        want = Fraction(float(np.float32(10000.0 ** (-i / 64)))) / Fraction(2 * math.pi)   # frequencies are 32-bit floats
        # two roundings in 64-bit floats, pow and the division (2^-52 of the value), and the
        # fixed point's last place
        assert abs(Fraction(p.phase[i], 2 ** 64) - want) <= want * Fraction(1, 2 ** 51) + Fraction(1, 2 ** 64)
    p = _plan(head_dim=64, sections=[8, 24], axis_ladder=True, theta=100.0)
    assert p.phase[0] == p.phase[8]            # both axes begin at one radian a step
    assert list(p.axis)[:32] == [0] * 8 + [1] * 24


def test_interleaved_axes(built_lib):
    p = _plan(head_dim=32, sections=[2, 5, 0, 1], rot_dim=16, interleave=True)
    assert list(p.axis)[:8] == [0, 1, 3, 0, 1, 1, 1, 1]


@pytest.mark.parametrize("kw", [
    dict(head_dim=12, sections=[6]), dict(head_dim=520, sections=[260]), dict(head_dim=64, sections=[8], rot_dim=32),
    dict(head_dim=64, sections=[12]), dict(head_dim=64, sections=[48]), dict(head_dim=64, sections=[40, -8]),
    dict(head_dim=64, sections=[8, 8, 8, 4, 4]), dict(head_dim=64, sections=[]), dict(head_dim=64, sections=[32], theta=0.0),
    dict(head_dim=64, sections=[32], theta=float("inf")), dict(head_dim=64, sections=[32], freq_factors=[0.0] * 32),
    dict(head_dim=64, sections=[32], freq_factors=[float("nan")] * 32),
    dict(head_dim=64, sections=[32], freq_factors=[1e-39] * 32)])
def test_plan_refusals(built_lib, kw):
    with pytest.raises(RuntimeError):
        _plan(**kw)


def test_null_plan(built_lib):
    import spb200
    L = spb200.lib()
    assert L.sp_rope_axes_init(None, 64, 64, 0, 1, (C.c_int * 1)(32), 0, 1e4, None) == spb200.SP_ERR_ARG
    assert L.sp_cuda_q8_cache_init(None, None, 0, 64, 1, 128, None) == spb200.SP_ERR_ARG
    L.sp_cuda_q8_cache_free(None)
