"""By which loop a 4-bit product goes on a device of 148 SMs, 74 pairs of CTAs: what was faster when both were timed."""
import ctypes

import pytest

from hcomm_b200 import _lib


def estimate(m, n, k, experts=0, gated=False, sms=148, pairs=74):
    us = (ctypes.c_double * 2)()
    _lib.load().HcommToolFp4Estimate(m, n, k, experts, int(gated), sms, pairs, us)
    return list(us)


@pytest.mark.parametrize("shape", [(500, 3584, 8192), (256, 8192, 28672), (1024, 1024, 4096), (64, 7168, 2048, 32), (1000, 2048, 7168, 32, True), (5003, 2048, 7168, 32, True),
                                   (3000, 7168, 2048, 32), (300, 14336, 4096, 8, True)])
def test_single_ctas(shape):
    single, pair = estimate(*shape)
    assert single <= pair


@pytest.mark.parametrize("shape", [(777, 3584, 8192), (1000, 4096, 4096), (200, 28672, 8192), (512, 8192, 3584), (2048, 4096, 1024), (4096, 4096, 4096), (8192, 28672, 8192),
                                   (8192, 1000, 2080), (8000, 7168, 2048, 32), (16000, 2048, 7168, 32, True), (4000, 4096, 14336, 8)])
def test_pairs(shape):
    single, pair = estimate(*shape)
    assert pair < single


def test_estimates_are_near_what_was_measured():
    for shape, single, pair in (((777, 3584, 8192), 21.5, 16.0), ((4096, 4096, 4096), 37.5, 29.1), ((16000, 7168, 2048, 32), 180, 144), ((256, 8192, 28672), 34.8, 41.1)):
        got = estimate(*shape)
        assert abs(got[0] / single - 1) < 0.25 and abs(got[1] / pair - 1) < 0.25, (shape, got)
    assert all(v > 0 for v in estimate(1, 1, 32)) and all(v > 0 for v in estimate(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 32, 1024, True))
