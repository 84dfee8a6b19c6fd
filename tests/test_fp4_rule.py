"""By which loop a 4-bit product goes on a device of 148 SMs, 74 pairs of CTAs: what was faster when both were timed."""
import ctypes

import pytest

from hcomm_b200 import _lib


def ask(m, n, k, experts=0, gated=False, sms=148, pairs=74, clusters=(74, 33, 15)):
    us = (ctypes.c_double * 2)()
    split = _lib.load().HcommToolFp4Estimate(m, n, k, experts, int(gated), sms, pairs, (ctypes.c_int * 3)(*clusters), us)
    return split, list(us)


def estimate(*shape):
    return ask(*shape)[1]


@pytest.mark.parametrize("shape", [(500, 3584, 8192), (256, 8192, 28672), (1024, 1024, 4096), (64, 7168, 2048, 32), (1000, 2048, 7168, 32, True), (5003, 2048, 7168, 32, True),
                                   (3000, 7168, 2048, 32), (5003, 7168, 2048, 32), (300, 14336, 4096, 8, True)])
def test_single_ctas(shape):
    single, pair = estimate(*shape)
    assert single <= pair


@pytest.mark.parametrize("shape", [(777, 3584, 8192), (1000, 4096, 4096), (200, 28672, 8192), (512, 8192, 3584), (2048, 4096, 1024), (4096, 4096, 4096), (8192, 28672, 8192),
                                   (8192, 1000, 2080), (16000, 7168, 2048, 32), (16000, 2048, 7168, 32, True), (4000, 4096, 14336, 8)])
def test_pairs(shape):
    single, pair = estimate(*shape)
    assert pair < single


@pytest.mark.parametrize("shape,splits", [((16, 8192, 28672), (2,)), ((1, 4096, 14336), (4,)), ((100, 4096, 14336), (4,)), ((1, 3584, 8192), (4,)), ((16, 8192, 3584), (1,)),
                                          ((16, 4096, 4096), (2, 4)), ((128, 1024, 4096), (4, 8)), ((16, 4096, 1024), (1,)), ((16, 28672, 8192), (1,)), ((16, 136, 96), (1,)),
                                          ((300, 1024, 4096), (4,))])
def test_ctas_that_share_a_tile(shape, splits):
    assert ask(*shape)[0] in splits


def test_nothing_is_shared_where_clusters_do_not_fit():
    assert ask(1, 4096, 14336, clusters=(31, 0, 0))[0] == 1 and ask(1, 4096, 14336, clusters=(32, 0, 0))[0] == 2
    # by expert: as many tiles as any split of the rows makes
    assert ask(8, 7168, 2048, 32)[0] == 1 and ask(1, 4096, 14336, 8)[0] == 4 and ask(2, 4096, 14336, 8)[0] == 2 and ask(2, 4096, 14336, 8, clusters=(63, 33, 15))[0] == 1
    assert ask(1, 128, 512)[0] <= 2                 # never more CTAs than stages


def test_estimates_are_near_what_was_measured():
    for shape, single, pair in (((777, 3584, 8192), 21.5, 16.0), ((4096, 4096, 4096), 36, 29), ((16000, 7168, 2048, 32), 153, 142), ((2048, 4096, 1024), 11.5, 10.5), ((256, 8192, 28672), 34.8, 41.1)):
        got = estimate(*shape)
        assert abs(got[0] / single - 1) < 0.25 and abs(got[1] / pair - 1) < 0.25, (shape, got)
    assert all(v > 0 for v in estimate(1, 1, 32)) and all(v > 0 for v in estimate(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 32, 1024, True))
