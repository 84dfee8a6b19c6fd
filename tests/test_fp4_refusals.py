"""What the 4-bit operators refuse, and their layout of scales, without a GPU."""
import ctypes

import pytest
import torch

from hcomm_b200 import _lib
from hcomm_b200.ops.fp4 import Fp4Tensor, _check_operand, _scale_tiles, dequantize_fp4, gemm_fp4, gemm_fp4_swiglu, quantize_fp4

PARA, PTR = 1, 2


def i64(v):
    return ctypes.c_int64(v)


@pytest.mark.parametrize("shape", [(1, 32), (130, 96), (3, 129, 416), (2, 256, 128)])
def test_scales_go_into_tiles_and_back(shape):
    g = torch.Generator().manual_seed(1)
    plain = torch.randint(0, 256, (*shape[:-1], shape[-1] // 32), generator=g, dtype=torch.uint8)
    q = Fp4Tensor.from_parts(torch.zeros((*shape[:-1], shape[-1] // 2), dtype=torch.uint8), plain)
    assert q.shape == shape and torch.equal(q.block_scales(), plain)
    *batch, rows, cols = shape
    flat, tiles = q.scales.view(-1), -(-cols // 128)
    for b in range(batch[0] if batch else 1):
        for r in range(0, rows, 7):
            for c in range(cols // 32):
                tile = (b * -(-rows // 128) + r // 128) * tiles + c // 4
                assert flat[tile * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4] == plain.view(-1, rows, cols // 32)[b, r, c]


def test_bytes_of_scales():
    size = _lib.load().HcommFp4ScaleBytes
    size.restype = ctypes.c_uint64
    for batch, rows, cols, experts in ((1, 1, 32, 0), (1, 128, 128, 0), (3, 129, 160, 0), (1, 300, 256, 4), (1, 2, 64, 100), (1, 0, 64, 5), (1, 1 << 30, 8192, 1024)):
        assert size(i64(batch), i64(rows), i64(cols), experts) == 512 * _scale_tiles(batch, rows, cols, experts)


def quantize(x=64, kind=_lib.BF16, xs=0, batch=1, rows=4, cols=64, batch_pitch=0, row_pitch=64, scale_pitch=0, offsets=0, experts=0, values=64, scales=64):
    p = ctypes.c_void_p
    return _lib.load().HcommFp4Quantize(p(x), kind, p(xs), i64(batch), i64(rows), i64(cols), i64(batch_pitch), i64(row_pitch), i64(scale_pitch), p(offsets), experts,
                                        p(values), p(scales), p(0))


def test_quantise_refuses():
    for bad in (dict(cols=48), dict(cols=-32), dict(rows=-1), dict(rows=1 << 31), dict(rows=(1 << 31) - 1), dict(batch=1 << 20, rows=1 << 11), dict(row_pitch=-1), dict(batch_pitch=-1, batch=2), dict(values=72), dict(scales=72), dict(kind=_lib.FP64), dict(kind=_lib.INT8),
                dict(kind=_lib.FP8E4M3, xs=64), dict(kind=_lib.FP8E4M3, xs=64, cols=128, row_pitch=128, scale_pitch=-1), dict(kind=_lib.FP8E4M3, xs=64, cols=128, row_pitch=128, batch=2, scale_pitch=1),
                dict(experts=2), dict(offsets=64), dict(offsets=64, experts=1025), dict(offsets=64, experts=2, batch=2), dict(experts=-1)):
        assert quantize(**bad) == PARA, bad
    for bad in (dict(x=0), dict(values=0), dict(scales=0), dict(kind=_lib.FP8E4M3, cols=128, row_pitch=128, scale_pitch=1)):
        assert quantize(**bad) == PTR, bad
    for empty in (dict(rows=0), dict(cols=0), dict(batch=0), dict(rows=0, x=0, values=0, scales=0)):
        assert quantize(**empty) == 0, empty


def test_dequantise_refuses():
    def call(values=64, scales=64, batch=1, rows=4, cols=64, offsets=0, experts=0, out=64, kind=_lib.BF16):
        p = ctypes.c_void_p
        return _lib.load().HcommFp4Dequantize(p(values), p(scales), i64(batch), i64(rows), i64(cols), p(offsets), experts, p(out), kind, p(0))
    for bad in (dict(cols=40), dict(out=72), dict(kind=_lib.FP8E4M3), dict(experts=3), dict(offsets=64, experts=2, batch=3)):
        assert call(**bad) == PARA, bad
    for bad in (dict(values=0), dict(scales=0), dict(out=0)):
        assert call(**bad) == PTR, bad
    assert call(rows=0) == 0


def test_products_refuse():
    def call(m=4, n=8, k=64, ld=8, offsets=0, experts=0, out=64, ops=(64,) * 6, gated=False):
        p = ctypes.c_void_p
        fn = _lib.load().HcommFp4GemmSwiglu if gated else _lib.load().HcommFp4Gemm
        return fn(*[p(o) for o in ops[:6 if gated else 4]], p(out), m, n, k, i64(ld), p(offsets), experts, p(0))
    for gated in (False, True):
        for bad in (dict(k=48), dict(k=0), dict(m=-1), dict(n=-1), dict(m=(1 << 31) - 1), dict(n=(1 << 31) - 1, ld=1 << 31), dict(ld=7), dict(experts=2), dict(offsets=64), dict(offsets=64, experts=1025), dict(out=65),
                    dict(ops=(72, 64, 64, 64, 64, 64)), dict(ops=(64, 64, 64, 72, 64, 64))):
            assert call(gated=gated, **bad) == PARA, bad
        for bad in (dict(out=0), dict(ops=(0, 64, 64, 64, 64, 64)), dict(ops=(64, 64, 64, 0, 64, 64))):
            assert call(gated=gated, **bad) == PTR, bad
        for empty in (dict(m=0), dict(n=0)):
            assert call(gated=gated, **empty) == 0
    assert call(gated=True, ops=(64, 64, 64, 64, 0, 64)) == PTR


def test_host_tensors_and_parts_that_do_not_fit():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_fp4(x)
    u8 = torch.uint8
    q = Fp4Tensor.from_parts(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 2, dtype=u8))
    for call in (lambda: dequantize_fp4(q), lambda: gemm_fp4(q, q), lambda: gemm_fp4_swiglu(q, q, q)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        gemm_fp4(x, q)
    with pytest.raises(TypeError):
        _check_operand("it", x)
    with pytest.raises(TypeError):
        Fp4Tensor.from_parts(torch.zeros(4, 32), torch.zeros(4, 2))
    for values, scales in (((4, 32), (4, 3)), ((4, 32), (5, 2)), ((4, 24), (4, 2))):
        with pytest.raises(ValueError):
            Fp4Tensor.from_parts(torch.zeros(values, dtype=u8), torch.zeros(scales, dtype=u8))
    grouped = Fp4Tensor(q.values, q.scales, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        grouped.block_scales()


@pytest.mark.parametrize("m, n", [((1 << 32) + 5, 8), (8, (1 << 32) + 5), ((1 << 31) - 256, 8)])
def test_products_refuse_more_rows_than_they_count(monkeypatch, m, n):
    """Sizes go to the library as 32-bit numbers: none may be cut to its lower bits."""
    from hcomm_b200.ops import fp4
    monkeypatch.setattr(fp4, "_on_device", lambda what, *tensors: tensors[0].device)

    def operand(rows):
        return Fp4Tensor(torch.empty((rows, 16), dtype=torch.uint8, device="meta"), torch.empty((_scale_tiles(1, rows, 32, 0), 512), dtype=torch.uint8, device="meta"))
    with pytest.raises(ValueError, match="at most"):
        fp4._result("gemm_fp4", operand(m), (operand(n),), None)


@pytest.mark.parametrize("k", [(1 << 31) - 256, (1 << 31) - 224, (1 << 31) - 128, (1 << 31) - 32])
@pytest.mark.parametrize("gated", [False, True])
def test_products_refuse_a_depth_that_32_bits_cannot_round_up(k, gated):
    p = ctypes.c_void_p
    fn = _lib.load().HcommFp4GemmSwiglu if gated else _lib.load().HcommFp4Gemm
    assert fn(*[p(64)] * (6 if gated else 4), p(64), 1, 1, k, i64(1), p(0), 0, p(0)) == PARA


@pytest.mark.parametrize("rows,cols", [((1 << 30) + (1 << 26), 288), ((1 << 31) - (1 << 20) - 1, 32), ((1 << 31) - (1 << 20) - 1, 288), ((1 << 31) - (1 << 20) - 1, 640), (1 << 30, 384), (5, 288),
                                       (1, 32 * 200001), (100000, 8192)])
@pytest.mark.parametrize("kind", [_lib.BF16, _lib.FP8E4M3])
def test_no_team_of_the_quantiser_takes_a_row_that_is_not_its_own(rows, cols, kind):
    """A team goes round as often as the busiest; the numbers of the rows behind the last one must not come back as those of others."""
    cols = -(-cols // 128) * 128 if kind == _lib.FP8E4M3 else cols
    walk = _lib.load().HcommToolFp4Walk
    walk.restype = ctypes.c_int64

    def follow(team):
        return walk(i64(rows), i64(cols), kind, 148, i64(team))
    teams = follow(0)
    assert teams >= -(-cols // 128)
    for team in (teams - 1, teams - 2, teams // 2, 1):
        assert follow(team) == teams, team


@pytest.mark.parametrize("shape", [(0, 64), (4, 0), (0, 4, 64), (3, 0, 64), (3, 4, 0)])
def test_parts_of_nothing(shape):
    """What quantize_fp4 makes of an empty matrix: an expert that a rank does not have, or a layer without rows."""
    scales = torch.zeros((*shape[:-1], shape[-1] // 32), dtype=torch.uint8)
    q = Fp4Tensor.from_parts(torch.zeros((*shape[:-1], shape[-1] // 2), dtype=torch.uint8), scales)
    *batch, rows, cols = shape
    assert q.shape == shape and q.scales.shape == (_scale_tiles(batch[0] if batch else 1, rows, cols, 0), 512)
    assert torch.equal(q.block_scales(), scales)
