"""What the routing entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

from hcomm_b200 import _lib

PARA, PTR = 1, 2
p, f32, i64 = ctypes.c_void_p, ctypes.c_float, ctypes.c_int64


def forward(logits=64, kind=_lib.FP32, ld=8, tokens=4, experts=8, topk=2, scoring=0, bias=0, idx=64, gates=64, counts=64, scratch=64):
    return _lib.load().HcommMoeRoute(p(logits), kind, i64(ld), tokens, experts, topk, scoring, 1, f32(1), p(bias), p(0), p(idx), p(gates), p(counts), p(0), f32(0), p(0), p(scratch), p(0))


def backward(logits=64, kind=_lib.FP32, ld=8, tokens=4, experts=8, topk=2, scoring=0, idx=64, dgates=64, counts=64, dloss=64, grad=64, ld_grad=8):
    return _lib.load().HcommMoeRouteBackward(p(logits), kind, i64(ld), tokens, experts, topk, scoring, 1, f32(1), p(0), p(idx), p(dgates), p(counts), f32(1), p(dloss), p(grad), i64(ld_grad), p(0))


def test_shapes_types_and_pointers():
    for call in (forward, backward):
        for bad in (dict(kind=_lib.FP64), dict(kind=_lib.INT8), dict(tokens=-1), dict(experts=0), dict(experts=1025, ld=1025), dict(topk=0), dict(topk=9), dict(experts=64, ld=64, topk=17),
                    dict(ld=7), dict(scoring=2), dict(logits=66), dict(logits=65, kind=_lib.BF16)):
            assert call(**bad) == PARA, bad
        assert call(logits=0) == PTR
    assert forward(bias=64) == PARA
    for bad in (dict(idx=0), dict(gates=0), dict(counts=0), dict(tokens=100000, scratch=0)):
        assert forward(**bad) == PTR, bad
    assert backward(ld_grad=7) == PARA and backward(grad=66) == PARA
    for bad in (dict(grad=0), dict(idx=0), dict(counts=0)):
        assert backward(**bad) == PTR, bad
    assert backward(tokens=0, logits=0, grad=0) == 0
    loss = _lib.load().HcommMoeBalanceLoss
    assert loss(p(64), p(64), 0, 1, f32(1), p(64), p(0)) == PARA and loss(p(64), p(64), 8, 17, f32(1), p(64), p(0)) == PARA
    for bad in ((0, 64, 64), (64, 0, 64), (64, 64, 0)):
        assert loss(p(bad[0]), p(bad[1]), 8, 2, f32(1), p(bad[2]), p(0)) == PTR


def test_scratch_grows_with_the_blocks():
    from hcomm_b200.ops.router import _scratch_bytes
    assert _scratch_bytes(0, 64) == _scratch_bytes(32, 64) == 0 and _scratch_bytes(33, 64) == 2 * 129 * 4
    assert _scratch_bytes(1 << 30, 1024) == 256 * 2049 * 4
    assert _scratch_bytes(-1, 64) == _scratch_bytes(4, 0) == 0


def test_host_tensors():
    from hcomm_b200.ops.router import route
    with pytest.raises(ValueError, match="CUDA"):
        route(torch.zeros(4, 8), 2)


def test_more_tokens_than_are_counted():
    from hcomm_b200.ops.router import _scratch_bytes, route
    for tokens in ((1 << 31) - 1, (1 << 31) - 31):
        assert forward(tokens=tokens) == PARA and backward(tokens=tokens) == PARA and _scratch_bytes(tokens, 8) == 0
    with pytest.raises(ValueError, match="tokens"):
        route(torch.empty((1 << 32) + 4, 8, device="meta"), 2)
